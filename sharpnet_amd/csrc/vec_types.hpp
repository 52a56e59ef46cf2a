// Loads and stores of the row operators: four consecutive elements of a row at a time, fp32 or bf16 in memory, fp32 in
// registers.
#pragma once
#include <hip/hip_runtime.h>

namespace snhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

// Elements [c, c + 4) of a row of `cols`; `whole`: the row starts on four elements' alignment and cols is a multiple of
// four, so the piece is one 16- or 8-byte access; otherwise element by element, zeros behind the row's end.
__device__ __forceinline__ f32x4 load4(const float* row, int c, int cols, bool whole) {
    if (whole) return *reinterpret_cast<const f32x4*>(row + c);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < cols) v[j] = row[c + j];
    return v;
}
__device__ __forceinline__ f32x4 load4(const __bf16* row, int c, int cols, bool whole) {
    if (whole) return __builtin_convertvector(*reinterpret_cast<const bf16x4*>(row + c), f32x4);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < cols) v[j] = (float)row[c + j];
    return v;
}
__device__ __forceinline__ void store4(float* row, int c, int cols, bool whole, f32x4 v) {
    if (whole) {
        *reinterpret_cast<f32x4*>(row + c) = v;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < cols) row[c + j] = v[j];
}
// (the conversion rounds to nearest even)
__device__ __forceinline__ void store4(__bf16* row, int c, int cols, bool whole, f32x4 v) {
    if (whole) {
        *reinterpret_cast<bf16x4*>(row + c) = __builtin_convertvector(v, bf16x4);
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < cols) row[c + j] = (__bf16)v[j];
}
// v as it reads back after a store in type T
__device__ __forceinline__ f32x4 as_stored(f32x4 v, const float*) { return v; }
__device__ __forceinline__ f32x4 as_stored(f32x4 v, const __bf16*) {
    return __builtin_convertvector(__builtin_convertvector(v, bf16x4), f32x4);
}

}  // namespace snhip
