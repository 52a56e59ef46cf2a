// Loads and stores of the row operators: four consecutive elements of a row at a time, fp32 or bf16 in memory, fp32 in
// registers.
#pragma once
#include <hip/hip_runtime.h>

namespace snhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Raw4;  // four elements as they lie in memory
template <>
struct Raw4<float> {
    typedef f32x4 type;
};
template <>
struct Raw4<__bf16> {
    typedef bf16x4 type;
};

// Elements [c, c + 4) of a row of `cols`; `whole`: the row starts on four elements' alignment and cols is a multiple of
// four, so the piece is one 16- or 8-byte access; otherwise element by element, zeros behind the row's end.
// As they lie in memory: nothing is done with them in the branch, so nothing waits for them there and the loads of several
// rows are under way together (a conversion beside each load costs half the bandwidth).
template <typename T>
__device__ __forceinline__ typename Raw4<T>::type load4_raw(const T* row, int c, int cols, bool whole) {
    typedef typename Raw4<T>::type raw;
    if (whole) return *reinterpret_cast<const raw*>(row + c);
    raw v = {(T)0.0f, (T)0.0f, (T)0.0f, (T)0.0f};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < cols) v[j] = row[c + j];
    return v;
}
__device__ __forceinline__ f32x4 widen(f32x4 v) { return v; }
__device__ __forceinline__ f32x4 widen(bf16x4 v) { return __builtin_convertvector(v, f32x4); }
template <typename T>
__device__ __forceinline__ f32x4 load4(const T* row, int c, int cols, bool whole) {
    return widen(load4_raw(row, c, cols, whole));
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
