// Loads, stores and sums of the row operators: four consecutive elements of a row at a time, fp32 or bf16 in memory, fp32 in
// registers.
#pragma once
#include <hip/hip_runtime.h>

namespace snhip {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
// the same at any address of an element: the hardware takes wide accesses there, a row may start anywhere
typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef bf16x4 bf16x4_any __attribute__((aligned(2)));

template <typename T>
struct Raw4;  // four elements as they lie in memory
template <>
struct Raw4<float> {
    typedef f32x4 type;
    typedef f32x4_any any;
};
template <>
struct Raw4<__bf16> {
    typedef bf16x4 type;
    typedef bf16x4_any any;
};
template <typename T>
using raw4 = typename Raw4<T>::type;

__device__ __forceinline__ f32x4 widen(f32x4 v) { return v; }
__device__ __forceinline__ f32x4 widen(bf16x4 v) { return __builtin_convertvector(v, f32x4); }
// (rounds to nearest even)
__device__ __forceinline__ f32x4 narrow(f32x4 v, const float*) { return v; }
__device__ __forceinline__ bf16x4 narrow(f32x4 v, const __bf16*) { return __builtin_convertvector(v, bf16x4); }
// v as it reads back after a store in type T
template <typename T>
__device__ __forceinline__ f32x4 as_stored(f32x4 v) {
    return widen(narrow(v, static_cast<const T*>(nullptr)));
}

// Four whole elements from `at` on.  The loads return them as they lie in memory: a conversion beside each load would wait
// for it, and the loads of several rows would not be under way together (half the bandwidth).
template <typename T>
__device__ __forceinline__ raw4<T> load4_whole(const T* at) {
    return *reinterpret_cast<const typename Raw4<T>::any*>(at);
}
template <typename T>
__device__ __forceinline__ void store4_whole(T* at, f32x4 v) {
    *reinterpret_cast<typename Raw4<T>::any*>(at) = narrow(v, static_cast<const T*>(nullptr));
}
// The same for data that is read or written once and will not be found in a cache again.
template <typename T>
__device__ __forceinline__ raw4<T> load4_once(const T* at) {
    return __builtin_nontemporal_load(reinterpret_cast<const typename Raw4<T>::any*>(at));
}
template <typename T>
__device__ __forceinline__ void store4_once(T* at, f32x4 v) {
    __builtin_nontemporal_store(narrow(v, static_cast<const T*>(nullptr)), reinterpret_cast<typename Raw4<T>::any*>(at));
}
// The same for a piece of which `left` elements exist (0 or less: none): one access, or element by element at a row's end;
// what does not exist reads as zero.
template <typename T, bool ONCE = false>
__device__ __forceinline__ raw4<T> load4(const T* at, int left) {
    if (left >= 4) return ONCE ? load4_once(at) : load4_whole(at);
    raw4<T> v = {};
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < left) v[j] = at[j];
    return v;
}
template <typename T, bool ONCE = false>
__device__ __forceinline__ void store4(T* at, int left, f32x4 v) {
    if (left >= 4) return ONCE ? store4_once(at, v) : store4_whole(at, v);
#pragma unroll
    for (int j = 0; j < 3; ++j)
        if (j < left) at[j] = (T)v[j];
}

// Columns [c, c + 4) of a row of dim elements, c a multiple of four: the loads of many rows without a branch in between.  Near
// the row's end (and behind it) the row's last four elements are read; existing() moves those that are asked for to their
// places and clears the rest, once they are used.
template <typename T, bool ONCE = false>
__device__ __forceinline__ raw4<T> load4_row(const T* row, int c, int dim) {
    if (dim >= 4) {
        const T* at = row + (c < dim - 4 ? c : dim - 4);
        return ONCE ? load4_once(at) : load4_whole(at);
    }
    raw4<T> v = {};
#pragma unroll
    for (int j = 0; j < 3; ++j)  // (a row of up to three: as the end of one of four)
        if (c == 0 && j < dim) v[j + 4 - dim] = row[j];
    return v;
}
// `ends`: whether a lane of the wavefront is at a row's end (most pieces have none: nothing to do).
__device__ __forceinline__ f32x4 existing(f32x4 v, int left, bool ends) {
    if (!ends || left >= 4) return v;
    f32x4 r = {0.0f, 0.0f, 0.0f, 0.0f};
    if (left == 3) r = f32x4{v[1], v[2], v[3], 0.0f};
    if (left == 2) r = f32x4{v[2], v[3], 0.0f, 0.0f};
    if (left == 1) r[0] = v[3];
    return r;
}

// Sums over 16 or 32 neighbouring lanes / over the wavefront, in every lane of them, without going through LDS: rotations within
// rows of 16 lanes are free operands of the additions (ds_bpermute, what a shuffle becomes, is a round trip each).
template <int ROTATE>
__device__ __forceinline__ float add_rotated(float v) {
    constexpr int row_ror = 0x120;
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), row_ror + ROTATE, 0xf, 0xf, false));
}
__device__ __forceinline__ float row16_sum(float v) {
    v = add_rotated<8>(v);
    v = add_rotated<4>(v);
    v = add_rotated<2>(v);
    return add_rotated<1>(v);
}
__device__ __forceinline__ float wave64_sum(float v) {
    const int r = __float_as_int(row16_sum(v));
    const float a = __int_as_float(__builtin_amdgcn_readlane(r, 0)), b = __int_as_float(__builtin_amdgcn_readlane(r, 16));
    const float c = __int_as_float(__builtin_amdgcn_readlane(r, 32)), d = __int_as_float(__builtin_amdgcn_readlane(r, 48));
    return (a + b) + (c + d);
}
__device__ __forceinline__ float half32_sum(float v) {
    const int r = __float_as_int(row16_sum(v));
    const float a = __int_as_float(__builtin_amdgcn_readlane(r, 0)), b = __int_as_float(__builtin_amdgcn_readlane(r, 16));
    const float c = __int_as_float(__builtin_amdgcn_readlane(r, 32)), d = __int_as_float(__builtin_amdgcn_readlane(r, 48));
    return threadIdx.x & 32 ? c + d : a + b;
}

// Launches that can have more workgroups than the 2^32 - 1 threads of a grid's x hold are spread over x and z, with up to 8 z
// workgroups too many: a kernel looks at its number.
inline dim3 many_blocks(long long blocks, unsigned int y = 1) {
    const long long z = (blocks + 65535) >> 16, x = z > 1 ? ((blocks + z - 1) / z + 7) / 8 * 8 : blocks;
    return dim3((unsigned int)x, y, (unsigned int)z);
}
__device__ __forceinline__ long long block_number() { return (long long)blockIdx.z * gridDim.x + blockIdx.x; }

}  // namespace snhip
