// AdamW over the elements of many tensors in one launch (definitions: include/sharpnet_hip.h, snhip_adamw_create).
// Bound by HBM: 28 bytes an element with states in 32 bits, 16 with states in 8 (and an fp32 gradient), each read and
// written once: 143M elements with fp32 states and bf16 copies (4.28 GB) 700 to 740 us, 5.8 to 6.1 TB/s; 353M with states in 8
// bits, bf16 gradients and copies (5.66 GB) 960 to 985 us, 5.8 TB/s.  The 8-bit form is near the vector units' rate as well:
// with a correctly rounded square root, maxima through LDS and 64-bit addresses it took 1120 us.
// A workgroup of 256 threads updates a chunk of a tensor, four neighbouring elements to a thread: longer chunks only put off
// the next loads (66M elements, states in 32 / 8 bits: 315 / 178 us, chunks of four times the length 324 / 187 us).
// FULL: all of a chunk's elements exist; the tail of a tensor goes the other way.
#pragma once
#include <hip/hip_runtime.h>

#include "philox.hpp"
#include "vec_types.hpp"

namespace snhip {

typedef unsigned int u32_any __attribute__((aligned(1)));  // four bytes at any address

constexpr int kAdamwBlock = 256;              // elements that share a power of two (states in 8 bits)
constexpr int kAdamwChunk = 4 * kAdamwBlock;  // elements of a workgroup
// ONCE, from this many elements on: a plan's data does not go through the caches.  A step on less finds all of it in the 256 MB
// behind the L2s again (3.2 million: 14.5 us both ways); one on more writes over what it would have found (7.1 million: 34.5 us
// through the caches, 33.0 around them; 33 million: 170 us, 151).
constexpr long long kAdamwOnce = 1LL << 22;

struct AdamwEntry {
    float* p;
    const void* g;
    void *m, *v;
    unsigned char *m_scale, *v_scale;
    __bf16* copy;
    long long count;
    long long first_chunk;  // of the launch
    float decay;
    int g_bf16;
};

struct AdamwScalars {
    float beta1, rest1, beta2, rest2;  // rest = 1 - beta, taken in 64 bits
    float rate, step_size, root_scale, eps, grad_scale;  // learning rate; rate / (1 - beta1^t); 1 / sqrt(1 - beta2^t)
    unsigned int key0, key1, step;
};

// m' and v' with every product and sum rounded by itself, so that the 8-bit states are a function of their definition
// alone and not of how a compiler contracts them.
__device__ __forceinline__ float moment1(float m, float g, const AdamwScalars& s) {
#pragma clang fp contract(off)
    const float a = m * s.beta1, b = g * s.rest1;
    return a + b;
}
__device__ __forceinline__ float moment2(float v, float g, const AdamwScalars& s) {
#pragma clang fp contract(off)
    const float a = v * s.beta2, b = (g * g) * s.rest2;
    return a + b;
}
// (The hardware's square root, 1 ulp for a normal number: a smaller one goes in times 2^96.  The hardware's reciprocal, 1 ulp:
// the denominator is 0 or between 1e-23 and 1e20.)
__device__ __forceinline__ float new_parameter(float p, float m, float v, float keep, const AdamwScalars& s) {
    const bool tiny = v < 0x1p-96f;
    const float root = __builtin_amdgcn_sqrtf(tiny ? v * 0x1p+96f : v) * (tiny ? s.root_scale * 0x1p-48f : s.root_scale);
    return p * keep - s.step_size * (m * __builtin_amdgcn_rcpf(root + s.eps));
}

// ---- access ------------------------------------------------------------------------------------------------------
// Elements [i, i + 4) from a base that is the same for the whole wavefront (`left` of them exist if not FULL).  The addresses
// come out of a table in memory: that they are global memory has to be said.
#define SNHIP_GLOBAL __attribute__((address_space(1)))
template <typename T, bool ONCE, bool FULL>
__device__ __forceinline__ raw4<T> take4(const T* base, unsigned int i, int left) {
    if constexpr (FULL) {
        typedef typename Raw4<T>::any any;
        const SNHIP_GLOBAL any* at = (const SNHIP_GLOBAL any*)((const SNHIP_GLOBAL char*)base + i * (unsigned int)sizeof(T));
        return ONCE ? __builtin_nontemporal_load(at) : *at;
    } else {
        return load4<T, ONCE>(base + i, left);
    }
}
template <typename T, bool ONCE, bool FULL>
__device__ __forceinline__ void give4(T* base, unsigned int i, int left, f32x4 v) {
    if constexpr (FULL) {
        typedef typename Raw4<T>::any any;
        SNHIP_GLOBAL any* at = (SNHIP_GLOBAL any*)((SNHIP_GLOBAL char*)base + i * (unsigned int)sizeof(T));
        if (ONCE)
            __builtin_nontemporal_store(narrow(v, static_cast<const T*>(nullptr)), at);
        else
            *at = narrow(v, static_cast<const T*>(nullptr));
    } else {
        store4<T, ONCE>(base + i, left, v);
    }
}
// four bytes of an 8-bit state
template <bool FULL>
__device__ __forceinline__ unsigned int take_bytes(const unsigned char* base, unsigned int i, int left) {
    if constexpr (FULL) return *(const SNHIP_GLOBAL u32_any*)((const SNHIP_GLOBAL char*)base + i);
    unsigned int bytes = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < left) bytes |= (unsigned int)base[i + j] << (8 * j);
    return bytes;
}
template <bool FULL>
__device__ __forceinline__ void give_bytes(unsigned char* base, unsigned int i, int left, unsigned int bytes) {
    if constexpr (FULL) {
        *(SNHIP_GLOBAL u32_any*)((SNHIP_GLOBAL char*)base + i) = bytes;
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (j < left) base[i + j] = (unsigned char)(bytes >> (8 * j));
}
// Four elements of the gradient as they lie in memory, and what they are worth: the conversion is kept away from the load,
// so that the other loads of the same elements do not wait for it.
struct RawGradient {
    f32x4 f;
    bf16x4 b;
};
template <bool ONCE, bool FULL>
__device__ __forceinline__ RawGradient take_gradient(const AdamwEntry& t, long long from, unsigned int i, int left) {
    RawGradient r = {};
    if (t.g_bf16)
        r.b = take4<__bf16, ONCE, FULL>(static_cast<const __bf16*>(t.g) + from, i, left);
    else
        r.f = take4<float, ONCE, FULL>(static_cast<const float*>(t.g) + from, i, left);
    return r;
}
__device__ __forceinline__ f32x4 gradient_of(const AdamwEntry& t, const RawGradient& r, float scale) {
    return (t.g_bf16 ? widen(r.b) : r.f) * scale;
}

// ---- states in 32 bits -----------------------------------------------------------------------------------------------
template <bool ONCE, bool FULL>
__device__ __forceinline__ void adamw32_chunk(const AdamwEntry& t, long long from, float keep, const AdamwScalars& s) {
    const unsigned int i = threadIdx.x * 4;
    const int left = FULL || t.count - from - i >= 4 ? 4 : (int)(t.count - from - i);
    if (left <= 0) return;
    float *p = t.p + from, *m = static_cast<float*>(t.m) + from, *v = static_cast<float*>(t.v) + from;
    const RawGradient raw = take_gradient<ONCE, FULL>(t, from, i, left);
    f32x4 pp = take4<float, ONCE, FULL>(p, i, left), mm = take4<float, ONCE, FULL>(m, i, left), vv = take4<float, ONCE, FULL>(v, i, left);
    const f32x4 g = gradient_of(t, raw, s.grad_scale);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        mm[j] = moment1(mm[j], g[j], s);
        vv[j] = moment2(vv[j], g[j], s);
        pp[j] = new_parameter(pp[j], mm[j], vv[j], keep, s);
    }
    give4<float, ONCE, FULL>(p, i, left, pp);
    give4<float, ONCE, FULL>(m, i, left, mm);
    give4<float, ONCE, FULL>(v, i, left, vv);
    if (t.copy != nullptr) give4<__bf16, ONCE, FULL>(t.copy + from, i, left, pp);
}

template <bool ONCE>
__global__ void __launch_bounds__(256) adamw32_kernel(const AdamwEntry* __restrict__ entries, const int* __restrict__ owner,
                                                      long long chunks, AdamwScalars s) {
    const long long chunk = block_number();
    if (chunk >= chunks) return;
    const AdamwEntry t = entries[owner[chunk]];
    const long long from = (chunk - t.first_chunk) * kAdamwChunk;
    const float keep = 1.0f - s.rate * t.decay;
    if (from + kAdamwChunk <= t.count)
        adamw32_chunk<ONCE, true>(t, from, keep, s);
    else
        adamw32_chunk<ONCE, false>(t, from, keep, s);
}

// ---- states in 8 bits ------------------------------------------------------------------------------------------------
// |x| >= 0 (already divided by its block's power of two) rounded up or down by 16 random bits to MANTISSA bits after the point,
// below 2^LOWEST to a multiple of 2^(LOWEST - MANTISSA).  A normal number takes the random bits below its last kept one, a
// carry going into the exponent as it should; a smaller one does the same as a fixed-point number.
template <int MANTISSA, int LOWEST>
__device__ __forceinline__ float round_at_random(float a, unsigned int random, bool never_zero) {
    const unsigned int add = random << (7 - MANTISSA);
    const float normal = __uint_as_float((__float_as_uint(a) + add) & ~((1u << (23 - MANTISSA)) - 1u));
    unsigned int k = ((unsigned int)(a * __uint_as_float((unsigned int)(23 - LOWEST + 127) << 23)) + add) >> (23 - MANTISSA);
    if (never_zero && k == 0) k = 1;
    const float small = (float)k * __uint_as_float((unsigned int)(LOWEST - MANTISSA + 127) << 23);
    return a < __uint_as_float((unsigned int)(LOWEST + 127) << 23) ? small : normal;
}

// The scale byte of a block whose largest finite magnitude has the bits `top`.
__device__ __forceinline__ unsigned int scale_code(unsigned int top, int room) {
    const int e = (int)(top >> 23) - room;
    return e < 1 ? 1u : (unsigned int)e;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned int)(e + 127) << 23); }
// bits of |x|; 0 where it is not finite and that is asked for
__device__ __forceinline__ unsigned int magnitude(float x, bool finite_only) {
    const unsigned int b = __float_as_uint(x) & 0x7fffffffu;
    return finite_only && b >= 0x7f800000u ? 0u : b;
}
// the largest over the wavefront
template <int ROTATE>
__device__ __forceinline__ unsigned int max_rotated(unsigned int v) {
    const unsigned int o = (unsigned int)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + ROTATE, 0xf, 0xf, false);
    return v > o ? v : o;
}
__device__ __forceinline__ unsigned int wave64_max(unsigned int v) {
    v = max_rotated<1>(max_rotated<2>(max_rotated<4>(max_rotated<8>(v))));
    const unsigned int a = __builtin_amdgcn_readlane(v, 0), b = __builtin_amdgcn_readlane(v, 16);
    const unsigned int c = __builtin_amdgcn_readlane(v, 32), d = __builtin_amdgcn_readlane(v, 48);
    const unsigned int ab = a > b ? a : b, cd = c > d ? c : d;
    return ab > cd ? ab : cd;
}

// The new states of a block: its elements' moments in the lanes (zeros behind the tensor's end).
template <bool FULL>
__device__ __forceinline__ void store_states(const AdamwEntry& t, long long from, unsigned int i, int left, const f32x4& mm, const f32x4& vv,
                                             int tensor, const AdamwScalars& s) {
    unsigned int m_top = 0, v_top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned int a = magnitude(mm[j], false), b = magnitude(vv[j], false);
        m_top = a > m_top ? a : m_top, v_top = b > v_top ? b : v_top;
    }
    m_top = wave64_max(m_top), v_top = wave64_max(v_top);
    const bool broken = m_top >= 0x7f800000u || v_top >= 0x7f800000u;  // (of the wavefront)
    if (broken) {
        m_top = v_top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned int a = magnitude(mm[j], true), b = magnitude(vv[j], true);
            m_top = a > m_top ? a : m_top, v_top = b > v_top ? b : v_top;
        }
        m_top = wave64_max(m_top), v_top = wave64_max(v_top);
    }
    const unsigned int m_code = scale_code(m_top, 7), v_code = scale_code(v_top, 14);
    const float m_inv = power_of_two(127 - (int)m_code), v_inv = power_of_two(127 - (int)v_code);
    const unsigned long long quad = (unsigned long long)(from + i) >> 2;
    const Philox4 r = philox4x32_10((unsigned int)quad, (unsigned int)(quad >> 32), (unsigned int)tensor, s.step, s.key0, s.key1);
    f32x4 m_out, v_out;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a = fabsf(mm[j] * m_inv), b = vv[j] * v_inv;
        if (broken) a = a < __builtin_inff() ? a : 0.0f, b = b < __builtin_inff() ? b : 0.0f;
        m_out[j] = copysignf(round_at_random<3, -6>(a, r.v[j] & 0xffffu, false), mm[j]);
        v_out[j] = round_at_random<2, -14>(b, r.v[j] >> 16, vv[j] > 0.0f);  // (b may have underflowed)
    }
    // (the values are exact in their formats: the conversions round nothing)
    unsigned int m_word = 0, v_word = 0;
    m_word = __builtin_amdgcn_cvt_pk_fp8_f32(m_out[0], m_out[1], m_word, false);
    m_word = __builtin_amdgcn_cvt_pk_fp8_f32(m_out[2], m_out[3], m_word, true);
    v_word = __builtin_amdgcn_cvt_pk_bf8_f32(v_out[0], v_out[1], v_word, false);
    v_word = __builtin_amdgcn_cvt_pk_bf8_f32(v_out[2], v_out[3], v_word, true);
    if (broken) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {  // 0x7f: NaN in both formats
            if (magnitude(mm[j], false) >= 0x7f800000u) m_word = (m_word & ~(0xffu << (8 * j))) | 0x7fu << (8 * j);
            if (magnitude(vv[j], false) >= 0x7f800000u) v_word = (v_word & ~(0xffu << (8 * j))) | 0x7fu << (8 * j);
        }
    }
    give_bytes<FULL>(static_cast<unsigned char*>(t.m) + from, i, left, m_word);
    give_bytes<FULL>(static_cast<unsigned char*>(t.v) + from, i, left, v_word);
    const long long block = from / kAdamwBlock;
    if ((threadIdx.x & 63) == 0) t.m_scale[block] = (unsigned char)m_code, t.v_scale[block] = (unsigned char)v_code;
}

// A wavefront's block of 256 elements: the block's largest magnitudes meet by rotations, the moments go back to 8 bits in the
// registers they were computed in.
template <bool ONCE, bool FULL>
__device__ __forceinline__ void adamw8_block(const AdamwEntry& t, long long from, int tensor, float keep, const AdamwScalars& s) {
    const unsigned int i = (threadIdx.x & 63) * 4;
    const int left = FULL || t.count - from - i >= 4 ? 4 : (int)(t.count - from - i);  // <= 0: behind the tensor's end
    const long long block = from / kAdamwBlock;
    const RawGradient raw = take_gradient<ONCE, FULL>(t, from, i, left);
    f32x4 pp = take4<float, ONCE, FULL>(t.p + from, i, left), mm, vv;
    const unsigned int mbits = take_bytes<FULL>(static_cast<const unsigned char*>(t.m) + from, i, left);
    const unsigned int vbits = take_bytes<FULL>(static_cast<const unsigned char*>(t.v) + from, i, left);
    const float m_unit = power_of_two((int)t.m_scale[block] - 127), v_unit = power_of_two((int)t.v_scale[block] - 127);
    const f32x4 g = gradient_of(t, raw, s.grad_scale);
    mm[0] = __builtin_amdgcn_cvt_f32_fp8(mbits, 0), mm[1] = __builtin_amdgcn_cvt_f32_fp8(mbits, 1);
    mm[2] = __builtin_amdgcn_cvt_f32_fp8(mbits, 2), mm[3] = __builtin_amdgcn_cvt_f32_fp8(mbits, 3);
    vv[0] = __builtin_amdgcn_cvt_f32_bf8(vbits, 0), vv[1] = __builtin_amdgcn_cvt_f32_bf8(vbits, 1);
    vv[2] = __builtin_amdgcn_cvt_f32_bf8(vbits, 2), vv[3] = __builtin_amdgcn_cvt_f32_bf8(vbits, 3);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        mm[j] = moment1(mm[j] * m_unit, g[j], s);
        vv[j] = moment2(vv[j] * v_unit, g[j], s);
        pp[j] = new_parameter(pp[j], mm[j], vv[j], keep, s);
    }
    give4<float, ONCE, FULL>(t.p + from, i, left, pp);
    if (t.copy != nullptr) give4<__bf16, ONCE, FULL>(t.copy + from, i, left, pp);
    store_states<FULL>(t, from, i, left, mm, vv, tensor, s);
}

template <bool ONCE>
__global__ void __launch_bounds__(256) adamw8_kernel(const AdamwEntry* __restrict__ entries, const int* __restrict__ owner,
                                                     long long chunks, AdamwScalars s) {
    const long long chunk = block_number();
    if (chunk >= chunks) return;
    const int tensor = owner[chunk], w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const AdamwEntry t = entries[tensor];
    const long long from = (chunk - t.first_chunk) * kAdamwChunk + w * kAdamwBlock;
    const float keep = 1.0f - s.rate * t.decay;
    if (from + kAdamwBlock <= t.count)
        adamw8_block<ONCE, true>(t, from, tensor, keep, s);
    else if (from < t.count)
        adamw8_block<ONCE, false>(t, from, tensor, keep, s);
}

}  // namespace snhip
