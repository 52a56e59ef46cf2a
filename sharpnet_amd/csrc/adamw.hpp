// AdamW over the elements of many tensors in one launch (definitions: include/sharpnet_hip.h, snhip_adamw_create).
// Bound by HBM: 28 bytes an element with states in 32 bits, 16 with states in 8 (and an fp32 gradient), each read and
// written once.  ONCE: around the caches, for plans that are larger than they are (kAdamwOnce).
#pragma once
#include <hip/hip_runtime.h>

#include "philox.hpp"
#include "vec_types.hpp"

namespace snhip {

typedef unsigned int u32_any __attribute__((aligned(1)));  // four bytes at any address

constexpr int kAdamwBlock = 256;   // elements that share a power of two (states in 8 bits)
constexpr int kAdamwChunk = 4096;  // elements of a tensor that a workgroup of 256 threads updates

// Elements from which on a plan's data does not go through the caches: a step on 4 million (112 MB of fp32 states) finds some
// of it in the 256 MB behind the L2s again, a step on more than they hold does not and runs at 5.3 instead of 5.15 TB/s.
constexpr long long kAdamwOnce = 1LL << 23;

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
// (the hardware's reciprocal, 1 ulp: the denominator is 0 or between 1e-23 and 1e20, where it is exact to that)
__device__ __forceinline__ float new_parameter(float p, float m, float v, float keep, const AdamwScalars& s) {
    return p * keep - s.step_size * (m * __builtin_amdgcn_rcpf(sqrtf(v) * s.root_scale + s.eps));
}

// Four elements of the gradient as they lie in memory, and what they are worth: the conversion is kept away from the load,
// so that the other loads of the same elements do not wait for it.
struct RawGradient {
    f32x4 f;
    bf16x4 b;
};
template <bool ONCE>
__device__ __forceinline__ RawGradient load_gradient(const AdamwEntry& t, long long i, int left) {
    RawGradient r;
    if (t.g_bf16)
        r.b = load4<__bf16, ONCE>(static_cast<const __bf16*>(t.g) + i, left);
    else
        r.f = load4<float, ONCE>(static_cast<const float*>(t.g) + i, left);
    return r;
}
__device__ __forceinline__ f32x4 gradient_of(const AdamwEntry& t, const RawGradient& r, float scale) {
    return (t.g_bf16 ? widen(r.b) : r.f) * scale;
}

template <bool ONCE>
__global__ void __launch_bounds__(256) adamw32_kernel(const AdamwEntry* __restrict__ entries, const int* __restrict__ owner,
                                                      AdamwScalars s) {
    const AdamwEntry t = entries[owner[blockIdx.x]];
    const long long base = (blockIdx.x - t.first_chunk) * kAdamwChunk;
    const float keep = 1.0f - s.rate * t.decay;
    float *m = static_cast<float*>(t.m), *v = static_cast<float*>(t.v);
#pragma unroll
    for (int k = 0; k < kAdamwChunk / 1024; ++k) {
        const long long i = base + k * 1024 + threadIdx.x * 4;
        if (i >= t.count) break;
        const int left = t.count - i < 4 ? (int)(t.count - i) : 4;
        const RawGradient raw = load_gradient<ONCE>(t, i, left);
        f32x4 pp = load4<float, ONCE>(t.p + i, left), mm = load4<float, ONCE>(m + i, left), vv = load4<float, ONCE>(v + i, left);
        const f32x4 g = gradient_of(t, raw, s.grad_scale);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mm[j] = moment1(mm[j], g[j], s);
            vv[j] = moment2(vv[j], g[j], s);
            pp[j] = new_parameter(pp[j], mm[j], vv[j], keep, s);
        }
        store4<float, ONCE>(t.p + i, left, pp);
        store4<float, ONCE>(m + i, left, mm);
        store4<float, ONCE>(v + i, left, vv);
        if (t.copy != nullptr) store4<__bf16, ONCE>(t.copy + i, left, pp);
    }
}

// ---- states in 8 bits ------------------------------------------------------------------------------------------
// |x| (already divided by its block's power of two) as k steps of its binade, k rounded up where the 16 random bits ask
// for it: MANTISSA bits after the point, binades from 2^LOWEST on (below it the step stays, as in the format).
template <int MANTISSA, int LOWEST>
__device__ __forceinline__ float round_at_random(float x, unsigned int random, bool never_zero) {
    const float a = fabsf(x);
    int e = (int)(__float_as_uint(a) >> 23) - 127;
    if (e < LOWEST) e = LOWEST;
    // a / 2^(e - 23): a whole number for a normal number of the format, cut to one below
    const unsigned int whole = (unsigned int)(a * __uint_as_float((unsigned int)(23 - e + 127) << 23));
    unsigned int k = (whole + (random << (7 - MANTISSA))) >> (23 - MANTISSA);
    if (never_zero && k == 0 && a > 0.0f) k = 1;
    return copysignf((float)k * __uint_as_float((unsigned int)(e - MANTISSA + 127) << 23), x);
}

// The scale byte of a block whose largest finite magnitude has the bits `top`.
__device__ __forceinline__ unsigned int scale_code(unsigned int top, int room) {
    const int e = (int)(top >> 23) - room;
    return e < 1 ? 1u : (unsigned int)e;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned int)(e + 127) << 23); }
// bits of |x|, 0 where it is not finite
__device__ __forceinline__ unsigned int magnitude(float x) {
    const unsigned int b = __float_as_uint(x) & 0x7fffffffu;
    return b < 0x7f800000u ? b : 0u;
}

// A wavefront takes blocks of 256 elements, four to a lane: the block's largest magnitudes meet by shuffles, the moments
// go back to 8 bits in the registers they were computed in.
template <bool ONCE>
__global__ void __launch_bounds__(256) adamw8_kernel(const AdamwEntry* __restrict__ entries, const int* __restrict__ owner,
                                                     AdamwScalars s) {
    const int tensor = owner[blockIdx.x];
    const AdamwEntry t = entries[tensor];
    const long long base = (blockIdx.x - t.first_chunk) * kAdamwChunk;
    const float keep = 1.0f - s.rate * t.decay;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    unsigned char *m8 = static_cast<unsigned char*>(t.m), *v8 = static_cast<unsigned char*>(t.v);
#pragma unroll
    for (int k = 0; k < kAdamwChunk / 1024; ++k) {
        const long long b0 = base + (4 * k + w) * kAdamwBlock;  // the wavefront's block
        if (b0 >= t.count) break;
        const long long i = b0 + lane * 4;
        const int left = t.count - i < 4 ? (int)(t.count - i) : 4;  // <= 0: behind the tensor's end
        unsigned int mbits = 0, vbits = 0;
        RawGradient raw = {};
        f32x4 pp = {0.0f, 0.0f, 0.0f, 0.0f}, mm, vv;
        if (left > 0) {
            raw = load_gradient<ONCE>(t, i, left);
            pp = load4<float, ONCE>(t.p + i, left);
            if (left == 4) {
                mbits = *reinterpret_cast<const u32_any*>(m8 + i);
                vbits = *reinterpret_cast<const u32_any*>(v8 + i);
            } else {
                for (int j = 0; j < left; ++j) {
                    mbits |= (unsigned int)m8[i + j] << (8 * j);
                    vbits |= (unsigned int)v8[i + j] << (8 * j);
                }
            }
        }
        const f32x4 g = gradient_of(t, raw, s.grad_scale);
        const long long block = b0 / kAdamwBlock;
        const float m_unit = power_of_two((int)t.m_scale[block] - 127), v_unit = power_of_two((int)t.v_scale[block] - 127);
        mm[0] = __builtin_amdgcn_cvt_f32_fp8(mbits, 0), mm[1] = __builtin_amdgcn_cvt_f32_fp8(mbits, 1);
        mm[2] = __builtin_amdgcn_cvt_f32_fp8(mbits, 2), mm[3] = __builtin_amdgcn_cvt_f32_fp8(mbits, 3);
        vv[0] = __builtin_amdgcn_cvt_f32_bf8(vbits, 0), vv[1] = __builtin_amdgcn_cvt_f32_bf8(vbits, 1);
        vv[2] = __builtin_amdgcn_cvt_f32_bf8(vbits, 2), vv[3] = __builtin_amdgcn_cvt_f32_bf8(vbits, 3);
        unsigned int m_top = 0, v_top = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mm[j] = moment1(mm[j] * m_unit, g[j], s);
            vv[j] = moment2(vv[j] * v_unit, g[j], s);
            pp[j] = new_parameter(pp[j], mm[j], vv[j], keep, s);
            const unsigned int a = magnitude(mm[j]), b = magnitude(vv[j]);
            m_top = a > m_top ? a : m_top;
            v_top = b > v_top ? b : v_top;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) {
            const unsigned int a = (unsigned int)__shfl_xor((int)m_top, off, 64), b = (unsigned int)__shfl_xor((int)v_top, off, 64);
            m_top = a > m_top ? a : m_top;
            v_top = b > v_top ? b : v_top;
        }
        const unsigned int m_code = scale_code(m_top, 7), v_code = scale_code(v_top, 14);
        const float m_inv = power_of_two(127 - (int)m_code), v_inv = power_of_two(127 - (int)v_code);
        const Philox4 r = philox4x32_10((unsigned int)(i >> 2), (unsigned int)(i >> 34), (unsigned int)tensor, s.step, s.key0, s.key1);
        unsigned int m_bytes[4], v_bytes[4];
        float m_out[4], v_out[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool m_ok = fabsf(mm[j]) < __builtin_inff(), v_ok = fabsf(vv[j]) < __builtin_inff();
            m_out[j] = round_at_random<3, -6>(m_ok ? mm[j] * m_inv : 0.0f, r.v[j] & 0xffffu, false);
            v_out[j] = round_at_random<2, -14>(v_ok ? vv[j] * v_inv : 0.0f, r.v[j] >> 16, true);
        }
        // (the values are exact in their formats: the conversions round nothing)
        unsigned int m_word = 0, v_word = 0;
        m_word = __builtin_amdgcn_cvt_pk_fp8_f32(m_out[0], m_out[1], m_word, false);
        m_word = __builtin_amdgcn_cvt_pk_fp8_f32(m_out[2], m_out[3], m_word, true);
        v_word = __builtin_amdgcn_cvt_pk_bf8_f32(v_out[0], v_out[1], v_word, false);
        v_word = __builtin_amdgcn_cvt_pk_bf8_f32(v_out[2], v_out[3], v_word, true);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m_bytes[j] = (m_word >> (8 * j)) & 0xffu, v_bytes[j] = (v_word >> (8 * j)) & 0xffu;
            if (!(fabsf(mm[j]) < __builtin_inff())) m_bytes[j] = 0x7fu;  // NaN in both formats
            if (!(fabsf(vv[j]) < __builtin_inff())) v_bytes[j] = 0x7fu;
        }
        if (left > 0) {
            store4<float, ONCE>(t.p + i, left, pp);
            if (t.copy != nullptr) store4<__bf16, ONCE>(t.copy + i, left, pp);
            if (left == 4) {
                *reinterpret_cast<u32_any*>(m8 + i) = m_bytes[0] | m_bytes[1] << 8 | m_bytes[2] << 16 | m_bytes[3] << 24;
                *reinterpret_cast<u32_any*>(v8 + i) = v_bytes[0] | v_bytes[1] << 8 | v_bytes[2] << 16 | v_bytes[3] << 24;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < left) m8[i + j] = (unsigned char)m_bytes[j], v8[i + j] = (unsigned char)v_bytes[j];
            }
        }
        if (lane == 0) t.m_scale[block] = (unsigned char)m_code, t.v_scale[block] = (unsigned char)v_code;
    }
}

}  // namespace snhip
