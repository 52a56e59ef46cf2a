// Norms before and after a block with the block's gate and residual scale (definitions: include/sharpnet_hip.h,
// snhip_block_norm_desc).  One pass over the rows forward and backward, a row in the registers of TPR threads (N pieces of
// four columns each): every input is read once, every output written once, so both are bound by HBM.  Sums run in fp32:
// per thread, then over the row's threads; the variance is taken around the mean, from the registers.
#pragma once
#include <hip/hip_runtime.h>

#include "vec_types.hpp"

namespace snhip {

enum : int { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };
enum : int { GATE_NONE = 0, GATE_SIGMOID = 3, GATE_TANH = 4 };  // SNHIP_ACT_*

struct BlockNormParams {
    const void *x, *y, *gate;
    void *u, *h;
    const float *pre_w, *pre_b, *post_w, *post_b;
    float *pre_s, *post_s;
    const void *du, *dh;
    void *dx, *dy, *d_gate;
    long long rows, ld_x, ld_y, ld_u, ld_h, ld_gate;
    int dim, gate_rows, pre, post, act, whole;
    float eps, scale, inv_dim;
    // backward: a workgroup takes a chunk of rows
    float* partial;            // [vector][chunk][dim]: column sums of pre weight, pre bias, post weight, post bias, gate
    long long gate_groups;     // runs of rows with the same gate row (1 without a gate)
    long long rows_per_group;
    int flush;                 // 1: a chunk is `groups_per_chunk` whole groups; 0: one of `chunks_per_group` parts of a group
    int groups_per_chunk, chunks_per_group, rows_per_chunk, chunks;
    int slot[5];               // which vector of `partial` a column sum goes to, -1: not wanted
};

// Sum of A and B over the TPR threads of a row.  Up to a wavefront: by shuffles.  Beyond: the wavefronts' sums meet in LDS;
// `turn` alternates between two places, so that one barrier a sum is enough.
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float (*lds)[2][TPR / 64 + 1], int& turn) {
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) {
        a += __shfl_xor(a, off, 64);
        b += __shfl_xor(b, off, 64);
    }
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) lds[turn][0][w] = a, lds[turn][1][w] = b;
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) a += lds[turn][0][k], b += lds[turn][1][k];
        turn ^= 1;
    }
}
template <int TPR>
__device__ __forceinline__ float row_sum(float a, float (*lds)[2][TPR / 64 + 1], int& turn) {
    constexpr int W = TPR < 64 ? TPR : 64;
#pragma unroll
    for (int off = W / 2; off > 0; off >>= 1) a += __shfl_xor(a, off, 64);
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) lds[turn][0][w] = a;
        __syncthreads();
        a = 0.0f;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) a += lds[turn][0][k];
        turn ^= 1;
    }
    return a;
}

// Columns [c, c + 4) of a weight or bias vector; `missing` where there is no vector; 0 behind the row's end.
__device__ __forceinline__ f32x4 vector4(const float* v, int c, const BlockNormParams& p, float missing) {
    if (v != nullptr) return load4(v, c, p.dim, p.whole);
    f32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = c + j < p.dim ? missing : 0.0f;
    return r;
}

__device__ __forceinline__ float gate_value(float g, int act) {
    return act == GATE_SIGMOID ? 1.0f / (1.0f + expf(-g)) : act == GATE_TANH ? tanhf(g) : g;
}
__device__ __forceinline__ float gate_slope(float q, int act) {  // in terms of q = act(g)
    return act == GATE_SIGMOID ? q * (1.0f - q) : act == GATE_TANH ? 1.0f - q * q : 1.0f;
}
template <typename TB>
__device__ __forceinline__ f32x4 gate4(const BlockNormParams& p, long long row, int c) {
    if (p.gate_rows == 0) return load4(static_cast<const float*>(p.gate), c, p.dim, p.whole);
    return load4(static_cast<const TB*>(p.gate) + row / p.gate_rows * p.ld_gate, c, p.dim, p.whole);
}

// mean and 1 / deviation of the row in z
template <int TPR, int N>
__device__ __forceinline__ void row_statistics(const f32x4 (&z)[N], int lane, int kind, const BlockNormParams& p,
                                               float (*lds)[2][TPR / 64 + 1], int& turn, float& mean, float& rstd) {
    mean = 0.0f;
    if (kind == NORM_LAYER) {
        float s = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n) s += (z[n][0] + z[n][1]) + (z[n][2] + z[n][3]);
        mean = row_sum<TPR>(s, lds, turn) * p.inv_dim;
    }
    float s = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = 4 * (n * TPR + lane);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float d = z[n][j] - mean;
            if (c + j < p.dim) s += d * d;
        }
    }
    rstd = 1.0f / sqrtf(row_sum<TPR>(s, lds, turn) * p.inv_dim + p.eps);
}

template <typename TS, typename TB, int TPR, int N>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) block_norm_forward_kernel(const BlockNormParams p) {
    constexpr int NT = TPR > 256 ? TPR : 256, GROUPS = NT / TPR;
    __shared__ float lds[2][2][TPR / 64 + 1];
    int turn = 0;
    const int lane = threadIdx.x % TPR;
    const long long row = (long long)blockIdx.x * GROUPS + threadIdx.x / TPR;
    if (row >= p.rows) return;  // (with a barrier ahead a workgroup has one row)
    f32x4 u[N];
    const TS* x = static_cast<const TS*>(p.x) + row * p.ld_x;
    float mean, rstd;
    if (p.y != nullptr) {
        const TB* yr = static_cast<const TB*>(p.y) + row * p.ld_y;
        f32x4 y[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 4 * (n * TPR + lane);
            y[n] = u[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (c < p.dim) {
                y[n] = load4(yr, c, p.dim, p.whole);
                u[n] = load4(x, c, p.dim, p.whole);
            }
        }
        if (p.post != NORM_NONE) {
            row_statistics<TPR, N>(y, lane, p.post, p, lds, turn, mean, rstd);
            if (p.post_s != nullptr && lane == 0) p.post_s[2 * row] = mean, p.post_s[2 * row + 1] = rstd;
        }
        TS* ur = static_cast<TS*>(p.u) + row * p.ld_u;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 4 * (n * TPR + lane);
            if (c >= p.dim) continue;
            f32x4 v = y[n];
            if (p.post != NORM_NONE) v = (v - mean) * rstd * vector4(p.post_w, c, p, 1.0f) + vector4(p.post_b, c, p, 0.0f);
            if (p.gate != nullptr) {
                const f32x4 g = gate4<TB>(p, row, c);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] *= gate_value(g[j], p.act);
            }
            u[n] = as_stored(u[n] + p.scale * v, static_cast<const TS*>(nullptr));
            store4(ur, c, p.dim, p.whole, u[n]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j >= p.dim) u[n][j] = 0.0f;
        }
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = 4 * (n * TPR + lane);
            u[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (c < p.dim) u[n] = load4(x, c, p.dim, p.whole);
        }
    }
    if (p.pre == NORM_NONE) return;
    row_statistics<TPR, N>(u, lane, p.pre, p, lds, turn, mean, rstd);
    if (p.pre_s != nullptr && lane == 0) p.pre_s[2 * row] = mean, p.pre_s[2 * row + 1] = rstd;
    TB* hr = static_cast<TB*>(p.h) + row * p.ld_h;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = 4 * (n * TPR + lane);
        if (c < p.dim)
            store4(hr, c, p.dim, p.whole, (u[n] - mean) * rstd * vector4(p.pre_w, c, p, 1.0f) + vector4(p.pre_b, c, p, 0.0f));
    }
}

// dz = dN(z) * dn for the row in registers: in: hat = z normed, a = dn * weight; out: a becomes dz
template <int TPR, int N>
__device__ __forceinline__ void row_gradient(f32x4 (&a)[N], const f32x4 (&hat)[N], int kind, float rstd, const BlockNormParams& p,
                                             float (*lds)[2][TPR / 64 + 1], int& turn) {
    float s = 0.0f, m = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s += a[n][j] * hat[n][j], m += a[n][j];
    if (kind == NORM_LAYER) {
        row_sums<TPR>(s, m, lds, turn);
        m *= p.inv_dim;
    } else {
        s = row_sum<TPR>(s, lds, turn);
        m = 0.0f;
    }
    s *= p.inv_dim;
#pragma unroll
    for (int n = 0; n < N; ++n) a[n] = rstd * (a[n] - m - s * hat[n]);
}

// MODE 0: no block (the pre norm alone), 1: a block without a norm behind it, 2: with one.  BIAS / GATE: column sums for
// biases / a gate are kept.  A workgroup walks a chunk of rows and keeps the column sums of its columns in registers; at the
// end it writes them to `partial`, and column_parts_kernel adds the chunks in order.
template <typename TS, typename TB, int TPR, int N, int MODE, bool BIAS, bool GATE>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) block_norm_backward_kernel(const BlockNormParams p) {
    constexpr int NT = TPR > 256 ? TPR : 256, GROUPS = NT / TPR;
    __shared__ float lds[2][2][TPR / 64 + 1];
    __shared__ float meet[GROUPS > 1 ? GROUPS * TPR * N * 4 : 1];
    int turn = 0;
    const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
    constexpr f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 acc_w[N], acc_b[BIAS ? N : 1], acc_pw[MODE == 2 ? N : 1], acc_pb[MODE == 2 && BIAS ? N : 1], acc_g[GATE ? N : 1];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        acc_w[n] = zero;
        if constexpr (BIAS) acc_b[n] = zero;
        if constexpr (MODE == 2) acc_pw[n] = zero;
        if constexpr (MODE == 2 && BIAS) acc_pb[n] = zero;
        if constexpr (GATE) acc_g[n] = zero;
    }
    // segments of rows: with `flush` the gate groups of this chunk that this group of threads takes, else one
    const long long chunk = blockIdx.x;
    long long seg = chunk, seg_end = chunk + 1, seg_step = 1;
    if (p.flush) {
        seg = chunk * p.groups_per_chunk;
        seg_end = seg + p.groups_per_chunk < p.gate_groups ? seg + p.groups_per_chunk : p.gate_groups;
        seg += group, seg_step = GROUPS;
    }
    for (; seg < seg_end; seg += seg_step) {
        long long r, r_end, r_step;
        if (p.flush) {
            r = seg * p.rows_per_group, r_step = 1;
            r_end = r + p.rows_per_group < p.rows ? r + p.rows_per_group : p.rows;
        } else {
            const long long g = chunk / p.chunks_per_group, part = chunk % p.chunks_per_group;
            const long long g_end = (g + 1) * p.rows_per_group < p.rows ? (g + 1) * p.rows_per_group : p.rows;
            r = g * p.rows_per_group + part * p.rows_per_chunk;
            r_end = r + p.rows_per_chunk < g_end ? r + p.rows_per_chunk : g_end;
            r += group, r_step = GROUPS;
        }
        for (; r < r_end; r += r_step) {
            f32x4 t[N], hat[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = 4 * (n * TPR + lane);
                t[n] = zero;
                if (p.du != nullptr && c < p.dim) t[n] = load4(static_cast<const TS*>(p.du) + r * p.ld_u, c, p.dim, p.whole);
            }
            if (p.dh != nullptr) {
                f32x4 a[N];
                const float mean = p.pre_s[2 * r], rstd = p.pre_s[2 * r + 1];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int c = 4 * (n * TPR + lane);
                    a[n] = hat[n] = zero;
                    if (c < p.dim) {
                        const f32x4 dh = load4(static_cast<const TB*>(p.dh) + r * p.ld_h, c, p.dim, p.whole);
                        hat[n] = (load4(static_cast<const TS*>(p.u) + r * p.ld_u, c, p.dim, p.whole) - mean) * rstd;
                        acc_w[n] += dh * hat[n];
                        if constexpr (BIAS) acc_b[n] += dh;
                        a[n] = dh * vector4(p.pre_w, c, p, 1.0f);
                    }
                }
                row_gradient<TPR, N>(a, hat, p.pre, rstd, p, lds, turn);
#pragma unroll
                for (int n = 0; n < N; ++n) t[n] += a[n];
            }
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = 4 * (n * TPR + lane);
                if (c < p.dim) store4(static_cast<TS*>(p.dx) + r * p.ld_x, c, p.dim, p.whole, t[n]);
            }
            if constexpr (MODE > 0) {
                float mean = 0.0f, rstd = 1.0f;
                if constexpr (MODE == 2) mean = p.post_s[2 * r], rstd = p.post_s[2 * r + 1];
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int c = 4 * (n * TPR + lane);
                    t[n] *= p.scale;
                    if (c >= p.dim) {
                        t[n] = hat[n] = zero;
                        continue;
                    }
                    if constexpr (MODE == 2 || GATE) {
                        const f32x4 y = load4(static_cast<const TB*>(p.y) + r * p.ld_y, c, p.dim, p.whole);
                        hat[n] = MODE == 2 ? (y - mean) * rstd : y;
                    }
                    f32x4 w;
                    if constexpr (MODE == 2) w = vector4(p.post_w, c, p, 1.0f);
                    if constexpr (GATE) {
                        const f32x4 g = gate4<TB>(p, r, c);
                        f32x4 v = hat[n];
                        if constexpr (MODE == 2) v = v * w + vector4(p.post_b, c, p, 0.0f);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float q = gate_value(g[j], p.act);
                            acc_g[n][j] += t[n][j] * v[j] * gate_slope(q, p.act);
                            t[n][j] *= q;
                        }
                    }
                    if constexpr (MODE == 2) {
                        acc_pw[n] += t[n] * hat[n];
                        if constexpr (BIAS) acc_pb[n] += t[n];
                        t[n] *= w;
                    }
                }
                if constexpr (MODE == 2) row_gradient<TPR, N>(t, hat, p.post, rstd, p, lds, turn);
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int c = 4 * (n * TPR + lane);
                    if (c < p.dim) store4(static_cast<TB*>(p.dy) + r * p.ld_y, c, p.dim, p.whole, t[n]);
                }
            }
        }
        if constexpr (GATE) {
            if (p.flush) {  // the whole group's rows are in
                if (p.d_gate != nullptr) {
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const int c = 4 * (n * TPR + lane);
                        if (c < p.dim) store4(static_cast<TB*>(p.d_gate) + seg * p.ld_gate, c, p.dim, p.whole, acc_g[n]);
                    }
                }
#pragma unroll
                for (int n = 0; n < N; ++n) acc_g[n] = zero;
            }
        }
    }
    // the column sums of the chunk; groups of threads that share the columns meet in LDS
    auto put = [&](const f32x4* acc, int slot) {
        if (slot < 0) return;  // the same for the whole launch
        float* out = p.partial + ((long long)slot * p.chunks + chunk) * p.dim;
        const bool whole = (p.dim & 3) == 0;
        if constexpr (GROUPS > 1) {
            __syncthreads();
#pragma unroll
            for (int n = 0; n < N; ++n) *reinterpret_cast<f32x4*>(&meet[(group * TPR * N + n * TPR + lane) * 4]) = acc[n];
            __syncthreads();
            for (int k = threadIdx.x; k < TPR * N; k += NT) {
                f32x4 s = *reinterpret_cast<f32x4*>(&meet[k * 4]);
                for (int g = 1; g < GROUPS; ++g) s += *reinterpret_cast<f32x4*>(&meet[(g * TPR * N + k) * 4]);
                if (4 * k < p.dim) store4(out, 4 * k, p.dim, whole, s);
            }
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = 4 * (n * TPR + lane);
                if (c < p.dim) store4(out, c, p.dim, whole, acc[n]);
            }
        }
    };
    put(acc_w, p.slot[0]);
    if constexpr (BIAS) put(acc_b, p.slot[1]);
    if constexpr (MODE == 2) put(acc_pw, p.slot[2]);
    if constexpr (MODE == 2 && BIAS) put(acc_pb, p.slot[3]);
    if constexpr (GATE) put(acc_g, p.slot[4]);
}

}  // namespace snhip
