// Norms before and after a block with the block's gate and residual scale (definitions: include/sharpnet_hip.h,
// snhip_block_norm_desc).  One pass over the rows forward and backward, a row in the registers of TPR threads (N pieces of
// four columns each): every input is read once, every output written once, so both are bound by HBM.  Sums run in fp32:
// per thread, then over the row's threads; the variance is taken around the mean, from the registers.
// 16384 rows of 2048 (fp32 stream, bf16 block, both norms, gate in rows, 403 MB): 84 us, 4.8 TB/s.  Backward, 16384 rows of
// 4096 (1.48 GB): 304 to 307 us with the column sums, 4.8 TB/s.  8 rows of 4096: 4.1 us, which is two times the way to memory.
// What the backward pass spends beside memory on rows of bf16, a gate and two norms: 12000 x 1280, 53 us, vector units at work in 71 %
// of the busy cycles (80 operations an element), 6 of the 16 loads of a row's wavefront weights and gate once more.
// EXACT: dim is a multiple of four and rows start on 4-byte addresses, so that a piece is a row's or not at all.
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
    int dim, gate_rows, pre, post, act;
    int exact;                 // which instantiations serve it (EXACT)
    float eps, scale, inv_dim;
    // backward: a workgroup takes a chunk of rows
    float* partial;            // [vector][chunk][dim]: column sums of pre weight, pre bias, post weight, post bias, gate
    long long rows_per_group;  // rows with the same gate row (all without a gate)
    int flush;                 // 1: a chunk is `groups_per_chunk` whole groups; 0: one of `chunks_per_group` parts of a group
    int groups_per_chunk, chunks_per_group, rows_per_chunk, chunks;
    int slot[5];               // which vector of `partial` a column sum goes to, -1: not wanted
};

// ---- pieces of a row -----------------------------------------------------------------------------------------------
// Exact rows are read and written as buffers of their own length: the base is scalar, the place in the row a 32-bit offset
// (64-bit addresses for every piece of every tensor took a third of the vector registers), what is read behind the row's end is
// zero and what is written there is dropped, without a branch.  Other rows (a buffer counts in 32-bit elements), and 16 or 32
// threads to a row, which share a wavefront with rows of other bases: plain accesses, wide at any address, the end of the row checked
// (16384 x 1001: backward 110 us against 100 us for 1000 columns).
typedef unsigned int u32x2 __attribute__((vector_size(8)));
typedef unsigned int u32x4 __attribute__((vector_size(16)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_buffer(const void* row, int bytes) {
    // raw buffer of 32-bit elements
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(row), 0, bytes, 0x00027000);
}

template <int TPR, bool EXACT>
struct Piece {
    template <typename T>
    static constexpr bool BUFFER = TPR >= 64 && (EXACT || sizeof(T) == 4);
    __device__ __forceinline__ static int column(int n, int lane) { return 4 * (n * TPR + lane); }
    template <typename T>
    __device__ __forceinline__ static raw4<T> load(const T* row, int n, int lane, int dim) {
        const int c = column(n, lane);
        if constexpr (BUFFER<T>) {
            const __amdgpu_buffer_rsrc_t b = row_buffer(row, dim * (int)sizeof(T));
            if constexpr (!EXACT)  // (a row of such a kernel has over 64 elements) as load4_row
                return __builtin_bit_cast(raw4<T>, __builtin_amdgcn_raw_buffer_load_b128(b, 4 * (c < dim - 4 ? c : dim - 4), 0, 0));
            else if constexpr (sizeof(T) == 4)
                return __builtin_bit_cast(raw4<T>, __builtin_amdgcn_raw_buffer_load_b128(b, 4 * c, 0, 0));
            else
                return __builtin_bit_cast(raw4<T>, __builtin_amdgcn_raw_buffer_load_b64(b, 2 * c, 0, 0));
        } else if constexpr (EXACT) {
            return load4_whole(row + (c < dim ? c : dim - 4));
        } else {
            return load4_row(row, c, dim);
        }
    }
    template <typename T>
    __device__ __forceinline__ static void store(T* row, int n, int lane, int dim, f32x4 v) {
        const int c = column(n, lane);
        if constexpr (BUFFER<T>) {
            const __amdgpu_buffer_rsrc_t b = row_buffer(row, dim * (int)sizeof(T));
            const raw4<T> r = narrow(v, static_cast<const T*>(nullptr));
            if constexpr (!EXACT) {
                if (c + 4 <= dim) {
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), b, 4 * c, 0, 0);
                } else {
#pragma unroll
                    for (int j = 0; j < 3; ++j)  // (dropped behind the row's end)
                        __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned int, (float)v[j]), b, 4 * (c + j), 0, 0);
                }
            } else if constexpr (sizeof(T) == 4)
                __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, r), b, 4 * c, 0, 0);
            else
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, r), b, 2 * c, 0, 0);
        } else {
            store4(row + c, dim - c, v);
        }
    }
    // what a loaded piece is worth: zeros behind the row's end
    template <typename R>
    __device__ __forceinline__ static f32x4 value(R raw, int n, int lane, int dim) {
        if constexpr (EXACT && TPR >= 64)
            return widen(raw);
        else if constexpr (EXACT)
            return cut(widen(raw), n, lane, dim);
        else
            return existing(widen(raw), dim - column(n, lane), __ballot(dim - column(n, lane) < 4) != 0);
    }
    // zeros behind the row's end, where a computation has left something else
    __device__ __forceinline__ static f32x4 cut(f32x4 v, int n, int lane, int dim) {
        const int c = column(n, lane);
        if constexpr (EXACT) {
            if (c >= dim) v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (c + j >= dim) v[j] = 0.0f;
        }
        return v;
    }
    // of a weight or bias vector; `missing` where there is none
    __device__ __forceinline__ static f32x4 vector(const float* v, int n, int lane, int dim, float missing) {
        if (v == nullptr) return f32x4{missing, missing, missing, missing};
        return value(load(v, n, lane, dim), n, lane, dim);
    }
};

// ---- sums over a row -----------------------------------------------------------------------------------------------
// Over the TPR threads of a row, TPR = 16, 32 or a multiple of 64.  Beyond a wavefront the wavefronts' sums meet in LDS; `turn`
// alternates between two places, so that one barrier a sum is enough.
template <int TPR>
__device__ __forceinline__ float lanes_sum(float a) {
    if constexpr (TPR == 16)
        return row16_sum(a);
    else if constexpr (TPR == 32)
        return half32_sum(a);
    else
        return wave64_sum(a);
}
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float (*lds)[2][TPR / 64 + 1], int& turn) {
    a = lanes_sum<TPR>(a), b = lanes_sum<TPR>(b);
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
    a = lanes_sum<TPR>(a);
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

// ---- gate ------------------------------------------------------------------------------------------------------------
// The sigmoid from the hardware's exponential and reciprocal (1 ulp each; the exponent's rounding adds |g| 2^-24).
// tanh x = (1 - e) / (1 + e) with e = exp(-2 |x|) from |x| = 1/4 on, where the difference keeps its digits (4 ulp), and its
// Taylor series to x^9 below (the next term is under 2^-26 of x).
// (r = 1 / (1 + e))
__device__ __forceinline__ float tanh_from(float x, float e, float r) {
    const float z = x * x, large = copysignf((1.0f - e) * r, x);
    const float series = ((((62.0f / 2835.0f * z - 17.0f / 315.0f) * z + 2.0f / 15.0f) * z - 1.0f / 3.0f) * z) * x + x;
    return fabsf(x) < 0.25f ? series : large;
}
__device__ __forceinline__ f32x4 gate_values(f32x4 g, int act) {
    if (act == GATE_SIGMOID) {
#pragma unroll
        for (int j = 0; j < 4; ++j) g[j] = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g[j] * -1.44269504088896341f));
    } else if (act == GATE_TANH) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float e = __builtin_amdgcn_exp2f(fabsf(g[j]) * -2.88539008177792681f);
            g[j] = tanh_from(g[j], e, __builtin_amdgcn_rcpf(1.0f + e));
        }
    }
    return g;
}
// Backward through v * act(g): t becomes t * act(g), sum gets t * v * act'(g).  The slopes are q (1 - q) with 1 - q = e q, e = exp(-g),
// and 4 e / (1 + e)^2 with e = exp(-2 |g|): q - q q and 1 - q q of the rounded q lose the digits of a gate near its limit (a
// sigmoid's slope off by 6 % at g = 16 and zero from 18 on).
// IN_BRANCH: all of it within the activation's branch, where no slopes are kept, for the kernels of long rows, which have no
// register left (575 x 6240, fp32 stream, bf16 block, two norms with biases: 31 us, 45 us the other way); the others wait for v
// later without it (33520 x 1001 bf16, a gate vector: 154 us, 168 us).
template <bool IN_BRANCH>
__device__ __forceinline__ void gate_gradient(f32x4& t, f32x4& sum, f32x4 v, f32x4 g, int act) {
    f32x4 slope = {1.0f, 1.0f, 1.0f, 1.0f};
    auto put = [&](int j, float q, float s) {
        if constexpr (IN_BRANCH)
            sum[j] += t[j] * v[j] * s, t[j] *= q;
        else
            g[j] = q, slope[j] = s;
    };
    if (act == GATE_SIGMOID) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float e = __builtin_amdgcn_exp2f(g[j] * -1.44269504088896341f), q = __builtin_amdgcn_rcpf(1.0f + e);
            put(j, q, fminf(e, 0x1p+126f) * q * q);  // (beyond that q is zero)
        }
    } else if (act == GATE_TANH) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float e = __builtin_amdgcn_exp2f(fabsf(g[j]) * -2.88539008177792681f), r = __builtin_amdgcn_rcpf(1.0f + e);
            put(j, tanh_from(g[j], e, r), 4.0f * e * r * r);
        }
    } else if constexpr (IN_BRANCH) {
        sum += t * v, t *= g;
    }
    if constexpr (!IN_BRANCH) sum += t * v * slope, t *= g;
}

// which row of the workgroup's rows this thread works on: the same for a wavefront where a row takes one or more
template <int TPR>
__device__ __forceinline__ int row_group() {
    const int g = (int)threadIdx.x / TPR;
    if constexpr (TPR >= 64)
        return __builtin_amdgcn_readfirstlane(g);
    else
        return g;
}

// mean and 1 / deviation of the row in z (zeros behind its end)
template <bool EXACT, int TPR, int N>
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
        const f32x4 d = Piece<TPR, EXACT>::cut(z[n] - mean, n, lane, p.dim);
        s += (d[0] * d[0] + d[1] * d[1]) + (d[2] * d[2] + d[3] * d[3]);
    }
    // (the hardware's reciprocal root takes numbers below the normal ones for zeros: a small one goes in times 2^96)
    const float variance = row_sum<TPR>(s, lds, turn) * p.inv_dim + p.eps;
    const bool tiny = variance < 0x1p-96f;
    rstd = __builtin_amdgcn_rsqf(tiny ? variance * 0x1p+96f : variance) * (tiny ? 0x1p+48f : 1.0f);
}

template <typename TS, typename TB, int TPR, int N, bool EXACT>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) block_norm_forward_kernel(const BlockNormParams p) {
    constexpr int NT = TPR > 256 ? TPR : 256, GROUPS = NT / TPR;
    typedef Piece<TPR, EXACT> P;
    __shared__ float lds[2][2][TPR / 64 + 1];
    int turn = 0;
    const int lane = threadIdx.x % TPR, dim = p.dim;
    const long long row = block_number() * GROUPS + row_group<TPR>();
    if (row >= p.rows) return;  // (with a barrier ahead a workgroup has one row)
    f32x4 u[N];
    raw4<TS> x[N];
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = P::load(static_cast<const TS*>(p.x) + row * p.ld_x, n, lane, dim);
    float mean, rstd;
    if (p.y != nullptr) {
        raw4<TB> y_raw[N], g_raw[N];
        const bool gate_in_rows = p.gate != nullptr && p.gate_rows != 0;
#pragma unroll
        for (int n = 0; n < N; ++n) y_raw[n] = P::load(static_cast<const TB*>(p.y) + row * p.ld_y, n, lane, dim);
        if (gate_in_rows) {
            const TB* gate = static_cast<const TB*>(p.gate) + (long long)((unsigned int)row / (unsigned int)p.gate_rows) * p.ld_gate;
#pragma unroll
            for (int n = 0; n < N; ++n) g_raw[n] = P::load(gate, n, lane, dim);
        }
        f32x4 y[N];
#pragma unroll
        for (int n = 0; n < N; ++n) y[n] = P::value(y_raw[n], n, lane, dim);
        if (p.post != NORM_NONE) {
            row_statistics<EXACT, TPR, N>(y, lane, p.post, p, lds, turn, mean, rstd);
            if (p.post_s != nullptr && lane == 0) p.post_s[2 * row] = mean, p.post_s[2 * row + 1] = rstd;
#pragma unroll
            for (int n = 0; n < N; ++n)
                y[n] = (y[n] - mean) * rstd * P::vector(p.post_w, n, lane, dim, 1.0f) + P::vector(p.post_b, n, lane, dim, 0.0f);
        }
        if (p.gate != nullptr) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                f32x4 g;
                if (gate_in_rows)
                    g = P::value(g_raw[n], n, lane, dim);
                else
                    g = P::vector(static_cast<const float*>(p.gate), n, lane, dim, 1.0f);
                y[n] *= gate_values(g, p.act);
            }
        }
        TS* ur = static_cast<TS*>(p.u) + row * p.ld_u;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            u[n] = as_stored<TS>(P::value(x[n], n, lane, dim) + p.scale * y[n]);
            P::store(ur, n, lane, dim, u[n]);
            u[n] = P::cut(u[n], n, lane, dim);
        }
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n) u[n] = P::value(x[n], n, lane, dim);
    }
    if (p.pre == NORM_NONE) return;
    row_statistics<EXACT, TPR, N>(u, lane, p.pre, p, lds, turn, mean, rstd);
    if (p.pre_s != nullptr && lane == 0) p.pre_s[2 * row] = mean, p.pre_s[2 * row + 1] = rstd;
    TB* hr = static_cast<TB*>(p.h) + row * p.ld_h;
#pragma unroll
    for (int n = 0; n < N; ++n)
        P::store(hr, n, lane, dim, (u[n] - mean) * rstd * P::vector(p.pre_w, n, lane, dim, 1.0f) + P::vector(p.pre_b, n, lane, dim, 0.0f));
}

// dz = dN(z) * dn for the row in registers: in: hat = z normed, a = dn * weight (zeros behind the row's end); out: a becomes dz
template <int TPR, int N>
__device__ __forceinline__ void row_gradient(f32x4 (&a)[N], const f32x4 (&hat)[N], int kind, float rstd, const BlockNormParams& p,
                                             float (*lds)[2][TPR / 64 + 1], int& turn) {
    float s = 0.0f, m = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const f32x4 q = a[n] * hat[n];
        s += (q[0] + q[1]) + (q[2] + q[3]);
        m += (a[n][0] + a[n][1]) + (a[n][2] + a[n][3]);
    }
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
template <typename TS, typename TB, int TPR, int N, int MODE, bool BIAS, bool GATE, bool EXACT>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) block_norm_backward_kernel(const BlockNormParams p) {
    constexpr int NT = TPR > 256 ? TPR : 256, GROUPS = NT / TPR;
    typedef Piece<TPR, EXACT> P;
    constexpr bool HAS_Y = MODE == 2 || GATE, BOTH = N == 1;
    __shared__ float lds[2][2][TPR / 64 + 1];
    constexpr int VECTORS = 1 + (BIAS ? 1 : 0) + (MODE == 2 ? 1 + (BIAS ? 1 : 0) : 0) + (GATE ? 1 : 0);  // of column sums
    constexpr bool TOGETHER = VECTORS * GROUPS * TPR * N * sizeof(f32x4) <= 48 << 10;  // in LDS (2000 x 64: 7.4 us, one by one 9.0)
    __shared__ f32x4 meet[GROUPS > 1 ? (TOGETHER ? VECTORS : 1) * GROUPS * TPR * N : 1];
    int turn = 0;
    const int lane = threadIdx.x % TPR, group = row_group<TPR>(), dim = p.dim;
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
    // this group's rows: r, r + step ... below r_end.  With `flush` they are whole gate groups, and gate_row counts them;
    // else all have the same gate row
    const long long chunk = blockIdx.x;
    long long r, r_end, gate_row;
    int step = 1;
    if (p.flush) {
        const int each = p.groups_per_chunk / GROUPS;  // a multiple
        gate_row = chunk * p.groups_per_chunk + group * each;
        r = gate_row * p.rows_per_group, r_end = r + each * p.rows_per_group;
        if (r_end > p.rows) r_end = p.rows;
    } else {
        gate_row = chunk / p.chunks_per_group;
        r_end = (gate_row + 1) * p.rows_per_group < p.rows ? (gate_row + 1) * p.rows_per_group : p.rows;
        r = gate_row * p.rows_per_group + (chunk - gate_row * p.chunks_per_group) * p.rows_per_chunk;
        if (r + p.rows_per_chunk < r_end) r_end = r + p.rows_per_chunk;
        r += group, step = GROUPS;
    }
    long long left_in_group = p.rows_per_group;
    const bool gate_in_rows = p.gate_rows != 0;

    // what the norm ahead of the next block needs of a row, and what the norm behind this one needs: the first part of the
    // next row and the second part of this one are under way while the other is worked on.  (BOTH: with one piece to a thread the
    // work on the first is over too soon for that, and there are registers for the next row's second part, too.)
    struct Ahead {
        raw4<TS> u[N], du[N];
        raw4<TB> dh[N];
        float mean, rstd;
    } ahead = {};
    struct Behind {
        raw4<TB> y[HAS_Y ? N : 1], g[GATE ? N : 1];
        float mean, rstd;
    };
    auto fetch_ahead = [&](long long row) {
        if (p.dh != nullptr) {
            ahead.mean = p.pre_s[2 * row], ahead.rstd = p.pre_s[2 * row + 1];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                ahead.u[n] = P::load(static_cast<const TS*>(p.u) + row * p.ld_u, n, lane, dim);
                ahead.dh[n] = P::load(static_cast<const TB*>(p.dh) + row * p.ld_h, n, lane, dim);
            }
        }
        if (p.du != nullptr)
#pragma unroll
            for (int n = 0; n < N; ++n)
                ahead.du[n] = P::load(static_cast<const TS*>(p.du) + row * p.ld_u, n, lane, dim);
    };
    auto fetch_behind = [&](Behind& w, long long row, long long g_row) {
        if constexpr (HAS_Y)
#pragma unroll
            for (int n = 0; n < N; ++n) w.y[n] = P::load(static_cast<const TB*>(p.y) + row * p.ld_y, n, lane, dim);
        if constexpr (MODE == 2) w.mean = p.post_s[2 * row], w.rstd = p.post_s[2 * row + 1];
        if constexpr (GATE)
            if (gate_in_rows)
#pragma unroll
                for (int n = 0; n < N; ++n) w.g[n] = P::load(static_cast<const TB*>(p.gate) + g_row * p.ld_gate, n, lane, dim);
    };
    Behind now = {};
    if (r < r_end) {
        fetch_ahead(r);
        if constexpr (BOTH) fetch_behind(now, r, gate_row);
    }
    for (; r < r_end; r += step) {
        const bool last_of_group = p.flush && (left_in_group == 1 || r + step >= r_end);
        if constexpr (!BOTH) fetch_behind(now, r, gate_row);
        f32x4 t[N], hat[N];
        if (p.dh != nullptr) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const f32x4 dh = P::value(ahead.dh[n], n, lane, dim);
                hat[n] = (P::value(ahead.u[n], n, lane, dim) - ahead.mean) * ahead.rstd;
                acc_w[n] += dh * hat[n];
                if constexpr (BIAS) acc_b[n] += dh;
                t[n] = dh * P::vector(p.pre_w, n, lane, dim, 1.0f);
            }
            row_gradient<TPR, N>(t, hat, p.pre, ahead.rstd, p, lds, turn);
            if (p.du != nullptr)
#pragma unroll
                for (int n = 0; n < N; ++n) t[n] += P::value(ahead.du[n], n, lane, dim);
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) t[n] = P::value(ahead.du[n], n, lane, dim);
        }
        Behind next = {};
        if (r + step < r_end) {
            fetch_ahead(r + step);
            if constexpr (BOTH) fetch_behind(next, r + step, last_of_group ? gate_row + 1 : gate_row);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) P::store(static_cast<TS*>(p.dx) + r * p.ld_x, n, lane, dim, t[n]);
        if constexpr (MODE > 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                t[n] = P::cut(t[n] * p.scale, n, lane, dim);
                if constexpr (HAS_Y) {
                    hat[n] = P::value(now.y[n], n, lane, dim);
                    if constexpr (MODE == 2) hat[n] = (hat[n] - now.mean) * now.rstd;
                }
                f32x4 w;
                if constexpr (MODE == 2) w = P::vector(p.post_w, n, lane, dim, 1.0f);
                if constexpr (GATE) {
                    f32x4 v = hat[n], g;
                    if constexpr (MODE == 2) v = v * w + P::vector(p.post_b, n, lane, dim, 0.0f);
                    if (gate_in_rows)
                        g = P::value(now.g[n], n, lane, dim);
                    else
                        g = P::vector(static_cast<const float*>(p.gate), n, lane, dim, 1.0f);
                    gate_gradient<(TPR > 256)>(t[n], acc_g[n], v, g, p.act);
                }
                if constexpr (MODE == 2) {
                    acc_pw[n] += t[n] * hat[n];
                    if constexpr (BIAS) acc_pb[n] += t[n];
                    t[n] *= w;
                }
            }
            if constexpr (MODE == 2) row_gradient<TPR, N>(t, hat, p.post, now.rstd, p, lds, turn);
#pragma unroll
            for (int n = 0; n < N; ++n) P::store(static_cast<TB*>(p.dy) + r * p.ld_y, n, lane, dim, t[n]);
        }
        if constexpr (GATE) {
            if (last_of_group) {  // the group's rows are in
                if (p.d_gate != nullptr)
#pragma unroll
                    for (int n = 0; n < N; ++n)
                        P::store(static_cast<TB*>(p.d_gate) + gate_row * p.ld_gate, n, lane, dim, acc_g[n]);
#pragma unroll
                for (int n = 0; n < N; ++n) acc_g[n] = zero;
            }
        }
        if (last_of_group) ++gate_row;
        left_in_group = last_of_group ? p.rows_per_group : left_in_group - 1;
        if constexpr (BOTH) now = next;
    }
    // the column sums of the chunk; groups of threads that share the columns meet in LDS
    auto every = [&](auto&& each) {  // the sums there are, with the slot of each
        each(acc_w, 0);
        if constexpr (BIAS) each(acc_b, 1);
        if constexpr (MODE == 2) each(acc_pw, 2);
        if constexpr (MODE == 2 && BIAS) each(acc_pb, 3);
        if constexpr (GATE) each(acc_g, 4);
    };
    if constexpr (GROUPS > 1) {
        constexpr int PIECES = TPR * N;
        auto put = [&](const f32x4* acc, int v) {
#pragma unroll
            for (int n = 0; n < N; ++n) meet[(v * GROUPS + group) * PIECES + n * TPR + lane] = acc[n];
        };
        auto add_up = [&](int v, int piece, int slot) {
            f32x4 sum = meet[v * GROUPS * PIECES + piece];
            for (int g = 1; g < GROUPS; ++g) sum += meet[(v * GROUPS + g) * PIECES + piece];
            store4(p.partial + ((long long)slot * p.chunks + chunk) * dim + 4 * piece, dim - 4 * piece, sum);
        };
        if constexpr (TOGETHER) {
            int v = 0;
            every([&](const f32x4* acc, int) { put(acc, v++); });
            __syncthreads();
            for (int k = threadIdx.x; k < VECTORS * PIECES; k += NT) {
                const int piece = k % PIECES, vector = k / PIECES;
                int slot = -1, at = 0;
                every([&](const f32x4*, int s) {
                    if (at == vector) slot = p.slot[s];
                    ++at;
                });
                if (slot >= 0) add_up(vector, piece, slot);
            }
        } else {
            every([&](const f32x4* acc, int s) {
                if (p.slot[s] < 0) return;
                __syncthreads();
                put(acc, 0);
                __syncthreads();
                for (int piece = threadIdx.x; piece < PIECES; piece += NT) add_up(0, piece, p.slot[s]);
            });
        }
    } else {
        every([&](const f32x4* acc, int s) {
            if (p.slot[s] < 0) return;
            float* out = p.partial + ((long long)p.slot[s] * p.chunks + chunk) * dim;
#pragma unroll
            for (int n = 0; n < N; ++n) P::store(out, n, lane, dim, acc[n]);
        });
    }
}

}  // namespace snhip
