// Word embedding: the lookup with its scale, and the gradient of the table by sorted tokens.
//
//   y[t] = scale * W[id[t]]                           WordEmbeddingForwardPropagation   SinglePrecision.cu:617
//   dW[v] = scale * sum of dy[t] over id[t] = v       WordEmbeddingBackwardPropagation  SinglePrecision.cu:650
//
// Both are bound by HBM.  The gradient is built without float atomics, in an order that depends on the ids alone, so its
// bits repeat: the tokens are sorted by id (embedding_sort_kernel), runs of equal ids are added up in chunks of the sorted
// order (embedding_grad_kernel, which also clears the rows that no token has), and runs that cross a chunk's end are
// joined from their chunks' sums (embedding_join_kernel).
#pragma once
#include <hip/hip_runtime.h>

#include "vec_types.hpp"

namespace snhip {

// The id of token t, or -1 for one outside [0, vocabulary) (no token).  Ids stored as floats, as the reference keeps
// them, are rounded toward zero like its (int) cast; NaN is no token.
__device__ __forceinline__ int token_id(const float* ids, long long t, int vocabulary) {
    const float f = ids[t];
    return f > -1.0f && f < (float)vocabulary && (int)f < vocabulary ? (int)f : -1;
}
__device__ __forceinline__ int token_id(const int* ids, long long t, int vocabulary) {
    const int i = ids[t];
    return i >= 0 && i < vocabulary ? i : -1;
}
__device__ __forceinline__ int token_id(const long long* ids, long long t, int vocabulary) {
    const long long i = ids[t];
    return i >= 0 && i < vocabulary ? (int)i : -1;
}

struct EmbeddingParams {
    const void* ids;
    const void* in;   // forward: the table; gradient: dy
    void* out;        // forward: y; gradient: dW
    long long tokens, ld_in, ld_out;
    int vocabulary, dim;
    int padding;      // id whose tokens add nothing to the gradient, or -1
    float scale;
    int whole;        // rows of `in` and `out` can be accessed four elements at a time
    int lanes_log2;   // threads per row of a workgroup of 256
    int accumulate;   // gradient: dW += instead of dW =
    int bins;         // ids per workgroup of the sort
    int chunk;        // sorted tokens per group of threads of the gradient
    long long chunk_blocks;  // workgroups that add up chunks; those behind them clear rows without tokens
    int* order;       // [tokens]: token numbers, sorted by id
    int* sorted;      // [tokens]: their ids
    int* offsets;     // [vocabulary + 1]: where each id's run starts in `order`
    float* partial;   // [chunks][2][dim]: sums of the runs that came into a chunk / went on behind it
};

// A group of 2^lanes_log2 threads copies ROWS rows, all of whose loads are under way before the first store.
template <typename ID, typename TIN, typename TOUT, int ROWS>
__global__ void __launch_bounds__(256) embedding_forward_kernel(const EmbeddingParams p) {
    const int lane = threadIdx.x & ((1 << p.lanes_log2) - 1), group = threadIdx.x >> p.lanes_log2;
    const int groups = 256 >> p.lanes_log2;
    const long long t0 = ((long long)blockIdx.x * groups + group) * ROWS;
    const int c = (blockIdx.y << (p.lanes_log2 + 2)) + 4 * lane;
    if (c >= p.dim) return;
    int id[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        id[r] = t0 + r < p.tokens ? token_id(static_cast<const ID*>(p.ids), t0 + r, p.vocabulary) : -1;
    f32x4 v[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        v[r] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (id[r] >= 0) v[r] = load4(static_cast<const TIN*>(p.in) + (long long)id[r] * p.ld_in, c, p.dim, p.whole);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (t0 + r < p.tokens)
            store4(static_cast<TOUT*>(p.out) + (t0 + r) * p.ld_out, c, p.dim, p.whole, v[r] * p.scale);
}

// Sorts the tokens by id in one launch: a workgroup owns `bins` consecutive ids and reads all of them.  Its 16 wavefronts
// take a contiguous part of the tokens each and count their ids (LDS, [wavefront][id]) and the tokens with smaller ids
// (which is where the workgroup's part of `order` starts); after a scan over (id, wavefront) every wavefront walks its
// part again and puts each token behind the earlier ones of its id.  The order within an id is thus fixed: by wavefront,
// then by position.  Reading the ids in every workgroup costs 256 x tokens x 4..8 bytes from L2 and saves the launches of
// a radix sort.
template <typename ID>
__global__ void __launch_bounds__(1024) embedding_sort_kernel(const EmbeddingParams p) {
    extern __shared__ int count[];  // [16][bins], then the cursors
    __shared__ int below[16], wave_total[16];
    constexpr int U = 8;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int lo = blockIdx.x * p.bins;
    const int bins = p.vocabulary - lo < p.bins ? p.vocabulary - lo : p.bins;
    for (int i = tid; i < 16 * bins; i += 1024) count[i] = 0;
    __syncthreads();
    const long long per = ((p.tokens + 1023) / 1024) * 64;
    const long long begin = w * per < p.tokens ? w * per : p.tokens;
    const long long end = begin + per < p.tokens ? begin + per : p.tokens;
    const ID* ids = static_cast<const ID*>(p.ids);
    int smaller = 0;
    for (long long t = begin; t < end; t += 64 * U) {
        int id[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const long long tt = t + 64 * j + lane;
            id[j] = tt < end ? token_id(ids, tt, p.vocabulary) : -1;
            if (id[j] == p.padding) id[j] = -1;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int b = id[j] - lo;
            if (b >= 0 && b < bins) atomicAdd(&count[w * bins + b], 1);
            smaller += id[j] >= 0 && b < 0;
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) smaller += __shfl_xor(smaller, off, 64);
    if (lane == 0) below[w] = smaller;
    __syncthreads();
    // ids' totals, scanned over the ids (at most 512: the first eight wavefronts)
    int mine = 0;
    if (tid < bins)
        for (int k = 0; k < 16; ++k) mine += count[k * bins + tid];
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(upto, off, 64);
        if (lane >= off) upto += o;
    }
    if (lane == 63) wave_total[w] = upto;
    __syncthreads();
    int start = 0;
    for (int k = 0; k < 16; ++k) start += below[k];
    for (int k = 0; k < w; ++k) start += wave_total[k];
    start += upto - mine;
    if (tid < bins) {
        p.offsets[lo + tid] = start;
        if (lo + tid == p.vocabulary - 1) p.offsets[p.vocabulary] = start + mine;
        for (int k = 0; k < 16; ++k) {
            const int n = count[k * bins + tid];
            count[k * bins + tid] = start;
            start += n;
        }
    }
    __syncthreads();
    for (long long t = begin; t < end; t += 64 * U) {
        int id[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const long long tt = t + 64 * j + lane;
            id[j] = tt < end ? token_id(ids, tt, p.vocabulary) : -1;
            if (id[j] == p.padding) id[j] = -1;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int b = id[j] - lo;
            const bool in = b >= 0 && b < bins;
            unsigned long long left = __ballot(in);
            while (left != 0) {  // one turn per distinct id among the 64 tokens
                const int first = __ffsll(left) - 1;
                const int bb = __shfl(b, first, 64);
                const unsigned long long same = __ballot(in && b == bb);
                int at = 0;
                if (lane == first) at = atomicAdd(&count[w * bins + bb], __popcll(same));
                at = __shfl(at, first, 64);
                if (in && b == bb) {
                    at += __popcll(same & ((1ULL << lane) - 1));
                    p.order[at] = (int)(t + 64 * j + lane);
                    p.sorted[at] = id[j];
                }
                left &= ~same;
            }
        }
    }
}

__device__ __forceinline__ void put_gradient(const EmbeddingParams& p, int id, int c, f32x4 sum) {
    float* row = static_cast<float*>(p.out) + (long long)id * p.ld_out;
    sum *= p.scale;
    if (p.accumulate) sum += load4(row, c, p.dim, p.whole);
    store4(row, c, p.dim, p.whole, sum);
}

// A group of threads adds up `chunk` consecutive sorted tokens, U rows of dy under way at a time.  A run of equal ids that
// begins and ends inside the chunk is a finished row of dW; the others leave their part in `partial`: slot 0 the run that
// came in from the chunk before (also when it goes on behind this one), slot 1 the one that starts here and goes on.
template <typename T>
__global__ void __launch_bounds__(256) embedding_grad_kernel(const EmbeddingParams p) {
    constexpr int U = 8;
    const int lane = threadIdx.x & ((1 << p.lanes_log2) - 1), group = threadIdx.x >> p.lanes_log2;
    const int groups = 256 >> p.lanes_log2;
    const int c = (blockIdx.y << (p.lanes_log2 + 2)) + 4 * lane;
    if (c >= p.dim) return;
    if (blockIdx.x >= p.chunk_blocks) {  // rows that no token has
        constexpr int ROWS = 8;
        const long long r0 = ((blockIdx.x - p.chunk_blocks) * groups + group) * ROWS;
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const long long r = r0 + k;
            if (r < p.vocabulary && p.offsets[r] == p.offsets[r + 1])
                store4(static_cast<float*>(p.out) + r * p.ld_out, c, p.dim, p.whole, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        }
        return;
    }
    const long long k = (long long)blockIdx.x * groups + group;
    const long long n = p.offsets[p.vocabulary];
    const long long p0 = k * p.chunk;
    if (p0 >= n) return;
    const long long p1 = p0 + p.chunk < n ? p0 + p.chunk : n;
    const T* dy = static_cast<const T*>(p.in);
    int cur = p.sorted[p0];
    bool came_in = p0 > 0 && p.sorted[p0 - 1] == cur;
    const bool goes_on = p1 < n && p.sorted[p1] == p.sorted[p1 - 1];
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float* slot = p.partial + 2 * k * p.dim;
    const bool whole_slot = (p.dim & 3) == 0;
    for (long long q = p0; q < p1; q += U) {
        int id[U];
        f32x4 v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const bool in = q + j < p1;
            id[j] = in ? p.sorted[q + j] : -1;
            v[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (in) v[j] = load4(dy + (long long)p.order[q + j] * p.ld_in, c, p.dim, p.whole);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (id[j] < 0) continue;
            if (id[j] != cur) {  // the run before has ended
                if (came_in)
                    store4(slot, c, p.dim, whole_slot, sum);
                else
                    put_gradient(p, cur, c, sum);
                came_in = false;
                cur = id[j];
                sum = v[j];
            } else {
                sum += v[j];
            }
        }
    }
    if (came_in)
        store4(slot, c, p.dim, whole_slot, sum);
    else if (goes_on)
        store4(slot + p.dim, c, p.dim, whole_slot, sum);
    else
        put_gradient(p, cur, c, sum);
}

// The rows whose run crosses the end of a chunk: the group of the chunk where the run starts adds its part and those of the
// chunks behind it, in their order, in 64 bits (a frequent word has thousands of parts).
__global__ void __launch_bounds__(256) embedding_join_kernel(const EmbeddingParams p) {
    constexpr int U = 8;
    const int lane = threadIdx.x & ((1 << p.lanes_log2) - 1), group = threadIdx.x >> p.lanes_log2;
    const int groups = 256 >> p.lanes_log2;
    const int c = (blockIdx.y << (p.lanes_log2 + 2)) + 4 * lane;
    if (c >= p.dim) return;
    const long long k = (long long)blockIdx.x * groups + group;
    const long long n = p.offsets[p.vocabulary];
    const long long last = (k + 1) * p.chunk - 1;
    if (last + 1 >= n) return;
    const int id = p.sorted[last];
    if (p.sorted[last + 1] != id || p.offsets[id] < k * p.chunk) return;
    const long long k_end = (p.offsets[id + 1] - 1) / p.chunk;
    const bool whole_slot = (p.dim & 3) == 0;
    const f32x4 first = load4(p.partial + (2 * k + 1) * p.dim, c, p.dim, whole_slot);
    double sum[4] = {first[0], first[1], first[2], first[3]};
    for (long long q = k + 1; q <= k_end; q += U) {
        f32x4 v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            v[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (q + j <= k_end) v[j] = load4(p.partial + 2 * (q + j) * p.dim, c, p.dim, whole_slot);
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += v[j][e];
    }
    put_gradient(p, id, c, f32x4{(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]});
}

}  // namespace snhip
