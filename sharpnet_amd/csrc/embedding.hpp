// Word embedding: the lookup with its scale, and the gradient of the table by sorted tokens.
//
//   y[t] = scale * W[id[t]]                           WordEmbeddingForwardPropagation   SinglePrecision.cu:617
//   dW[v] = scale * sum of dy[t] over id[t] = v       WordEmbeddingBackwardPropagation  SinglePrecision.cu:650
//
// Both are bound by HBM.  The gradient is built without float atomics, in an order that depends on the ids alone, so its
// bits repeat: the tokens are sorted by id (embedding_sort_kernel), runs of equal ids are added up in chunks of the sorted
// order (embedding_grad_kernel), and runs that cross a chunk's end are joined from their chunks' sums
// (embedding_join_kernel, which also clears the rows that no token has).  65536 tokens x 1024 bf16 into 50000 rows: sort 5 and
// 13 us, sums 45 us (4.3 TB/s of rows that lie anywhere), joins and clearing 31 us; together 95 us.  Clearing beside the sums
// instead of beside the joins took 3 us more.  The lookup of 32768 x 2048, fp32 to bf16, 62 us.
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
    int lanes_log2;   // threads per row of a workgroup of 256
    int accumulate;   // gradient: dW += instead of dW =
    int sort_blocks, sort_log2;  // buckets of the sort, a power of two
    int fine_log2;               // ... over 256 of them: 2^fine_log2 times 256
    int bins, bins_log2;         // ids of each (at most 512), and the bits that number them
    int chunk;        // sorted tokens per group of threads of the gradient
    unsigned int join_blocks, join_columns;  // workgroups that join chunks, and how many of them share one's columns
    unsigned int clear_columns;              // the same of those behind them, which clear rows without tokens
    int* order;       // [tokens]: token numbers, sorted by key (see embedding_sort_kernel)
    int* sorted;      // [tokens]: their ids' keys
    int* offsets;     // [sort_blocks * bins + 1]: where each key's run starts in `order`
    int pieces;       // of embedding_bucket_kernel
    int *piece_id, *piece_token, *piece_start;
    long long chunks;
    int* crossing;    // [chunks][2]: key of the run that starts in the chunk and goes on behind it (or -1), its last chunk
    float* partial;   // [chunks][2][dim]: sums of the runs that came into a chunk / went on behind it
};

// A group of 2^lanes_log2 threads copies ROWS rows, all of whose loads are under way before the first store.
template <typename ID, typename TIN, typename TOUT, int ROWS>
__global__ void __launch_bounds__(256) embedding_forward_kernel(const EmbeddingParams p) {
    const int lane = threadIdx.x & ((1 << p.lanes_log2) - 1), group = threadIdx.x >> p.lanes_log2;
    const int groups = 256 >> p.lanes_log2;
    const long long t0 = (block_number() * groups + group) * ROWS;
    const int c = (blockIdx.y << (p.lanes_log2 + 2)) + 4 * lane;
    if (c >= p.dim) return;
    const bool ends = __ballot(p.dim - c < 4) != 0;
    int id[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        id[r] = t0 + r < p.tokens ? token_id(static_cast<const ID*>(p.ids), t0 + r, p.vocabulary) : -1;
    raw4<TIN> v[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        v[r] = raw4<TIN>{};
        if (id[r] >= 0) v[r] = load4_row(static_cast<const TIN*>(p.in) + (long long)id[r] * p.ld_in, c, p.dim);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
        if (t0 + r < p.tokens)
            store4(static_cast<TOUT*>(p.out) + (t0 + r) * p.ld_out + c, p.dim - c, existing(widen(v[r]), p.dim - c, ends) * p.scale);
}

// The sort.  Ids are dealt out to the workgroups of embedding_sort_kernel in turn (words come by frequency in most
// vocabularies: neighbours would put half of all tokens into one workgroup): id i is number i / B of bucket i % B, its key
// rank * bins + i / B with the buckets ranked by i % 256 first.  The workgroup of a bucket finds its tokens in the order of
// their positions, a contiguous part to each of its 16 wavefronts, and counts them by wavefront and id in LDS; after a scan
// over (id, wavefront) every wavefront puts its tokens behind the earlier ones of their ids.  The order of all this is a
// function of the ids alone.
// Where the tokens come from: with few of them every workgroup reads all ids, which saves a launch (8192 tokens of 512: 29 us
// instead of 36 us).  With many, embedding_bucket_kernel has sorted the tokens by bucket, in pieces, so that a workgroup
// reads its own alone (65536 tokens: 34 us the first way, 18 us the second).
constexpr int kSortDirect = 8192; // tokens up to which every workgroup reads all ids
constexpr int kPiece = 512;       // tokens that a workgroup of embedding_bucket_kernel sorts
constexpr int kBuckets = 256;     // ... by bucket (bucket modulo 256 if there are more)

// The lanes of `in` whose value (bits wide) is this lane's.
__device__ __forceinline__ unsigned long long same_value(bool in, int value, int bits) {
    unsigned long long same = __ballot(in);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long ones = __ballot((value >> b) & 1);
        same &= (value >> b) & 1 ? ones : ~ones;
    }
    return same;
}

// The place of every lane of `in` among the wavefront's tokens of its value: behind those that `cursors` has counted so far
// and those of the lanes before; counts them.
__device__ __forceinline__ int take_place(bool in, int value, int bits, int* cursors) {
    const int lane = threadIdx.x & 63;
    const unsigned long long before = (1ULL << lane) - 1, same = same_value(in, value, bits);
    int at = 0;
    if (in) {
        volatile int* cursor = &cursors[value];
        at = *cursor + __popcll(same & before);
        if ((same & ~before) == (1ULL << lane)) *cursor = at + 1;  // the last of its value
    }
    return at;
}

// count[WAVES][values] becomes the places where each wavefront's tokens of each value start, from `first` on; start: where
// the value of this thread (threadIdx.x < values) starts, total: how many there are of it.  values <= 512, one per thread.
template <int WAVES>
__device__ __forceinline__ void scan_counts(int* count, int values, int first, int* wave_total, int& start, int& total) {
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    int n[WAVES];
    total = 0;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
        n[k] = tid < values ? count[k * values + tid] : 0;
        total += n[k];
    }
    int upto = total;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(upto, off, 64);
        if (lane >= off) upto += o;
    }
    if (lane == 63) wave_total[w] = upto;
    __syncthreads();
    start = first + upto - total;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) start += k < w ? wave_total[k] : 0;
    int at = start;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
        if (tid < values) count[k * values + tid] = at;
        at += n[k];
    }
    __syncthreads();
}

// Pieces of kPiece tokens, sorted by bucket modulo 256: the piece's ids and positions at [piece * kPiece ...) of piece_id /
// piece_token, where each bucket starts in the piece at piece_start[bucket][piece] (and the piece's end as bucket 256).
template <typename ID>
__global__ void __launch_bounds__(256) embedding_bucket_kernel(const EmbeddingParams p) {
    __shared__ int count[4 * kBuckets], wave_total[4];
    __shared__ int sorted_id[kPiece], sorted_token[kPiece];
    constexpr int PER = kPiece / 256;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int mask = (p.sort_blocks < kBuckets ? p.sort_blocks : kBuckets) - 1;
    for (int i = tid; i < 4 * kBuckets; i += 256) count[i] = 0;
    const long long t0 = (long long)blockIdx.x * kPiece + w * (kPiece / 4) + lane;
    int id[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        id[j] = t0 + 64 * j < p.tokens ? token_id(static_cast<const ID*>(p.ids), t0 + 64 * j, p.vocabulary) : -1;
        if (id[j] == p.padding) id[j] = -1;
    }
    __syncthreads();
    int place[PER];  // among the wavefront's tokens of the bucket
#pragma unroll
    for (int j = 0; j < PER; ++j) place[j] = take_place(id[j] >= 0, id[j] & mask, 8, count + w * kBuckets);
    __syncthreads();
    int start, total;
    scan_counts<4>(count, kBuckets, 0, wave_total, start, total);
    int* starts = p.piece_start + blockIdx.x;
    starts[(long long)tid * p.pieces] = start;
    if (tid == kBuckets - 1) {
        starts[(long long)kBuckets * p.pieces] = start + total;
        wave_total[0] = start + total;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (id[j] < 0) continue;
        const int at = count[w * kBuckets + (id[j] & mask)] + place[j];
        sorted_id[at] = id[j], sorted_token[at] = (int)(t0 + 64 * j);
    }
    __syncthreads();
    const int n = wave_total[0];
    for (int i = tid; i < n; i += 256) {
        p.piece_id[(long long)blockIdx.x * kPiece + i] = sorted_id[i];
        p.piece_token[(long long)blockIdx.x * kPiece + i] = sorted_token[i];
    }
}

// How buckets are ranked: by their number modulo 256, then by the rest.
__device__ __forceinline__ int rank_of_id(const EmbeddingParams& p, int id) {
    const int b = id & (p.sort_blocks - 1);
    return ((b & (kBuckets - 1)) << p.fine_log2) | (b / kBuckets);
}

// Puts the wavefronts' counts of this workgroup's ids in place and notes where each id starts.
__device__ __forceinline__ void start_ids(const EmbeddingParams& p, int* count, const int* below, int* wave_total) {
    const int tid = threadIdx.x, rank = blockIdx.x;
    int first = 0, start, total;
#pragma unroll
    for (int k = 0; k < 16; ++k) first += below[k];
    scan_counts<16>(count, p.bins, first, wave_total, start, total);
    if (tid < p.bins) p.offsets[rank * p.bins + tid] = start;
    if (rank == p.sort_blocks - 1 && tid == p.bins - 1) p.offsets[p.sort_blocks * p.bins] = start + total;
}

// At most kSortDirect tokens.
template <typename ID>
__global__ void __launch_bounds__(1024) embedding_sort_kernel(const EmbeddingParams p) {
    extern __shared__ int count[];  // [16][bins], then the cursors
    __shared__ int below[16], wave_total[16];
    constexpr int PER = kSortDirect / 1024;                  // tokens per lane
    __shared__ unsigned short notes[16][kSortDirect / 16];  // places of the wavefront's tokens of this bucket in its part
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, rank = blockIdx.x;
    for (int i = tid; i < 16 * p.bins; i += 1024) count[i] = 0;
    __syncthreads();
    const int per = (int)((p.tokens + 1023) / 1024) * 64;
    const int begin = w * per, end = begin + per < p.tokens ? begin + per : (int)p.tokens;
    const ID* ids = static_cast<const ID*>(p.ids);
    const unsigned long long before = (1ULL << lane) - 1;
    int smaller = 0, noted = 0, id[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = begin + 64 * j + lane;
        id[j] = t < end ? token_id(ids, t, p.vocabulary) : -1;
        if (id[j] == p.padding) id[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int r = rank_of_id(p, id[j]);
        const bool mine = id[j] >= 0 && r == rank;
        smaller += id[j] >= 0 && r < rank;
        const unsigned long long hits = __ballot(mine);
        if (mine) {
            atomicAdd(&count[w * p.bins + (id[j] >> p.sort_log2)], 1);
            notes[w][noted + __popcll(hits & before)] = (unsigned short)(64 * j + lane);
        }
        noted += __popcll(hits);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) smaller += __shfl_xor(smaller, off, 64);
    if (lane == 0) below[w] = smaller;
    __syncthreads();
    start_ids(p, count, below, wave_total);
    for (int k = 0; k < noted; k += 64) {
        const bool in = k + lane < noted;
        const int t = begin + (in ? notes[w][k + lane] : 0);
        const int number = in ? token_id(ids, t, p.vocabulary) >> p.sort_log2 : 0;
        const int at = take_place(in, number, p.bins_log2, count + w * p.bins);
        if (in) p.order[at] = t, p.sorted[at] = rank * p.bins + number;
    }
}

// From embedding_bucket_kernel's pieces; a wavefront takes a run of pieces.
__global__ void __launch_bounds__(1024) embedding_sort_pieces_kernel(const EmbeddingParams p) {
    extern __shared__ int count[];  // [16][bins], then the cursors
    __shared__ int below[16], wave_total[16];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), rank = blockIdx.x;
    for (int i = tid; i < 16 * p.bins; i += 1024) count[i] = 0;
    __syncthreads();
    const int per = (p.pieces + 15) / 16;
    const int begin = w * per < p.pieces ? w * per : p.pieces, end = begin + per < p.pieces ? begin + per : p.pieces;
    const int* from = p.piece_start + (long long)(rank >> p.fine_log2) * p.pieces;
    const int* to = from + p.pieces;
    // Eight pieces at a time: a piece has a handful of tokens of a bucket, and one after the other each would wait for memory.
    constexpr int U = 8;
    int a[U], b[U], longest = 0, id[U], token[U], place[U];
    int* counts = count + w * p.bins;  // this wavefront's
    auto bounds = [&](int i0) {
        longest = 0;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int i = i0 + j < end ? i0 + j : end - 1;
            a[j] = from[i], b[j] = i0 + j < end ? to[i] : 0;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) longest = b[j] - a[j] > longest ? b[j] - a[j] : longest;
    };
    auto fetch = [&](int i0, int k) {  // up to 64 tokens of each, from the k-th on
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int at = a[j] + k + lane;
            const long long place = (long long)(i0 + j) * kPiece + at;
            id[j] = at < b[j] ? p.piece_id[place] : -1;
            token[j] = at < b[j] ? p.piece_token[place] : 0;
        }
    };
    int smaller = 0;
    for (int i0 = begin; i0 < end; i0 += U) {
        bounds(i0);
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (lane == 0 && i0 + j < end) smaller += a[j];
        for (int k = 0; k < longest; k += 64) {
            fetch(i0, k);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int r = rank_of_id(p, id[j]);
                smaller += id[j] >= 0 && r < rank;
                if (r != rank) id[j] = -1;
                if (__ballot(id[j] >= 0) != 0) place[j] = take_place(id[j] >= 0, id[j] >> p.sort_log2, p.bins_log2, counts);
            }
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) smaller += __shfl_xor(smaller, off, 64);
    if (lane == 0) below[w] = smaller;
    __syncthreads();
    start_ids(p, count, below, wave_total);
    // all of this wavefront's tokens are in its registers still
    const bool held = begin < end && end - begin <= U && longest > 0 && longest <= 64;
    auto put = [&](int j, int at) { p.order[at] = token[j], p.sorted[at] = rank * p.bins + (id[j] >> p.sort_log2); };
    if (held) {
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (id[j] >= 0) put(j, counts[id[j] >> p.sort_log2] + place[j]);
        return;
    }
    for (int i0 = begin; i0 < end; i0 += U) {
        bounds(i0);
        for (int k = 0; k < longest; k += 64) {
            fetch(i0, k);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const bool in = id[j] >= 0 && rank_of_id(p, id[j]) == rank;
                if (__ballot(in) == 0) continue;
                const int at = take_place(in, id[j] >> p.sort_log2, p.bins_log2, counts);
                if (in) put(j, at);
            }
        }
    }
}

__device__ __forceinline__ int id_of_key(const EmbeddingParams& p, int key) {
    const int rank = key / p.bins;
    return ((key - rank * p.bins) << p.sort_log2) | (rank >> p.fine_log2) | ((rank & ((1 << p.fine_log2) - 1)) * kBuckets);
}

__device__ __forceinline__ void put_gradient(const EmbeddingParams& p, int key, int c, f32x4 sum) {
    const int id = id_of_key(p, key);
    float* row = static_cast<float*>(p.out) + (long long)id * p.ld_out + c;
    sum *= p.scale;
    if (p.accumulate) sum += load4(row, p.dim - c);
    store4(row, p.dim - c, sum);
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
    const int left = p.dim - c;
    const bool ends = __ballot(left < 4) != 0;
    const int keys = p.sort_blocks * p.bins;
    const long long k = (long long)blockIdx.x * groups + group;
    const long long n = p.offsets[keys];
    const long long p0 = k * p.chunk;
    if (p0 >= n) {
        if (c == 0 && k < p.chunks) p.crossing[2 * k] = -1;
        return;
    }
    const long long p1 = p0 + p.chunk < n ? p0 + p.chunk : n;
    const T* dy = static_cast<const T*>(p.in);
    int cur = p.sorted[p0];
    bool came_in = p0 > 0 && p.sorted[p0 - 1] == cur;
    const bool goes_on = p1 < n && p.sorted[p1] == p.sorted[p1 - 1];
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float* slot = p.partial + 2 * k * p.dim + c;
    int key[U], token[U];
    auto fetch = [&](long long q) {  // behind the chunk's end: its last token again
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const long long at = q + j < p1 ? q + j : p1 - 1;
            key[j] = p.sorted[at], token[j] = p.order[at];
        }
    };
    fetch(p0);
    for (long long q = p0; q < p1; q += U) {
        raw4<T> v[U];
        int now[U];
        // (read once: kept out of the caches, 59 -> 44 us for 65536 rows of 1024 bf16)
        if (p.dim >= 4) {
            const T* at = dy + (left >= 4 ? c : p.dim - 4);  // as load4_row
#pragma unroll
            for (int j = 0; j < U; ++j) v[j] = load4_once(at + (long long)token[j] * p.ld_in);
        } else {
#pragma unroll
            for (int j = 0; j < U; ++j) v[j] = load4_row(dy + (long long)token[j] * p.ld_in, c, p.dim);
        }
#pragma unroll
        for (int j = 0; j < U; ++j) now[j] = q + j < p1 ? key[j] : -1;
        if (q + U < p1) fetch(q + U);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (now[j] < 0) continue;
            if (now[j] != cur) {  // the run before has ended
                if (came_in)
                    store4(slot, left, sum);
                else
                    put_gradient(p, cur, c, sum);
                came_in = false;
                cur = now[j];
                sum = existing(widen(v[j]), left, ends);
            } else {
                sum += existing(widen(v[j]), left, ends);
            }
        }
    }
    if (c == 0) {  // (the first column's thread) what the join has to know of this chunk
        const bool starts = !came_in && goes_on;
        p.crossing[2 * k] = starts ? cur : -1;
        p.crossing[2 * k + 1] = starts ? (int)((p.offsets[cur + 1] - 1) / p.chunk) : 0;
    }
    if (came_in)
        store4(slot, left, sum);
    else if (goes_on)
        store4(slot + p.dim, left, sum);
    else
        put_gradient(p, cur, c, sum);
}

constexpr int kClearRows = 8;  // that a group of threads looks at
constexpr int kJoinLanes = 16, kJoinGroups = 256 / kJoinLanes, kJoinColumns = 4 * kJoinLanes;
constexpr int kLongJoin = 16;  // parts that a group adds up by itself

// The rows whose run crosses the end of a chunk: the parts of the chunk where the run starts and of those behind it, added in
// 64 bits (a frequent word has thousands of parts) in an order that depends on their number alone.  A group of 16 threads
// takes 64 columns of a run, up to 16 parts, eight under way together; a longer run is all 16 groups' of the workgroup, every
// 16th part each, whose sums meet in LDS (15920 tokens x 80, 131 parts to the most frequent word: 16 us one after the other,
// 5 us).  The same launch clears the rows that no token has, while the sums wait for memory.
__global__ void __launch_bounds__(256) embedding_join_kernel(const EmbeddingParams p) {
    __shared__ double meet[kJoinGroups][4][kJoinLanes];
    __shared__ int long_runs[kJoinGroups], n_long;
    if (blockIdx.x >= p.join_blocks) {  // rows that no token has, in the order of their keys: neighbours in `offsets`
        const int lane = threadIdx.x & ((1 << p.lanes_log2) - 1), group = threadIdx.x >> p.lanes_log2;
        const int groups = 256 >> p.lanes_log2;
        const unsigned int block = blockIdx.x - p.join_blocks, at_key = block / p.clear_columns;
        const int c = (int)((block - at_key * p.clear_columns) << (p.lanes_log2 + 2)) + 4 * lane;
        if (c >= p.dim) return;
        const int keys = p.sort_blocks * p.bins;
        const long long k0 = ((long long)at_key * groups + group) * kClearRows;
        if (k0 >= keys) return;
        const int first = (int)k0, here = keys - first < kClearRows ? keys - first : kClearRows;
        int at[kClearRows + 1];
#pragma unroll
        for (int k = 0; k <= kClearRows; ++k) at[k] = p.offsets[first + (k < here ? k : here)];
#pragma unroll
        for (int k = 0; k < kClearRows; ++k) {
            const int id = id_of_key(p, first + k);
            if (k < here && at[k] == at[k + 1] && id < p.vocabulary)
                store4(static_cast<float*>(p.out) + (long long)id * p.ld_out + c, p.dim - c, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        }
        return;
    }
    const int lane = threadIdx.x & (kJoinLanes - 1), group = threadIdx.x / kJoinLanes;
    const unsigned int block = blockIdx.x / p.join_columns;
    const int c = (int)(blockIdx.x - block * p.join_columns) * kJoinColumns + 4 * lane, left = p.dim - c;
    const long long k = (long long)block * kJoinGroups + group;
    int key = -1, k_end = 0;
    if (k < p.chunks) key = p.crossing[2 * k], k_end = p.crossing[2 * k + 1];
    if (threadIdx.x == 0) n_long = 0;
    __syncthreads();
    // sum += the parts of chunks q, q + step ... to the last
    auto add_parts = [&](double (&sum)[4], long long q, long long last, int step) {
        constexpr int U = 8;
        for (; q <= last; q += U * step) {
            f32x4 v[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                v[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                if (q + j * step <= last) v[j] = load4(p.partial + 2 * (q + j * step) * p.dim + c, left);
            }
#pragma unroll
            for (int j = 0; j < U; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += v[j][e];
        }
    };
    if (key >= 0 && k_end - k > kLongJoin) {
        if (lane == 0) long_runs[atomicAdd(&n_long, 1)] = group;  // (in any order: their rows have nothing to do with each other)
    } else if (key >= 0 && left > 0) {
        const f32x4 first = load4(p.partial + (2 * k + 1) * p.dim + c, left);
        double sum[4] = {first[0], first[1], first[2], first[3]};
        add_parts(sum, k + 1, k_end, 1);
        put_gradient(p, key, c, f32x4{(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]});
    }
    __syncthreads();
    for (int i = 0; i < n_long; ++i) {
        const long long from = (long long)block * kJoinGroups + long_runs[i];
        const int run_key = p.crossing[2 * from], last = p.crossing[2 * from + 1];
        double sum[4] = {0.0, 0.0, 0.0, 0.0};
        if (left > 0) {
            if (group == 0) {
                const f32x4 first = load4(p.partial + (2 * from + 1) * p.dim + c, left);
                for (int e = 0; e < 4; ++e) sum[e] = first[e];
            }
            add_parts(sum, from + 1 + group, last, kJoinGroups);
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 4; ++e) meet[group][e][lane] = sum[e];
        __syncthreads();
        if (group == 0 && left > 0) {
            for (int g = 1; g < kJoinGroups; ++g)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += meet[g][e][lane];
            put_gradient(p, run_key, c, f32x4{(float)sum[0], (float)sum[1], (float)sum[2], (float)sum[3]});
        }
    }
}

// The whole gradient in one launch, for few tokens (kSmallTokens) and few elements of dy (kSmallElements): the workgroup of a
// bucket sorts its tokens in LDS as embedding_sort_kernel does and goes on to add up the rows of its ids.  A group of threads
// takes an id at a time; ids with more than a group's share of the bucket's tokens (and than kLongRun) are left to all groups
// together, whose sums meet in LDS (1024 x 512 into 32000 rows: 22 us with kLongRun = 32, 18 us with 8).  One workgroup sums a
// frequent word's rows alone, which is what bounds the size (4000 x 100: 19 us in three launches, 11.5 us in one; 2048 x 512
// 23 and 21 us; 2048 x 1024 38 and 49 us).
constexpr int kSmallTokens = 4096, kLongRun = 8, kSmallGroups = 128;  // (most groups of a workgroup: 8 threads each)
constexpr long long kSmallElements = 1LL << 20;

template <typename ID, typename T>
__global__ void __launch_bounds__(1024) embedding_small_kernel(const EmbeddingParams p) {
    extern __shared__ int count[];  // [16][bins], then the cursors; at the end the groups' sums, 16 KB
    __shared__ int wave_total[16], starts[513], long_runs[kSmallGroups], n_long;
    constexpr int PER = kSmallTokens / 1024, U = 8;
    if (threadIdx.x == 0) n_long = 0;
    __shared__ unsigned short notes[16][kSmallTokens / 16], order[kSmallTokens];
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, rank = blockIdx.x, bins = p.bins;
    for (int i = tid; i < 16 * bins; i += 1024) count[i] = 0;
    __syncthreads();
    const int tokens = (int)p.tokens, per = (tokens + 1023) / 1024 * 64;
    const int begin = w * per, end = begin + per < tokens ? begin + per : tokens;
    const ID* ids = static_cast<const ID*>(p.ids);
    int noted = 0, id[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int t = begin + 64 * j + lane;
        id[j] = t < end ? token_id(ids, t, p.vocabulary) : -1;
        if (id[j] == p.padding) id[j] = -1;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const bool mine = id[j] >= 0 && rank_of_id(p, id[j]) == rank;
        const unsigned long long hits = __ballot(mine);
        if (mine) {
            atomicAdd(&count[w * bins + (id[j] >> p.sort_log2)], 1);
            notes[w][noted + __popcll(hits & ((1ULL << lane) - 1))] = (unsigned short)(64 * j + lane);
        }
        noted += __popcll(hits);
    }
    __syncthreads();
    int start, total;
    scan_counts<16>(count, bins, 0, wave_total, start, total);
    const int glane = tid & ((1 << p.lanes_log2) - 1), group = tid >> p.lanes_log2, groups = 1024 >> p.lanes_log2;
    int share = 0;  // of the bucket's tokens: fewer than `groups` runs are longer
#pragma unroll
    for (int k = 0; k < 16; ++k) share += wave_total[k];
    share = share / groups > kLongRun ? share / groups : kLongRun;
    if (tid < bins) {
        starts[tid] = start;
        if (total > share) long_runs[atomicAdd(&n_long, 1)] = tid;  // (in any order: their rows have nothing to do with each other)
    }
    if (tid == bins - 1) starts[bins] = start + total;
    for (int k = 0; k < noted; k += 64) {
        const bool in = k + lane < noted;
        const int t = begin + (in ? notes[w][k + lane] : 0);
        const int number = in ? token_id(ids, t, p.vocabulary) >> p.sort_log2 : 0;
        const int at = take_place(in, number, p.bins_log2, count + w * bins);
        if (in) order[at] = (unsigned short)t;
    }
    __syncthreads();
    f32x4* sums = reinterpret_cast<f32x4*>(count);
    for (int c0 = 0; c0 < p.dim; c0 += 4 << p.lanes_log2) {
        const int c = c0 + 4 * glane, left = p.dim - c;
        const bool ends = __ballot(left < 4) != 0;
        const T* dy = static_cast<const T*>(p.in);
        // rows first, first + step ... of a run
        auto add_up = [&](int first, int last, int step) {
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
            if (left <= 0) return sum;
            for (int q = first; q < last; q += U * step) {
                raw4<T> v[U];
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    v[j] = raw4<T>{};
                    if (q + j * step < last) v[j] = load4_row(dy + (long long)order[q + j * step] * p.ld_in, c, p.dim);
                }
#pragma unroll
                for (int j = 0; j < U; ++j) sum += existing(widen(v[j]), left, ends);
            }
            return sum;
        };
        for (int number = group; number < bins; number += groups) {
            const int a = starts[number], b = starts[number + 1];
            const int row = (number << p.sort_log2) | rank;
            if (b - a > share || row >= p.vocabulary || left <= 0) continue;
            if (b > a)
                put_gradient(p, rank * bins + number, c, add_up(a, b, 1));
            else if (!p.accumulate)
                store4(static_cast<float*>(p.out) + row * p.ld_out + c, left, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
        }
        for (int k = 0; k < n_long; ++k) {
            const int number = long_runs[k], a = starts[number], b = starts[number + 1];
            __syncthreads();
            sums[tid] = add_up(a + group, b, groups);
            __syncthreads();
            if (group == 0 && left > 0) {
                f32x4 sum = sums[glane];
                for (int g = 1; g < groups; ++g) sum += sums[(g << p.lanes_log2) + glane];
                put_gradient(p, rank * bins + number, c, sum);
            }
        }
    }
}

}  // namespace snhip
