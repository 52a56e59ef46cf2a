// The block norm kernels for one combination of storage types, SNHIP_NORM_TYPES = 0, 1 or 2 (block_norm_launch.hpp).
#include "block_norm_launch.hpp"

#ifndef SNHIP_NORM_TYPES
#error "compile with -DSNHIP_NORM_TYPES=0..2"
#endif

namespace snhip {

#if SNHIP_NORM_TYPES == 0
typedef float Stream;
typedef float Block;
#define SNHIP_FORWARD block_norm_forward_0
#define SNHIP_BACKWARD block_norm_backward_0
#elif SNHIP_NORM_TYPES == 1
typedef float Stream;
typedef __bf16 Block;
#define SNHIP_FORWARD block_norm_forward_1
#define SNHIP_BACKWARD block_norm_backward_1
#else
typedef __bf16 Stream;
typedef __bf16 Block;
#define SNHIP_FORWARD block_norm_forward_2
#define SNHIP_BACKWARD block_norm_backward_2
#endif

namespace {

template <int TPR, int N>
void forward(const BlockNormParams& p, hipStream_t stream) {
    constexpr int NT = TPR > 256 ? TPR : 256, GROUPS = NT / TPR;
    const dim3 grid = many_blocks((p.rows + GROUPS - 1) / GROUPS);
    if (p.exact)
        hipLaunchKernelGGL((block_norm_forward_kernel<Stream, Block, TPR, N, true>), grid, dim3(NT), 0, stream, p);
    else
        hipLaunchKernelGGL((block_norm_forward_kernel<Stream, Block, TPR, N, false>), grid, dim3(NT), 0, stream, p);
}

template <int TPR, int N, int MODE, bool BIAS, bool GATE>
void backward(const BlockNormParams& p, hipStream_t stream) {
    constexpr int NT = TPR > 256 ? TPR : 256;
    const dim3 grid((unsigned)p.chunks);
    if constexpr (TPR != 256 || N != 1)  // (those are rows of another width than a multiple of four)
        if (p.exact) {
            hipLaunchKernelGGL((block_norm_backward_kernel<Stream, Block, TPR, N, MODE, BIAS, GATE, true>), grid, dim3(NT), 0, stream, p);
            return;
        }
    hipLaunchKernelGGL((block_norm_backward_kernel<Stream, Block, TPR, N, MODE, BIAS, GATE, false>), grid, dim3(NT), 0, stream, p);
}

template <int TPR, int N>
void backward_kind(const BlockNormParams& p, BlockNormKind k, hipStream_t stream) {
    if (k.mode == 0)
        k.bias ? backward<TPR, N, 0, true, false>(p, stream) : backward<TPR, N, 0, false, false>(p, stream);
    else if (k.mode == 1 && k.gate)
        k.bias ? backward<TPR, N, 1, true, true>(p, stream) : backward<TPR, N, 1, false, true>(p, stream);
    else if (k.mode == 1)
        k.bias ? backward<TPR, N, 1, true, false>(p, stream) : backward<TPR, N, 1, false, false>(p, stream);
    else if (k.gate)
        k.bias ? backward<TPR, N, 2, true, true>(p, stream) : backward<TPR, N, 2, false, true>(p, stream);
    else
        k.bias ? backward<TPR, N, 2, true, false>(p, stream) : backward<TPR, N, 2, false, false>(p, stream);
}

}  // namespace

// A row of up to 1024 elements is one wavefront's or less (no barrier), a longer one a workgroup's: 16384 x 1024 bf16 31 us, with
// 256 threads to a row 34; 16384 x 2048 57 us, with a wavefront to a row 66, with 1024 threads 118.  As many pieces to a thread as
// the row needs: what lies behind it costs time, too (6000 x 5120 with five pieces 58 us, with eight 79).  With few rows to go
// round a row is spread over as many threads as it has pieces of four: 8 x 1024 3.2 us instead of 4.0, 256 x 4096 4.4 instead
// of 5.2; rows of 513 to 1024 elements keep that up to 4096 of them (1024 x 1024: 4.1 us instead of 4.9; 4096 x 1024 9.4
// instead of 9.8).
void SNHIP_FORWARD(const BlockNormParams& p, hipStream_t stream) {
    const int units = (p.dim + 3) / 4;
    if (units <= 16) return forward<16, 1>(p, stream);
    if (units <= 32) return forward<32, 1>(p, stream);
    if (units <= 64) return forward<64, 1>(p, stream);
    if (p.rows <= 512) {
        if (units <= 256) return forward<256, 1>(p, stream);
        if (units <= 1024) return forward<1024, 1>(p, stream);
        return forward<1024, 2>(p, stream);
    }
    if (units <= 128) return forward<64, 2>(p, stream);
    if (units <= 256 && p.rows <= 4096) return forward<256, 1>(p, stream);
    if (units <= 192) return forward<64, 3>(p, stream);
    if (units <= 256) return forward<64, 4>(p, stream);
    if (units <= 512) return forward<256, 2>(p, stream);
    if (units <= 768) return forward<256, 3>(p, stream);
    if (units <= 1024) return forward<256, 4>(p, stream);
    if (units <= 1280) return forward<256, 5>(p, stream);
    if (units <= 1536) return forward<256, 6>(p, stream);
    forward<256, 8>(p, stream);
}

// A row of up to 1024 elements is one wavefront's or less, as above (32 threads to rows of up to 128: 30000 x 128 bf16 19 us, with 16
// and two pieces 23; 16384 x 768 with three pieces 46 us, with 256 threads to a row 57; 16384 x 1024 55 and 60 us), but not with
// four pieces and ends to look at, which take too many registers (8000 x 1001 fp32: 78 us, 256 threads 59).  Beyond that two
// pieces to a thread leave registers for the column sums.  (The groups of threads per workgroup: block_norm_backward_groups.)
void SNHIP_BACKWARD(const BlockNormParams& p, BlockNormKind kind, hipStream_t stream) {
    const int units = (p.dim + 3) / 4;
    if (units <= 16) return backward_kind<16, 1>(p, kind, stream);
    if (units <= 32) return backward_kind<32, 1>(p, kind, stream);
    if (units <= 64) return backward_kind<64, 1>(p, kind, stream);
    if (units <= 128) return backward_kind<64, 2>(p, kind, stream);
    if (units <= 192) return backward_kind<64, 3>(p, kind, stream);
    if (units <= 256 && p.dim % 4 == 0) return backward_kind<64, 4>(p, kind, stream);
    if (units <= 256) return backward_kind<256, 1>(p, kind, stream);
    if (units <= 512) return backward_kind<256, 2>(p, kind, stream);
    if (units <= 1024) return backward_kind<512, 2>(p, kind, stream);
    backward_kind<1024, 2>(p, kind, stream);
}

}  // namespace snhip
