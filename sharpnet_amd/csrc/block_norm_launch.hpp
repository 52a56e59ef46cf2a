// Launch functions of the block norm kernels, one pair per combination of storage types (block_norm.hip is compiled once
// for each, side by side), and what the entry points need to know about their shapes.
#pragma once
#include <hip/hip_runtime.h>

#include "block_norm.hpp"

namespace snhip {

constexpr int kBlockNormMaxDim = 8192;

// Rows that a workgroup of the backward kernel holds at a time.
inline int block_norm_backward_groups(int dim) { return dim <= 64 ? 16 : dim <= 128 ? 8 : dim <= 768 || (dim <= 1024 && dim % 4 == 0) ? 4 : 1; }

// mode, bias, gate: the template parameters of block_norm_backward_kernel
struct BlockNormKind {
    int mode;
    bool bias, gate;
};

// 0: stream and block fp32, 1: fp32 stream, bf16 block, 2: both bf16
void block_norm_forward_0(const BlockNormParams& p, hipStream_t stream);
void block_norm_forward_1(const BlockNormParams& p, hipStream_t stream);
void block_norm_forward_2(const BlockNormParams& p, hipStream_t stream);
void block_norm_backward_0(const BlockNormParams& p, BlockNormKind kind, hipStream_t stream);
void block_norm_backward_1(const BlockNormParams& p, BlockNormKind kind, hipStream_t stream);
void block_norm_backward_2(const BlockNormParams& p, BlockNormKind kind, hipStream_t stream);

}  // namespace snhip
