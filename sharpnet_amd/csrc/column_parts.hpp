// The second half of the block norms' column sums: the chunks' sums in their order.  Belongs to one translation unit.
#pragma once
#include <hip/hip_runtime.h>

namespace snhip {

__global__ void __launch_bounds__(256) clear_vector_kernel(float* dst, int count) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < count) dst[i] = 0.0f;
}

// Adds up chunks' column sums: job y of the launch is the sum of `count` consecutive rows of `dim` floats at `in`.  A
// workgroup owns 64 columns, its 16 wavefronts every 16th row each, four in flight; they meet in LDS in a fixed order.
struct ColumnJobs {
    const float* partial;
    float* out[4];       // the first `vectors` jobs: one slot of `partial` each, all chunks
    int slot[5];         // their slots; [4]: the gate's
    int vectors, chunks, dim;
    int chunks_per_group;  // the jobs behind them: one group of gate rows each
    void* gate_out;
    long long ld_gate;
    int gate_bf16, accumulate, accumulate_gate;
};
__global__ void __launch_bounds__(1024) column_parts_kernel(const ColumnJobs j) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane, job = blockIdx.y;
    const bool is_gate = job >= j.vectors;
    const long long first = is_gate ? (long long)j.slot[4] * j.chunks + (long long)(job - j.vectors) * j.chunks_per_group
                                    : (long long)j.slot[job] * j.chunks;
    const int count = is_gate ? j.chunks_per_group : j.chunks;
    float s0 = 0.0f, s1 = 0.0f, s2 = 0.0f, s3 = 0.0f;
    if (c < j.dim) {
        const float* in = j.partial + first * j.dim + c;
        int k = w;
        for (; k + 48 < count; k += 64) {
            s0 += in[(long long)k * j.dim];
            s1 += in[(long long)(k + 16) * j.dim];
            s2 += in[(long long)(k + 32) * j.dim];
            s3 += in[(long long)(k + 48) * j.dim];
        }
        for (; k < count; k += 16) s0 += in[(long long)k * j.dim];
    }
    part[w][lane] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    if (w != 0 || c >= j.dim) return;
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += part[k][lane];
    if (!is_gate) {
        float* out = j.out[job] + c;
        *out = j.accumulate ? *out + s : s;
    } else if (j.gate_bf16) {
        static_cast<__bf16*>(j.gate_out)[(job - j.vectors) * j.ld_gate + c] = (__bf16)s;
    } else {
        float* out = static_cast<float*>(j.gate_out) + (job - j.vectors) * j.ld_gate + c;
        *out = j.accumulate_gate ? *out + s : s;
    }
}

}  // namespace snhip
