// The second half of the block norms' column sums: the chunks' sums in their order.  Belongs to one translation unit.
#pragma once
#include <hip/hip_runtime.h>

namespace snhip {

__global__ void __launch_bounds__(256) clear_vector_kernel(float* dst, int count) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < count) dst[i] = 0.0f;
}

// Adds up chunks' column sums: job y of the launch is the sum of `count` consecutive rows of `dim` floats at `in`.  A
// workgroup owns 32 columns, its 32 groups of 32 threads every 32nd row each, eight in flight; they meet in LDS in a fixed
// order.  Bound by the way to memory and back (64 columns to a workgroup, so half of the workgroups, and 16 wavefronts with four
// rows in flight: 4.8 us for three vectors of 512 rows of 512, now 3.4; two vectors of 512 rows of 4096 7.1 us, now 5.7).
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
    __shared__ float part[32][33];
    const int col = threadIdx.x & 31, r = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + col, job = blockIdx.y;
    const bool is_gate = job >= j.vectors;
    const long long first = is_gate ? (long long)j.slot[4] * j.chunks + (long long)(job - j.vectors) * j.chunks_per_group
                                    : (long long)j.slot[job] * j.chunks;
    const int count = is_gate ? j.chunks_per_group : j.chunks;
    float s[8] = {};
    if (c < j.dim) {
        const float* in = j.partial + first * j.dim + c;
        int k = r;
        for (; k + 224 < count; k += 256) {
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += in[(long long)(k + 32 * i) * j.dim];
        }
        for (; k < count; k += 32) s[0] += in[(long long)k * j.dim];
    }
    part[r][col] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    __syncthreads();
    if (threadIdx.x >= 64) return;  // half of the groups to each 32 threads of the first wavefront
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) sum += part[16 * r + k][col];
    sum += __shfl_xor(sum, 32, 64);
    if (r != 0 || c >= j.dim) return;
    if (!is_gate) {
        float* out = j.out[job] + c;
        *out = j.accumulate ? *out + sum : sum;
    } else if (j.gate_bf16) {
        static_cast<__bf16*>(j.gate_out)[(job - j.vectors) * j.ld_gate + c] = (__bf16)sum;
    } else {
        float* out = static_cast<float*>(j.gate_out) + (job - j.vectors) * j.ld_gate + c;
        *out = j.accumulate_gate ? *out + sum : sum;
    }
}

}  // namespace snhip
