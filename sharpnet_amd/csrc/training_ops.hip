// C ABI of the operators around the Dense, attention and recurrent layers in a training step: argument checks, choice of
// launch shape, launches.  Declarations are in include/sharpnet_hip.h.
#include "../../include/sharpnet_hip.h"

#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <memory>
#include <new>
#include <vector>

#include "adamw.hpp"
#include "block_norm_launch.hpp"
#include "column_parts.hpp"
#include "embedding.hpp"
#include "handle.hpp"

using namespace snhip;

namespace {

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool is_storage_type(int type) { return type == SNHIP_TYPE_F32 || type == SNHIP_TYPE_BF16; }
size_t type_bytes(int type) { return type == SNHIP_TYPE_BF16 ? 2 : type == SNHIP_TYPE_I64 ? 8 : 4; }
size_t up256(size_t bytes) { return (bytes + 255) / 256 * 256; }

// ---- word embedding ------------------------------------------------------------------------------------------

int embedding_check_desc(const snhip_embedding_desc* d) {
    if (d == nullptr || d->struct_size != (int)sizeof(snhip_embedding_desc)) return SNHIP_STATUS_INVALID_VALUE;
    if (d->id_type != SNHIP_TYPE_F32 && d->id_type != SNHIP_TYPE_I32 && d->id_type != SNHIP_TYPE_I64)
        return SNHIP_STATUS_INVALID_VALUE;
    if (!is_storage_type(d->table_type) || !is_storage_type(d->output_type)) return SNHIP_STATUS_INVALID_VALUE;
    if (d->tokens < 0 || d->vocabulary < 0 || d->dim < 0 || d->padding_index < -1) return SNHIP_STATUS_INVALID_VALUE;
    if ((d->ld_table != 0 && d->ld_table < d->dim) || (d->ld_output != 0 && d->ld_output < d->dim))
        return SNHIP_STATUS_INVALID_VALUE;
    // token numbers, the places in the sorted order and the ids' keys in it are 32-bit integers
    if (d->tokens > 0x7fff0000LL || d->vocabulary > 0x3fffffff) return SNHIP_STATUS_NOT_SUPPORTED;
    return SNHIP_STATUS_SUCCESS;
}

EmbeddingParams embedding_params(const snhip_embedding_desc* d, const void* ids, const void* in, void* out, bool backward) {
    EmbeddingParams p{};
    p.ids = ids, p.in = in, p.out = out;
    p.tokens = d->tokens, p.vocabulary = d->vocabulary, p.dim = d->dim, p.scale = d->scale;
    const long long ldt = d->ld_table != 0 ? d->ld_table : d->dim, ldo = d->ld_output != 0 ? d->ld_output : d->dim;
    p.ld_in = backward ? ldo : ldt, p.ld_out = backward ? ldt : ldo;
    p.padding = backward && d->padding_index < d->vocabulary ? d->padding_index : -1;
    const int units = ceil_div(d->dim, 4);
    p.lanes_log2 = 3;
    while (p.lanes_log2 < 8 && (1 << p.lanes_log2) < units) ++p.lanes_log2;
    return p;
}

struct EmbeddingPlan {
    bool small;  // embedding_small_kernel: no workspace
    int sort_blocks, sort_log2, fine_log2, bins, bins_log2, chunk, pieces;
    long long chunks;
    size_t order, sorted, offsets, piece_id, piece_token, piece_start, crossing, partial, bytes;  // places in the workspace
};
EmbeddingPlan embedding_plan(const snhip_embedding_desc* d) {
    EmbeddingPlan e{};
    // a workgroup of the sort per compute unit, more where it would get over 512 ids
    e.sort_log2 = 0;
    while ((1LL << e.sort_log2) < d->vocabulary && (e.sort_log2 < 8 || (512LL << e.sort_log2) < d->vocabulary)) ++e.sort_log2;
    e.sort_blocks = 1 << e.sort_log2;
    e.fine_log2 = e.sort_log2 > 8 ? e.sort_log2 - 8 : 0;
    e.pieces = d->tokens > kSortDirect ? (int)((d->tokens + kPiece - 1) / kPiece) : 0;
    e.bins = (int)(((long long)d->vocabulary + e.sort_blocks - 1) >> e.sort_log2);
    if (e.bins < 1) e.bins = 1;
    while ((1 << e.bins_log2) < e.bins) ++e.bins_log2;
    e.small = d->tokens <= kSmallTokens && d->tokens * d->dim <= kSmallElements && e.fine_log2 == 0;
    if (e.small) return e;
    // short chunks for few tokens (more threads at work), long ones for many (fewer parts of frequent words to join): 8192 x
    // 512 28 us and 65536 x 512 95 us with chunks of 8, 30 and 60 us with 32
    e.chunk = d->tokens >= 16384 ? 32 : 8;
    e.chunks = (d->tokens + e.chunk - 1) / e.chunk;
    e.order = 0;
    e.sorted = e.order + up256((size_t)d->tokens * 4);
    e.offsets = e.sorted + up256((size_t)d->tokens * 4);
    e.piece_id = e.offsets + up256(((size_t)e.sort_blocks * e.bins + 1) * 4);
    e.piece_token = e.piece_id + up256((size_t)e.pieces * kPiece * 4);
    e.piece_start = e.piece_token + up256((size_t)e.pieces * kPiece * 4);
    e.crossing = e.piece_start + up256((size_t)e.pieces * (kBuckets + 1) * 4);
    e.partial = e.crossing + up256((size_t)e.chunks * 8);
    e.bytes = e.partial + up256((size_t)e.chunks * 2 * (size_t)d->dim * 4);
    return e;
}

template <typename ID, typename TIN, typename TOUT>
void embedding_forward_launch(const EmbeddingParams& p, hipStream_t stream) {
    constexpr int ROWS = 4;
    const int groups = 256 >> p.lanes_log2;
    const long long blocks = (p.tokens + (long long)groups * ROWS - 1) / ((long long)groups * ROWS);
    hipLaunchKernelGGL((embedding_forward_kernel<ID, TIN, TOUT, ROWS>),
                       many_blocks(blocks, (unsigned)ceil_div(ceil_div(p.dim, 4), 1 << p.lanes_log2)), dim3(256), 0, stream, p);
}
template <typename ID>
void embedding_forward_types(const EmbeddingParams& p, int table_type, int output_type, hipStream_t stream) {
    const bool tb = table_type == SNHIP_TYPE_BF16, ob = output_type == SNHIP_TYPE_BF16;
    if (tb && ob)
        embedding_forward_launch<ID, __bf16, __bf16>(p, stream);
    else if (tb)
        embedding_forward_launch<ID, __bf16, float>(p, stream);
    else if (ob)
        embedding_forward_launch<ID, float, __bf16>(p, stream);
    else
        embedding_forward_launch<ID, float, float>(p, stream);
}

template <typename ID>
void embedding_small_launch(const EmbeddingParams& p, int type, dim3 grid, size_t lds, hipStream_t stream) {
    lds = std::max(lds, (size_t)1024 * sizeof(f32x4));
    if (type == SNHIP_TYPE_BF16)
        hipLaunchKernelGGL((embedding_small_kernel<ID, __bf16>), grid, dim3(1024), lds, stream, p);
    else
        hipLaunchKernelGGL((embedding_small_kernel<ID, float>), grid, dim3(1024), lds, stream, p);
}

template <typename ID>
void embedding_sort_launch(const EmbeddingParams& p, dim3 grid, size_t lds, hipStream_t stream) {
    if (p.pieces == 0) {
        hipLaunchKernelGGL(embedding_sort_kernel<ID>, grid, dim3(1024), lds, stream, p);
    } else {
        hipLaunchKernelGGL(embedding_bucket_kernel<ID>, dim3((unsigned)p.pieces), dim3(256), 0, stream, p);
        hipLaunchKernelGGL(embedding_sort_pieces_kernel, grid, dim3(1024), lds, stream, p);
    }
}

// ---- block norm ----------------------------------------------------------------------------------------------

int block_norm_check_desc(const snhip_block_norm_desc* d, bool backward) {
    if (d == nullptr || d->struct_size != (int)sizeof(snhip_block_norm_desc)) return SNHIP_STATUS_INVALID_VALUE;
    if (!is_storage_type(d->stream_type) || !is_storage_type(d->block_type)) return SNHIP_STATUS_INVALID_VALUE;
    if (d->pre_norm < SNHIP_NORM_NONE || d->pre_norm > SNHIP_NORM_LAYER || d->post_norm < SNHIP_NORM_NONE ||
        d->post_norm > SNHIP_NORM_LAYER)
        return SNHIP_STATUS_INVALID_VALUE;
    if (d->gate_activation != SNHIP_ACT_NONE && d->gate_activation != SNHIP_ACT_SIGMOID && d->gate_activation != SNHIP_ACT_TANH)
        return SNHIP_STATUS_NOT_SUPPORTED;
    if (d->rows < 0 || d->dim < 0 || d->gate_rows < 0) return SNHIP_STATUS_INVALID_VALUE;
    const long long lds[] = {d->ld_x, d->ld_y, d->ld_u, d->ld_h, d->ld_gate};
    for (long long ld : lds)
        if (ld != 0 && ld < d->dim) return SNHIP_STATUS_INVALID_VALUE;
    if (!(d->epsilon >= 0.0f) || !(d->epsilon < INFINITY)) return SNHIP_STATUS_INVALID_VALUE;
    // a gate or a norm behind the block without a block; nothing to compute
    if (d->y == nullptr && (d->gate != nullptr || d->post_norm != SNHIP_NORM_NONE || d->pre_norm == SNHIP_NORM_NONE))
        return SNHIP_STATUS_INVALID_VALUE;
    if (d->dim > kBlockNormMaxDim || d->rows > 0x7fffffffLL) return SNHIP_STATUS_NOT_SUPPORTED;
    if (d->stream_type == SNHIP_TYPE_BF16 && d->block_type == SNHIP_TYPE_F32) return SNHIP_STATUS_NOT_SUPPORTED;
    const size_t sb = type_bytes(d->stream_type), bb = type_bytes(d->block_type), gb = d->gate_rows == 0 ? 4 : bb;
    const void* streams[] = {d->x, d->u, d->du, d->dx};
    const void* blocks[] = {d->y, d->h, d->dh, d->dy};
    const void* floats[] = {d->pre_weight, d->pre_bias, d->post_weight, d->post_bias, d->pre_statistics, d->post_statistics,
                            d->d_pre_weight, d->d_pre_bias, d->d_post_weight, d->d_post_bias};
    for (const void* p : streams)
        if (!aligned(p, sb)) return SNHIP_STATUS_INVALID_VALUE;
    for (const void* p : blocks)
        if (!aligned(p, bb)) return SNHIP_STATUS_INVALID_VALUE;
    for (const void* p : floats)
        if (!aligned(p, 4)) return SNHIP_STATUS_INVALID_VALUE;
    if (!aligned(d->gate, gb) || !aligned(d->d_gate, gb)) return SNHIP_STATUS_INVALID_VALUE;
    if (d->rows == 0 || d->dim == 0) return SNHIP_STATUS_SUCCESS;
    if (!backward) {
        if (d->x == nullptr || (d->y != nullptr && d->u == nullptr) || (d->pre_norm != SNHIP_NORM_NONE && d->h == nullptr))
            return SNHIP_STATUS_INVALID_VALUE;
        return SNHIP_STATUS_SUCCESS;
    }
    if (d->dx == nullptr || (d->y != nullptr && d->dy == nullptr) || (d->du == nullptr && d->dh == nullptr))
        return SNHIP_STATUS_INVALID_VALUE;
    if (d->pre_norm == SNHIP_NORM_NONE && d->dh != nullptr) return SNHIP_STATUS_INVALID_VALUE;
    if (d->dh != nullptr && (d->u == nullptr || d->pre_statistics == nullptr)) return SNHIP_STATUS_INVALID_VALUE;
    if (d->post_norm != SNHIP_NORM_NONE && d->post_statistics == nullptr) return SNHIP_STATUS_INVALID_VALUE;
    if (d->gate == nullptr && d->d_gate != nullptr) return SNHIP_STATUS_INVALID_VALUE;
    return SNHIP_STATUS_SUCCESS;
}

struct BlockNormPlan {
    int slots[5];       // pre weight, pre bias, post weight, post bias, gate: their vector of partial sums, or -1
    int vectors;
    bool flush;
    long long groups, rows_per_group;
    int groups_per_chunk, chunks_per_group, rows_per_chunk, chunks;
    size_t bytes;
};
// How the rows are cut into chunks, one workgroup each: as many as the compute units hold at a time.  More would only add
// column sums on their way to memory and back (16384 x 4096, two vectors: 1024 chunks 13 us for them, 512 8 us, before they took
// 5.7); with few rows fewer are enough.
long long block_norm_chunks(const snhip_block_norm_desc* d) {
    const bool gated = d->gate != nullptr, normed = d->post_norm != SNHIP_NORM_NONE, narrow = d->stream_type == SNHIP_TYPE_BF16;
    // 16 wavefronts: one of a compute unit, two of the smallest kind (4096 x 8192 bf16: 512 chunks 131 us, 256 124 us; the norm
    // alone 6000 x 5120 71 us and 79 us)
    if (d->dim > 4096) return gated || normed || !narrow ? 256 : 512;
    if (d->dim > 2048) return 512;
    if (d->dim <= 256) return 1024;
    if (d->dim > 512 && d->dim <= 1024) return block_norm_backward_groups(d->dim) > 1 ? 512 : 1024;
    // Two pieces to a thread: four of a compute unit, or three with a gate and a norm to undo (12000 x 1280 bf16: 512 chunks 88
    // us, 1024 71 us; fp32 768 92 us instead of 101 us; 20000 x 300 fp32 1024 chunks 52 us, 512 45 us), if that leaves eight
    // turns to each (2048 x 2048 fp32: 512 chunks 29 us, 1024 33 us).
    const bool three = gated && normed && (!narrow || d->dim % 4 != 0);
    if (d->dim <= 512 && !three) return 1024;
    const long long most = three ? 768 : 1024;
    return d->rows >= 8 * most * block_norm_backward_groups(d->dim) ? most : 512;
}
BlockNormPlan block_norm_plan(const snhip_block_norm_desc* d) {
    BlockNormPlan b{};
    const bool gate_rows = d->gate != nullptr && d->gate_rows > 0;
    b.rows_per_group = gate_rows && d->gate_rows < d->rows ? d->gate_rows : d->rows;
    if (b.rows_per_group < 1) b.rows_per_group = 1;
    b.groups = (d->rows + b.rows_per_group - 1) / b.rows_per_group;
    const int at_once = block_norm_backward_groups(d->dim);
    const long long wanted = block_norm_chunks(d);
    long long c = (d->rows + wanted - 1) / wanted;
    // (a turn each would give the column sums more to do than the rows: 1024 x 1024 bf16 13.2 us, two turns 11.8)
    const int least = d->rows > 512LL * at_once ? 2 * at_once : at_once;
    if (c < least) c = least;
    b.flush = gate_rows && b.rows_per_group <= c;
    if (b.flush) {
        b.groups_per_chunk = (int)((c / b.rows_per_group + at_once - 1) / at_once * at_once);
        b.chunks = (int)((b.groups + b.groups_per_chunk - 1) / b.groups_per_chunk);
    } else if (d->rows > 0) {
        b.chunks_per_group = (int)((b.rows_per_group + c - 1) / c);
        b.rows_per_chunk = (int)((b.rows_per_group + b.chunks_per_group - 1) / b.chunks_per_group);
        b.chunks = (int)(b.groups * b.chunks_per_group);
    }
    const bool sums[5] = {d->d_pre_weight != nullptr && d->dh != nullptr, d->d_pre_bias != nullptr && d->dh != nullptr,
                            d->d_post_weight != nullptr && d->post_norm != SNHIP_NORM_NONE,
                            d->d_post_bias != nullptr && d->post_norm != SNHIP_NORM_NONE, d->d_gate != nullptr && !b.flush};
    for (int k = 0; k < 5; ++k) b.slots[k] = sums[k] ? b.vectors++ : -1;
    b.bytes = up256((size_t)b.vectors * (size_t)b.chunks * (size_t)d->dim * 4);
    return b;
}

BlockNormParams block_norm_params(const snhip_block_norm_desc* d) {
    BlockNormParams p{};
    p.x = d->x, p.y = d->y, p.gate = d->gate, p.u = d->u, p.h = d->h;
    p.pre_w = d->pre_weight, p.pre_b = d->pre_bias, p.post_w = d->post_weight, p.post_b = d->post_bias;
    p.pre_s = d->pre_statistics, p.post_s = d->post_statistics;
    p.du = d->du, p.dh = d->dh, p.dx = d->dx, p.dy = d->dy, p.d_gate = d->d_gate;
    p.rows = d->rows, p.dim = d->dim, p.gate_rows = d->gate_rows;
    p.ld_x = d->ld_x ? d->ld_x : d->dim, p.ld_y = d->ld_y ? d->ld_y : d->dim, p.ld_u = d->ld_u ? d->ld_u : d->dim;
    p.ld_h = d->ld_h ? d->ld_h : d->dim, p.ld_gate = d->ld_gate ? d->ld_gate : d->dim;
    p.pre = d->pre_norm, p.post = d->post_norm, p.act = d->gate_activation;
    p.eps = d->epsilon, p.scale = d->residual_scale, p.inv_dim = 1.0f / (float)(d->dim > 0 ? d->dim : 1);
    // four bf16 in one access need a 4-byte address; fp32 rows always have one
    const bool block_ok = d->block_type == SNHIP_TYPE_F32 ||
                          (p.ld_y % 2 == 0 && p.ld_h % 2 == 0 && p.ld_gate % 2 == 0 && aligned(d->y, 4) && aligned(d->h, 4) &&
                           aligned(d->dh, 4) && aligned(d->dy, 4) && aligned(d->gate, 4) && aligned(d->d_gate, 4));
    const bool stream_ok = d->stream_type == SNHIP_TYPE_F32 || (p.ld_x % 2 == 0 && p.ld_u % 2 == 0 && aligned(d->x, 4) &&
                                                                aligned(d->u, 4) && aligned(d->du, 4) && aligned(d->dx, 4));
    p.exact = p.dim % 4 == 0 && block_ok && stream_ok;
    return p;
}

// 0: both fp32, 1: fp32 stream and bf16 block, 2: both bf16
int block_norm_types(const snhip_block_norm_desc* d) {
    return d->stream_type == SNHIP_TYPE_BF16 ? 2 : d->block_type == SNHIP_TYPE_BF16 ? 1 : 0;
}

// ---- AdamW ------------------------------------------------------------------------------------------------------

struct AdamwPlan {
    int device = 0, state_bits = 32;
    long long chunks = 0;
    bool once = false;  // kAdamwOnce elements or more
    void* table = nullptr;  // entries, then the owner of each chunk
    const int* owner = nullptr;
};

constexpr long long kAdamwMaxChunks = 0x7fffffff;  // their numbers are 32-bit integers

struct Range {
    uintptr_t begin, end;
    bool written;
};
// whether a written range meets any other one
bool overlapping(std::vector<Range>& ranges) {
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    uintptr_t end = 0, written_end = 0;
    for (const Range& r : ranges) {
        if (r.begin < (r.written ? end : written_end)) return true;
        end = std::max(end, r.end);
        if (r.written) written_end = std::max(written_end, r.end);
    }
    return false;
}

int adamw_build(Handle* h, const snhip_adamw_tensor* tensors, int count, int state_bits, void** plan) {
    std::vector<AdamwEntry> entries((size_t)count);
    std::vector<Range> ranges;
    long long elements = 0, chunks = 0;
    const size_t sb = state_bits == 32 ? 4 : 1;
    for (int k = 0; k < count; ++k) {
        const snhip_adamw_tensor& t = tensors[k];
        if (t.count < 0 || !is_storage_type(t.gradient_type) || !isfinite(t.weight_decay)) return SNHIP_STATUS_INVALID_VALUE;
        AdamwEntry& e = entries[(size_t)k];
        e = AdamwEntry{t.parameter, t.gradient, t.moment1, t.moment2, t.scale1, t.scale2, static_cast<__bf16*>(t.bf16_copy),
                       t.count, 0, t.weight_decay, t.gradient_type == SNHIP_TYPE_BF16};
        if (t.count == 0) continue;
        if (t.count > kAdamwMaxChunks * kAdamwChunk) return SNHIP_STATUS_NOT_SUPPORTED;
        e.first_chunk = chunks;
        chunks += (t.count + kAdamwChunk - 1) / kAdamwChunk;
        if (chunks > kAdamwMaxChunks) return SNHIP_STATUS_NOT_SUPPORTED;
        const size_t gb = type_bytes(t.gradient_type);
        if (t.parameter == nullptr || t.gradient == nullptr || t.moment1 == nullptr || t.moment2 == nullptr ||
            (state_bits == 8 && (t.scale1 == nullptr || t.scale2 == nullptr)))
            return SNHIP_STATUS_INVALID_VALUE;
        if (!aligned(t.parameter, 4) || !aligned(t.gradient, gb) || !aligned(t.moment1, sb) || !aligned(t.moment2, sb) ||
            !aligned(t.bf16_copy, 2))
            return SNHIP_STATUS_INVALID_VALUE;
        const size_t n = (size_t)t.count, blocks = (n + kAdamwBlock - 1) / kAdamwBlock;
        auto add = [&ranges](const void* p, size_t bytes, bool written) {
            const uintptr_t b = reinterpret_cast<uintptr_t>(p);
            if (p != nullptr) ranges.push_back(Range{b, b + bytes, written});
        };
        add(t.parameter, 4 * n, true);
        add(t.moment1, sb * n, true);
        add(t.moment2, sb * n, true);
        add(t.bf16_copy, 2 * n, true);
        if (state_bits == 8) add(t.scale1, blocks, true), add(t.scale2, blocks, true);
        add(t.gradient, gb * n, false);
        elements += t.count;
    }
    if (overlapping(ranges)) return SNHIP_STATUS_INVALID_VALUE;
    DeviceScope scope(h->device);
    if (!scope.ok()) return SNHIP_STATUS_NOT_INITIALIZED;
    std::vector<int> owner((size_t)chunks);
    for (int k = 0; k < count; ++k) {
        const long long n = (entries[(size_t)k].count + kAdamwChunk - 1) / kAdamwChunk;
        std::fill_n(owner.begin() + entries[(size_t)k].first_chunk, n, k);
    }
    std::unique_ptr<AdamwPlan> a(new AdamwPlan);
    a->device = h->device, a->state_bits = state_bits, a->chunks = chunks, a->once = elements >= kAdamwOnce;
    if (chunks > 0) {
        const size_t entry_bytes = up256(entries.size() * sizeof(AdamwEntry));
        hipError_t e = hipMalloc(&a->table, entry_bytes + owner.size() * sizeof(int));
        if (e == hipSuccess) e = hipMemcpy(a->table, entries.data(), entries.size() * sizeof(AdamwEntry), hipMemcpyHostToDevice);
        if (e == hipSuccess)
            e = hipMemcpy(static_cast<char*>(a->table) + entry_bytes, owner.data(), owner.size() * sizeof(int), hipMemcpyHostToDevice);
        if (e != hipSuccess) {
            (void)hipGetLastError();
            if (a->table != nullptr) (void)hipFree(a->table);
            return hip_to_status(e);
        }
        a->owner = reinterpret_cast<const int*>(static_cast<char*>(a->table) + entry_bytes);
    }
    *plan = a.release();
    return SNHIP_STATUS_SUCCESS;
}

}  // namespace

extern "C" {

int snhip_sizeof_embedding_desc(void) { return (int)sizeof(snhip_embedding_desc); }

int snhip_embedding_forward(void* handle, const snhip_embedding_desc* desc, const void* ids, const void* table, void* y) {
    const int st = embedding_check_desc(desc);
    if (st != SNHIP_STATUS_SUCCESS) return st;
    Handle* h = static_cast<Handle*>(handle);
    if (h == nullptr) return SNHIP_STATUS_NOT_INITIALIZED;
    if (desc->tokens == 0 || desc->dim == 0) return SNHIP_STATUS_SUCCESS;
    if (ids == nullptr || y == nullptr || (table == nullptr && desc->vocabulary > 0)) return SNHIP_STATUS_INVALID_VALUE;
    if (!aligned(ids, type_bytes(desc->id_type)) || !aligned(table, type_bytes(desc->table_type)) ||
        !aligned(y, type_bytes(desc->output_type)))
        return SNHIP_STATUS_INVALID_VALUE;
    DeviceScope scope(h->device);
    if (!scope.ok()) return SNHIP_STATUS_NOT_INITIALIZED;
    const EmbeddingParams p = embedding_params(desc, ids, table, y, false);
    if (ceil_div(ceil_div(p.dim, 4), 1 << p.lanes_log2) > 65535) return SNHIP_STATUS_NOT_SUPPORTED;
    if (desc->id_type == SNHIP_TYPE_F32)
        embedding_forward_types<float>(p, desc->table_type, desc->output_type, h->stream);
    else if (desc->id_type == SNHIP_TYPE_I32)
        embedding_forward_types<int>(p, desc->table_type, desc->output_type, h->stream);
    else
        embedding_forward_types<long long>(p, desc->table_type, desc->output_type, h->stream);
    return hip_to_status(hipGetLastError());
}

int snhip_embedding_backward_workspace_size(const snhip_embedding_desc* desc, size_t* bytes) {
    const int st = embedding_check_desc(desc);
    if (st != SNHIP_STATUS_SUCCESS) return st;
    if (bytes == nullptr) return SNHIP_STATUS_INVALID_VALUE;
    *bytes = embedding_plan(desc).bytes;
    return SNHIP_STATUS_SUCCESS;
}

int snhip_embedding_backward(void* handle, const snhip_embedding_desc* desc, const void* ids, const void* dy,
                             float* table_gradient, int accumulate, void* workspace, size_t workspace_bytes) {
    const int st = embedding_check_desc(desc);
    if (st != SNHIP_STATUS_SUCCESS) return st;
    Handle* h = static_cast<Handle*>(handle);
    if (h == nullptr) return SNHIP_STATUS_NOT_INITIALIZED;
    if (desc->vocabulary == 0 || desc->dim == 0 || (desc->tokens == 0 && accumulate)) return SNHIP_STATUS_SUCCESS;
    if (table_gradient == nullptr || (desc->tokens > 0 && (ids == nullptr || dy == nullptr))) return SNHIP_STATUS_INVALID_VALUE;
    if (!aligned(ids, type_bytes(desc->id_type)) || !aligned(dy, type_bytes(desc->output_type)) || !aligned(table_gradient, 4))
        return SNHIP_STATUS_INVALID_VALUE;
    const EmbeddingPlan e = embedding_plan(desc);
    if (e.bytes > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < e.bytes)) return SNHIP_STATUS_INVALID_VALUE;
    DeviceScope scope(h->device);
    if (!scope.ok()) return SNHIP_STATUS_NOT_INITIALIZED;
    EmbeddingParams p = embedding_params(desc, ids, dy, table_gradient, true);
    const int col_blocks = ceil_div(ceil_div(p.dim, 4), 1 << p.lanes_log2);
    if (col_blocks > 65535) return SNHIP_STATUS_NOT_SUPPORTED;
    p.accumulate = accumulate != 0;
    p.sort_blocks = e.sort_blocks, p.sort_log2 = e.sort_log2, p.bins = e.bins, p.bins_log2 = e.bins_log2, p.chunk = e.chunk;
    p.fine_log2 = e.fine_log2, p.pieces = e.pieces;
    const dim3 sort_grid((unsigned)p.sort_blocks);
    const size_t lds = (size_t)16 * p.bins * sizeof(int);
    if (e.small) {
        if (desc->id_type == SNHIP_TYPE_F32)
            embedding_small_launch<float>(p, desc->output_type, sort_grid, lds, h->stream);
        else if (desc->id_type == SNHIP_TYPE_I32)
            embedding_small_launch<int>(p, desc->output_type, sort_grid, lds, h->stream);
        else
            embedding_small_launch<long long>(p, desc->output_type, sort_grid, lds, h->stream);
        return hip_to_status(hipGetLastError());
    }
    char* ws = static_cast<char*>(workspace);
    p.order = reinterpret_cast<int*>(ws + e.order), p.sorted = reinterpret_cast<int*>(ws + e.sorted);
    p.offsets = reinterpret_cast<int*>(ws + e.offsets), p.partial = reinterpret_cast<float*>(ws + e.partial);
    p.piece_id = reinterpret_cast<int*>(ws + e.piece_id), p.piece_token = reinterpret_cast<int*>(ws + e.piece_token);
    p.piece_start = reinterpret_cast<int*>(ws + e.piece_start);
    p.crossing = reinterpret_cast<int*>(ws + e.crossing), p.chunks = e.chunks;
    const int groups = 256 >> p.lanes_log2;
    const long long chunk_blocks = (e.chunks + groups - 1) / groups;
    if (desc->id_type == SNHIP_TYPE_F32)
        embedding_sort_launch<float>(p, sort_grid, lds, h->stream);
    else if (desc->id_type == SNHIP_TYPE_I32)
        embedding_sort_launch<int>(p, sort_grid, lds, h->stream);
    else
        embedding_sort_launch<long long>(p, sort_grid, lds, h->stream);
    const long long keys = (long long)p.sort_blocks * p.bins;
    const long long clear_blocks = p.accumulate ? 0 : (keys + kClearRows * groups - 1) / (kClearRows * groups);
    const dim3 chunk_grid((unsigned)chunk_blocks, (unsigned)col_blocks);
    if (chunk_blocks > 0) {
        if (desc->output_type == SNHIP_TYPE_BF16)
            hipLaunchKernelGGL(embedding_grad_kernel<__bf16>, chunk_grid, dim3(256), 0, h->stream, p);
        else
            hipLaunchKernelGGL(embedding_grad_kernel<float>, chunk_grid, dim3(256), 0, h->stream, p);
    }
    p.join_columns = (unsigned)ceil_div(p.dim, kJoinColumns), p.clear_columns = (unsigned)col_blocks;
    p.join_blocks = e.chunks <= 1 ? 0 : (unsigned)((e.chunks + kJoinGroups - 1) / kJoinGroups * p.join_columns);
    if (p.join_blocks + clear_blocks > 0)
        hipLaunchKernelGGL(embedding_join_kernel, dim3((unsigned)(p.join_blocks + clear_blocks * col_blocks)), dim3(256), 0, h->stream, p);
    return hip_to_status(hipGetLastError());
}

int snhip_sizeof_block_norm_desc(void) { return (int)sizeof(snhip_block_norm_desc); }

int snhip_block_norm_forward(void* handle, const snhip_block_norm_desc* desc) {
    const int st = block_norm_check_desc(desc, false);
    if (st != SNHIP_STATUS_SUCCESS) return st;
    Handle* h = static_cast<Handle*>(handle);
    if (h == nullptr) return SNHIP_STATUS_NOT_INITIALIZED;
    if (desc->rows == 0 || desc->dim == 0) return SNHIP_STATUS_SUCCESS;
    DeviceScope scope(h->device);
    if (!scope.ok()) return SNHIP_STATUS_NOT_INITIALIZED;
    const BlockNormParams p = block_norm_params(desc);
    switch (block_norm_types(desc)) {
        case 0: block_norm_forward_0(p, h->stream); break;
        case 1: block_norm_forward_1(p, h->stream); break;
        default: block_norm_forward_2(p, h->stream); break;
    }
    return hip_to_status(hipGetLastError());
}

int snhip_block_norm_backward_workspace_size(const snhip_block_norm_desc* desc, size_t* bytes) {
    const int st = block_norm_check_desc(desc, true);
    if (st != SNHIP_STATUS_SUCCESS) return st;
    if (bytes == nullptr) return SNHIP_STATUS_INVALID_VALUE;
    *bytes = block_norm_plan(desc).bytes;
    return SNHIP_STATUS_SUCCESS;
}

int snhip_block_norm_backward(void* handle, const snhip_block_norm_desc* desc, void* workspace, size_t workspace_bytes) {
    const int st = block_norm_check_desc(desc, true);
    if (st != SNHIP_STATUS_SUCCESS) return st;
    Handle* h = static_cast<Handle*>(handle);
    if (h == nullptr) return SNHIP_STATUS_NOT_INITIALIZED;
    if (desc->dim == 0) return SNHIP_STATUS_SUCCESS;
    const BlockNormPlan b = block_norm_plan(desc);
    if (b.bytes > 0 && (workspace == nullptr || !aligned(workspace, 16) || workspace_bytes < b.bytes))
        return SNHIP_STATUS_INVALID_VALUE;
    DeviceScope scope(h->device);
    if (!scope.ok()) return SNHIP_STATUS_NOT_INITIALIZED;
    BlockNormParams p = block_norm_params(desc);
    p.partial = static_cast<float*>(workspace);
    p.rows_per_group = b.rows_per_group, p.flush = b.flush;
    p.groups_per_chunk = b.groups_per_chunk, p.chunks_per_group = b.chunks_per_group, p.rows_per_chunk = b.rows_per_chunk;
    p.chunks = b.chunks;
    for (int k = 0; k < 5; ++k) p.slot[k] = b.slots[k];
    if (desc->rows > 0) {
        const BlockNormKind kind{desc->y == nullptr ? 0 : desc->post_norm == SNHIP_NORM_NONE ? 1 : 2,
                                 b.slots[1] >= 0 || b.slots[3] >= 0, desc->gate != nullptr};
        switch (block_norm_types(desc)) {
            case 0: block_norm_backward_0(p, kind, h->stream); break;
            case 1: block_norm_backward_1(p, kind, h->stream); break;
            default: block_norm_backward_2(p, kind, h->stream); break;
        }
    }
    // the sums over the chunks; wanted gradients without a source (no dh, no rows) are zeros
    ColumnJobs j{};
    j.partial = p.partial, j.chunks = b.chunks, j.dim = p.dim, j.chunks_per_group = b.chunks_per_group;
    j.accumulate = desc->accumulate != 0, j.accumulate_gate = desc->accumulate != 0 && desc->gate_rows == 0;
    j.slot[4] = b.slots[4];
    j.gate_out = desc->d_gate, j.ld_gate = p.ld_gate;
    j.gate_bf16 = desc->gate_rows > 0 && desc->block_type == SNHIP_TYPE_BF16;
    float* outs[4] = {desc->d_pre_weight, desc->d_pre_bias, desc->d_post_weight, desc->d_post_bias};
    for (int k = 0; k < 4; ++k) {
        if (outs[k] == nullptr) continue;
        if (b.slots[k] >= 0)
            j.out[j.vectors] = outs[k], j.slot[j.vectors] = b.slots[k], ++j.vectors;
        else if (!j.accumulate)
            hipLaunchKernelGGL(clear_vector_kernel, dim3((unsigned)ceil_div(p.dim, 256)), dim3(256), 0, h->stream, outs[k], p.dim);
    }
    // (a gate vector without rows has one group and no chunks: its gradient is cleared like the others)
    const long long gate_jobs = b.slots[4] < 0 ? 0 : desc->gate_rows == 0 ? 1 : b.groups;
    if (j.vectors + gate_jobs > 0)
        hipLaunchKernelGGL(column_parts_kernel, dim3((unsigned)ceil_div(p.dim, 32), (unsigned)(j.vectors + gate_jobs)), dim3(1024), 0,
                           h->stream, j);
    return hip_to_status(hipGetLastError());
}

int snhip_sizeof_adamw_tensor(void) { return (int)sizeof(snhip_adamw_tensor); }
int snhip_sizeof_adamw_step_desc(void) { return (int)sizeof(snhip_adamw_step_desc); }

int snhip_adamw_create(void* handle, const snhip_adamw_tensor* tensors, int count, int state_bits, void** plan) {
    if (plan == nullptr) return SNHIP_STATUS_INVALID_VALUE;
    *plan = nullptr;
    Handle* h = static_cast<Handle*>(handle);
    if (h == nullptr) return SNHIP_STATUS_NOT_INITIALIZED;
    if (count < 0 || (count > 0 && tensors == nullptr)) return SNHIP_STATUS_INVALID_VALUE;
    if (state_bits != 8 && state_bits != 32) return SNHIP_STATUS_NOT_SUPPORTED;
    try {
        return adamw_build(h, tensors, count, state_bits, plan);
    } catch (const std::bad_alloc&) {
        return SNHIP_STATUS_ALLOC_FAILED;
    } catch (...) {
        return SNHIP_STATUS_INTERNAL_ERROR;
    }
}

int snhip_adamw_destroy(void* plan) {
    if (plan == nullptr) return SNHIP_STATUS_SUCCESS;
    AdamwPlan* a = static_cast<AdamwPlan*>(plan);
    hipError_t e = hipSuccess;
    if (a->table != nullptr) {
        DeviceScope scope(a->device);
        e = scope.ok() ? hipFree(a->table) : hipErrorNoDevice;
    }
    delete a;
    return hip_to_status(e);
}

int snhip_adamw_step(void* handle, void* plan, const snhip_adamw_step_desc* d) {
    if (d == nullptr || d->struct_size != (int)sizeof(snhip_adamw_step_desc)) return SNHIP_STATUS_INVALID_VALUE;
    Handle* h = static_cast<Handle*>(handle);
    if (h == nullptr || plan == nullptr) return SNHIP_STATUS_NOT_INITIALIZED;
    const AdamwPlan* a = static_cast<const AdamwPlan*>(plan);
    if (a->device != h->device) return SNHIP_STATUS_INVALID_VALUE;
    if (d->step < 1 || !isfinite(d->learning_rate) || !(d->beta1 >= 0.0 && d->beta1 < 1.0) || !(d->beta2 >= 0.0 && d->beta2 < 1.0) ||
        !(d->epsilon >= 0.0) || !isfinite(d->epsilon) || !isfinite(d->gradient_scale))
        return SNHIP_STATUS_INVALID_VALUE;
    // What the kernels are given in fp32 has to fit: an epsilon below the normal numbers would be a zero to the reciprocal, a rate
    // beyond the largest one times nothing not a number.
    const double step_size = d->learning_rate / (1.0 - pow(d->beta1, d->step));
    if ((d->epsilon > 0.0 && d->epsilon < FLT_MIN) || fabs(d->learning_rate) > FLT_MAX || fabs(step_size) > FLT_MAX)
        return SNHIP_STATUS_INVALID_VALUE;
    if (a->chunks == 0) return SNHIP_STATUS_SUCCESS;
    DeviceScope scope(h->device);
    if (!scope.ok()) return SNHIP_STATUS_NOT_INITIALIZED;
    AdamwScalars s{};
    s.beta1 = (float)d->beta1, s.rest1 = (float)(1.0 - d->beta1);
    s.beta2 = (float)d->beta2, s.rest2 = (float)(1.0 - d->beta2);
    s.rate = (float)d->learning_rate;
    s.step_size = (float)step_size;
    s.root_scale = (float)(1.0 / sqrt(1.0 - pow(d->beta2, d->step)));
    s.eps = (float)d->epsilon, s.grad_scale = d->gradient_scale;
    s.key0 = (unsigned int)d->seed, s.key1 = (unsigned int)(d->seed >> 32), s.step = (unsigned int)d->step;
    const AdamwEntry* entries = static_cast<const AdamwEntry*>(a->table);
    const auto kernel = a->state_bits == 8 ? (a->once ? adamw8_kernel<true> : adamw8_kernel<false>)
                                           : (a->once ? adamw32_kernel<true> : adamw32_kernel<false>);
    hipLaunchKernelGGL(kernel, many_blocks(a->chunks), dim3(256), 0, h->stream, entries, a->owner, a->chunks, s);
    return hip_to_status(hipGetLastError());
}

}  // extern "C"
