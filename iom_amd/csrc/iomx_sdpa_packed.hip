// Attention of packed rows: the rows of S sequences of different lengths share one axis, each
// sees the cached tokens of its sequence (in pages) and rows of its own sequence.
//
//   sdpa_packed_rows   one wave per row and head, any head size up to 256 and any page size
#include <cmath>

#include "iomx_packed.hpp"

namespace iomx {

struct SdpaPackedArgs {
    const uint8_t *q, *k, *v, *k_pages, *v_pages;
    uint8_t* out;
    uint64_t q_head, k_head, v_head;                          // bytes
    uint64_t k_page, k_page_head, v_page, v_page_head;
    IndexMatrix starts, table, lengths, tree;                 // table.base, tree.base null: none
    uint32_t T, sequences, Hq, Hkv, group, D, d_tiles, out_tile_cols;
    uint32_t pages, page_rows, max_rows;
    FastDiv div_group, div_page_rows;
    float scale;                                              // 1 / sqrt(D)
};

constexpr uint32_t kTile16 = 512;      // bytes of a tile of a 16-bit leaf
constexpr uint32_t kMaxPackedWidth = 256;

template <int DT>
__device__ __forceinline__ float wide16(uint32_t h) {
    if constexpr (DT == IOMX_DT_BF16) return as_f32(h << 16);
    else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
template <int DT>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
    if constexpr (DT == IOMX_DT_BF16) return pack_bf16(lo, hi);
    else return pack_f16(lo, hi);
}

// What a workgroup needs to know of a sequence, every value clamped into its tensors.
struct PackedSequence {
    uint32_t start, rows, cached;
};
__device__ __forceinline__ PackedSequence packed_sequence(const SdpaPackedArgs& a, uint32_t s) {
    PackedSequence p;
    p.start = clamped(a.starts.at(s), a.T);
    const uint32_t end = clamped(a.starts.at(s + 1), a.T);
    p.rows = end > p.start ? end - p.start : 0;
    const uint64_t capacity = (uint64_t)a.table.cols * a.page_rows;
    p.cached = a.table.base ? clamped(a.lengths.at(s), (uint32_t)capacity) : 0;
    return p;
}

// One wave = one row of one head: 64 tokens at a time, a lane forms the score of one token, then
// the lanes take the features.  Running maximum and sum; everything in F32.
template <int DT>
__global__ __launch_bounds__(256) void sdpa_packed_rows_kernel(const SdpaPackedArgs a) {
    __shared__ float q_rows[4][kMaxPackedWidth];
    const float inf = __builtin_inff();
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t s = blockIdx.z;
    const PackedSequence seq = packed_sequence(a, s);
    const uint32_t rows = seq.rows < a.max_rows ? seq.rows : a.max_rows;
    const uint32_t head = blockIdx.y, hkv = divided(head, a.group, a.div_group);
    const uint8_t* kb = a.k + hkv * a.k_head;
    const uint8_t* vb = a.v + hkv * a.v_head;
    const int32_t* pages = a.table.base ? a.table.row(s) : nullptr;
    const uint32_t row_tiles = a.d_tiles * kTile16;
    // address of a token's row (null: absent)
    auto token_row = [&](const uint8_t* own, const uint8_t* pool, uint64_t page_bytes, uint64_t head_bytes,
                         uint32_t x) -> const uint8_t* {
        if (x >= seq.cached) {
            const uint32_t t = seq.start + (x - seq.cached);
            return own + (uint64_t)(t >> 4) * row_tiles + (t & 15u) * 32;
        }
        const uint32_t slot = divided(x, a.page_rows, a.div_page_rows);
        const uint32_t page = (uint32_t)pages[(uint64_t)(slot >> 4) * kTileSlots + (slot & 15u)];
        if (page >= a.pages) return nullptr;
        const uint32_t r = x - slot * a.page_rows;
        return pool + page * page_bytes + hkv * head_bytes + (uint64_t)(r >> 4) * row_tiles + (r & 15u) * 32;
    };
    auto element = [&](const uint8_t* row, uint32_t d) {
        return wide16<DT>(*reinterpret_cast<const uint16_t*>(row + (d >> 4) * kTile16 + (d & 15u) * 2));
    };
    for (uint32_t i = blockIdx.x * 4 + wave; i < rows; i += gridDim.x * 4) {
        const uint32_t t = seq.start + i;
        const uint8_t* qr = a.q + head * a.q_head + (uint64_t)(t >> 4) * row_tiles + (t & 15u) * 32;
        for (uint32_t d = lane; d < a.D; d += 64) q_rows[wave][d] = element(qr, d) * a.scale;
        __builtin_amdgcn_wave_barrier();
        const uint32_t own = a.tree.base ? (a.tree.cols * 32 < seq.rows ? a.tree.cols * 32 : seq.rows) : i + 1;
        const uint32_t tokens = seq.cached + own;
        float m = -inf, sum = 0.0f, acc[4] = {0, 0, 0, 0};
        for (uint32_t x0 = 0; x0 < tokens; x0 += 64) {
            const uint32_t x = x0 + lane;
            bool seen = x < tokens;
            if (seen && x >= seq.cached && a.tree.base) {
                const uint32_t j = x - seq.cached;
                seen = ((uint32_t)a.tree.at(t, j >> 5) >> (j & 31u)) & 1u;
            }
            const uint8_t* kr = seen ? token_row(kb, a.k_pages, a.k_page, a.k_page_head, x) : nullptr;
            seen = kr != nullptr;
            float score = -inf;
            if (seen) {
                score = 0.0f;
                for (uint32_t d = 0; d < a.D; ++d) score = __builtin_fmaf(q_rows[wave][d], element(kr, d), score);
            }
            float top = score;
            for (int off = 1; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
            const float m2 = fmaxf(m, top);
            const float base = m2 == -inf ? 0.0f : m2;
            const float p = seen ? expf(score - base) : 0.0f;   // a NaN score stays one
            const float keep = m == -inf ? 0.0f : expf(m - base);
            float part = p;
            for (int off = 1; off < 64; off *= 2) part += __shfl_xor(part, off);
            sum = sum * keep + part;
            m = m2;
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] *= keep;
            const uint64_t any = __ballot(seen);
            for (uint32_t y = 0; y < 64; ++y) {
                if (!((any >> y) & 1u)) continue;
                const float py = __shfl(p, y);
                const uint8_t* vr = token_row(vb, a.v_pages, a.v_page, a.v_page_head, x0 + y);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t d = lane + 64 * c;
                    if (d < a.D) acc[c] = __builtin_fmaf(py, element(vr, d), acc[c]);
                }
            }
        }
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint8_t* ob = a.out + (uint64_t)(t >> 4) * a.out_tile_cols * kTile16 + (t & 15u) * 32;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t d = lane + 64 * c;
            if (d >= a.D) continue;
            const uint32_t col = head * a.D + d;
            *reinterpret_cast<uint16_t*>(ob + (uint64_t)(col >> 4) * kTile16 + (col & 15u) * 2) =
                    (uint16_t)narrow2<DT>(sum == 0.0f ? 0.0f : acc[c] * inverse, 0.0f);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

namespace {

int sdpa_packed_request(int dtype, const iomx_view* q, const iomx_view* k, const iomx_view* v, const iomx_view* out,
                        const iomx_view* starts, const iomx_view* k_pages, const iomx_view* v_pages,
                        const iomx_view* table, const iomx_view* lengths, const iomx_view* tree, uint64_t max_rows,
                        SdpaPackedArgs* a) {
    IOMX_TRY(check_view(q, 16));
    IOMX_TRY(check_view(k, 16));
    IOMX_TRY(check_view(v, 16));
    IOMX_TRY(check_view(out, 16));
    if (q->rank != 3 || k->rank != 3 || out->rank != 2 || !same_extents(*k, *v)) return IOMX_ERR_INVALID;
    const Matrix qm = matrix_of(*q), om = matrix_of(*out);
    const uint64_t Hq = q->dims[0], Hkv = k->dims[0];
    uint64_t width;
    if (mul_overflows(Hq, qm.cols, &width)) return IOMX_ERR_OVERFLOW;
    if (Hq % Hkv != 0 || k->dims[1] != qm.rows || k->dims[2] != qm.cols) return IOMX_ERR_INVALID;
    if (om.rows != qm.rows || om.cols != width || max_rows == 0) return IOMX_ERR_INVALID;
    const bool cached = k_pages || v_pages || table || lengths;
    if (cached) {
        if (!k_pages || !v_pages || !table || !lengths) return IOMX_ERR_INVALID;
        IOMX_TRY(check_pools(k, k_pages, v_pages, 16));
        IOMX_TRY(sequence_operands(starts, table, lengths, &a->starts, &a->table, &a->lengths));
        if ((uint64_t)a->table.cols * k_pages->dims[2] > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    } else {
        IOMX_TRY(index_matrix(starts, &a->starts));
        if (a->starts.rows != 1 || a->starts.cols < 2) return IOMX_ERR_INVALID;
    }
    if (tree) {
        IOMX_TRY(index_matrix(tree, &a->tree));
        if (a->tree.rows != qm.rows) return IOMX_ERR_INVALID;
        if (a->tree.cols > (1u << 20)) return IOMX_ERR_UNSUPPORTED;
    }
    for (const iomx_view* in : {q, k, v, starts, k_pages, v_pages, table, lengths, tree})
        if (in && in->base == out->base) return IOMX_ERR_INVALID;
    if (dtype != IOMX_DT_BF16 && dtype != IOMX_DT_F16) return IOMX_ERR_UNSUPPORTED;
    if (qm.cols > kMaxPackedWidth) return IOMX_ERR_UNSUPPORTED;
    // rows times heads of a KV head are counted in 32 bits
    uint64_t paired;
    if (width > 0x7FFFFFF0ull || mul_overflows(qm.rows, Hq, &paired) || paired > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    uint8_t* base = nullptr;
    uint64_t strides[2];
    plane_bytes_of(*q, 16, &base, &a->q_head);
    a->q = base;
    plane_bytes_of(*k, 16, &base, &a->k_head);
    a->k = base;
    plane_bytes_of(*v, 16, &base, &a->v_head);
    a->v = base;
    plane_bytes_of(*out, 16, &a->out, strides);
    if (cached) {
        plane_bytes_of(*k_pages, 16, &base, strides);
        a->k_pages = base; a->k_page = strides[0]; a->k_page_head = strides[1];
        plane_bytes_of(*v_pages, 16, &base, strides);
        a->v_pages = base; a->v_page = strides[0]; a->v_page_head = strides[1];
        a->pages = (uint32_t)k_pages->dims[0];
        a->page_rows = (uint32_t)k_pages->dims[2];
        a->div_page_rows = make_fast_div(a->page_rows);
    }
    a->T = (uint32_t)qm.rows;
    a->sequences = a->starts.cols - 1;
    a->Hq = (uint32_t)Hq;
    a->Hkv = (uint32_t)Hkv;
    a->group = (uint32_t)(Hq / Hkv);
    a->div_group = make_fast_div(a->group);
    a->D = (uint32_t)qm.cols;
    a->d_tiles = (uint32_t)qm.tile_cols;
    a->out_tile_cols = (uint32_t)om.tile_cols;
    a->max_rows = (uint32_t)(max_rows < qm.rows ? max_rows : qm.rows);
    a->scale = 1.0f / std::sqrt((float)a->D);
    return IOMX_OK;
}

}  // namespace

}  // namespace iomx

using namespace iomx;

extern "C" int iomx_sdpa_packed_workspace(int dtype, const iomx_view* q, const iomx_view* k, const iomx_view* v,
                                          const iomx_view* out, const iomx_view* starts, const iomx_view* k_pages,
                                          const iomx_view* v_pages, const iomx_view* table, const iomx_view* lengths,
                                          const iomx_view* tree, uint64_t max_rows, uint64_t* bytes,
                                          uint64_t* alignment) {
    if (!bytes || !alignment) return IOMX_ERR_INVALID;
    SdpaPackedArgs a = {};
    IOMX_TRY(sdpa_packed_request(dtype, q, k, v, out, starts, k_pages, v_pages, table, lengths, tree, max_rows, &a));
    *bytes = 0;
    *alignment = 1;
    return IOMX_OK;
}

extern "C" int iomx_launch_sdpa_packed(int dtype, const iomx_view* q, const iomx_view* k, const iomx_view* v,
                                       const iomx_view* out, const iomx_view* starts, const iomx_view* k_pages,
                                       const iomx_view* v_pages, const iomx_view* table, const iomx_view* lengths,
                                       const iomx_view* tree, uint64_t max_rows, void* workspace,
                                       uint64_t workspace_bytes, int path, iomx_stream_t stream) {
    (void)workspace;
    (void)workspace_bytes;
    SdpaPackedArgs a = {};
    IOMX_TRY(sdpa_packed_request(dtype, q, k, v, out, starts, k_pages, v_pages, table, lengths, tree, max_rows, &a));
    if (path < 0 || path > 1) return IOMX_ERR_INVALID;
    if (a.Hq > 65535 || a.sequences > 65535) return IOMX_ERR_OVERFLOW;
    const uint32_t blocks = (a.max_rows + 3) / 4;
    const dim3 grid(blocks < 65535 ? blocks : 65535, a.Hq, a.sequences);
    if (dtype == IOMX_DT_BF16)
        hipLaunchKernelGGL(sdpa_packed_rows_kernel<IOMX_DT_BF16>, grid, dim3(256), 0, native(stream), a);
    else
        hipLaunchKernelGGL(sdpa_packed_rows_kernel<IOMX_DT_F16>, grid, dim3(256), 0, native(stream), a);
    record_launch("sdpa_packed_rows", grid.x * grid.y * grid.z, 256, (uint64_t)a.T * a.Hq);
    IOMX_HIP(hipGetLastError());
    return IOMX_OK;
}
