// What the operations on packed rows share: the small I32 operands (starts, lengths, page
// tables, positions), which are tiled views like every other tensor.
#pragma once
#include "iomx_common.hpp"

namespace iomx {

// A rank-two view of 32-bit values on the device.
struct IndexMatrix {
    const int32_t* base;   // the view's own plane
    uint32_t rows, cols, tile_cols;

#if defined(__HIPCC__)
    __device__ __forceinline__ int32_t at(uint32_t r, uint32_t c) const {
        return base[((uint64_t)(r >> 4) * tile_cols + (c >> 4)) * kTileSlots + (r & 15u) * kTile + (c & 15u)];
    }
    __device__ __forceinline__ int32_t at(uint32_t c) const { return base[(uint64_t)(c >> 4) * kTileSlots + (c & 15u)]; }
    // first entry of a row: element m of the row is entry (m / 16) * 256 + m % 16 from here
    __device__ __forceinline__ const int32_t* row(uint32_t r) const {
        return base + (uint64_t)(r >> 4) * tile_cols * kTileSlots + (r & 15u) * kTile;
    }
#endif
};

inline int index_matrix(const iomx_view* v, IndexMatrix* m) {
    IOMX_TRY(check_view(v, 32));
    if (v->rank != 2) return IOMX_ERR_INVALID;
    const Matrix g = matrix_of(*v);
    if (g.rows > 0x7FFFFFF0ull || g.cols > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    m->base = static_cast<const int32_t*>(v->base) + v->plane_offset * g.plane_elems;
    m->rows = (uint32_t)g.rows;
    m->cols = (uint32_t)g.cols;
    m->tile_cols = (uint32_t)g.tile_cols;
    return IOMX_OK;
}

// starts [1, S+1], table [S, M], lengths [1, S]
inline int sequence_operands(const iomx_view* starts, const iomx_view* table, const iomx_view* lengths,
                             IndexMatrix* s, IndexMatrix* t, IndexMatrix* l) {
    IOMX_TRY(index_matrix(starts, s));
    IOMX_TRY(index_matrix(table, t));
    IOMX_TRY(index_matrix(lengths, l));
    if (s->rows != 1 || l->rows != 1 || s->cols < 2) return IOMX_ERR_INVALID;
    if (t->rows != s->cols - 1 || l->cols != s->cols - 1) return IOMX_ERR_INVALID;
    return IOMX_OK;
}

// A [planes.., rows, cols] view of `rank` axes as the address of its first plane and a byte
// stride for each leading axis (rank - 2 of them).
inline void plane_bytes_of(const iomx_view& v, uint32_t bits, uint8_t** base, uint64_t* strides) {
    const uint64_t plane = matrix_of(v).plane_elems * bits / 8;
    *base = static_cast<uint8_t*>(v.base) + v.plane_offset * plane;
    for (uint32_t a = 0; a + 2 < v.rank; ++a) strides[a] = v.plane_strides[a] * plane;
}

inline bool same_extents(const iomx_view& a, const iomx_view& b) {
    if (a.rank != b.rank) return false;
    for (uint32_t i = 0; i < a.rank; ++i)
        if (a.dims[i] != b.dims[i]) return false;
    return true;
}

// k and v [Hkv,T,D] next to pools k_pages and v_pages [N,Hkv,P,D]
inline int check_pools(const iomx_view* k, const iomx_view* k_pages, const iomx_view* v_pages, uint32_t bits) {
    IOMX_TRY(check_view(k_pages, bits));
    IOMX_TRY(check_view(v_pages, bits));
    if (k_pages->rank != 4 || !same_extents(*k_pages, *v_pages)) return IOMX_ERR_INVALID;
    if (k_pages->dims[1] != k->dims[0] || k_pages->dims[3] != k->dims[2]) return IOMX_ERR_INVALID;
    if (k_pages->dims[0] > 0x7FFFFFF0ull || k_pages->dims[2] > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    return IOMX_OK;
}

#if defined(__HIPCC__)

// n / d for any d >= 1 (fast_div needs two)
__device__ __forceinline__ uint32_t divided(uint32_t n, uint32_t d, FastDiv f) { return d == 1 ? n : fast_div(n, f); }

// a device value as a count of at most `most`
__device__ __forceinline__ uint32_t clamped(int32_t value, uint32_t most) {
    const uint32_t v = value < 0 ? 0u : (uint32_t)value;
    return v < most ? v : most;
}

#endif

}  // namespace iomx
