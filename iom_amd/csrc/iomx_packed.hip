// Row operations of packed steps: rotary position encoding with a position for every row, and
// the append of rows to a cache in pages.  Both are bound by memory: every element is read once
// and written once.
#include <cmath>

#include "iomx_packed.hpp"

namespace iomx {

// ---------------------------------------------------------------------------
// rope_packed: out[c] = x[c] cos - x[c + D/2] sin, out[c + D/2] = x[c + D/2] cos + x[c] sin,
// the angle positions[t] * theta^(-2c/D).
// ---------------------------------------------------------------------------

constexpr uint32_t kMaxRopeWidth = 512;

struct RopePackedArgs {
    const uint8_t* x;
    uint8_t* out;
    uint64_t x_head, out_head;            // bytes
    IndexMatrix positions;
    uint32_t width, tile_cols;
    uint32_t chunks;                      // 16-byte chunks of a half row
    uint32_t chunk_tiles;                 // tiles that hold them
    uint32_t tile_rows;
    FastDiv div_chunk_tiles;
    double revolutions[kMaxRopeWidth / 2];  // theta^(-2c/D) / 2 pi: turns per position
};

// sine and cosine of an angle given as a fraction of a turn in [-1/2, 1/2].  The 16-bit leaves
// take the hardware's (absolute error near 2^-20, a result's half step is 2^-9 or 2^-12 of the
// larger component), F32 the library's.  The angle is formed and reduced in binary64 and its fraction of a turn
// rounded to F32 once: at most 2^-26 of a turn, 9.4e-8 of the larger component, next to a result's half step of up to
// 6.0e-8 (32 heads of 6001 rows F32: 5.9e-8 of the norm in all, 4.2e-8 with sine and cosine in 64 bits).
template <int DT>
__device__ __forceinline__ void turn(float revolutions, float* sine, float* cosine) {
    if constexpr (DT == IOMX_DT_F32) sincospif(2.0f * revolutions, sine, cosine);
    else {
        *sine = __builtin_amdgcn_sinf(revolutions);
        *cosine = __builtin_amdgcn_cosf(revolutions);
    }
}

template <int DT>
__device__ __forceinline__ void unpack(u32x4 w, float* f) {
    if constexpr (DT == IOMX_DT_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = as_f32(w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == IOMX_DT_BF16) { f[2 * i] = bf16_lo(w[i]); f[2 * i + 1] = bf16_hi(w[i]); }
            else { const f32x2 p = f16_pair(w[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
        }
    }
}
template <int DT>
__device__ __forceinline__ u32x4 pack(const float* f) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == IOMX_DT_F32) w[i] = as_u32(canonical(f[i]));
        else if constexpr (DT == IOMX_DT_BF16) w[i] = pack_bf16(f[2 * i], f[2 * i + 1]);
        else w[i] = pack_f16(f[2 * i], f[2 * i + 1]);
    }
    return w;
}

// A lane turns one 16-byte chunk of the first half of a row with its partner of the second.  Lanes
// follow the tiles (row in tile, chunk in tile row), so a wave's accesses are whole runs of 512 or
// 1024 bytes.  The angles are formed anew for every head: two or four heads for a lane, which then
// form them once, take 36.8 and 37.8 us instead of 36.0 (32 heads of 6001 rows of 128 F32), for the
// vector units have time to spare next to the memory and the launch has fewer waves in flight.  That
// call is bound by memory: 28.7 us in the kernel for 197 MB.
template <int DT>
__global__ __launch_bounds__(256) void rope_packed_kernel(const RopePackedArgs a) {
    constexpr uint32_t kElems = DT == IOMX_DT_F32 ? 4 : 8;     // of a chunk
    constexpr uint32_t kPerRow = kTile / kElems;               // chunks of a tile row
    constexpr uint32_t kTileSize = kTileSlots * 16 / kElems;   // bytes
    const uint32_t lane = blockIdx.x * 256 + threadIdx.x;
    const uint32_t tile = lane / (kTile * kPerRow), in_tile = lane % (kTile * kPerRow);
    const uint32_t tr = divided(tile, a.chunk_tiles, a.div_chunk_tiles), tc = tile - tr * a.chunk_tiles;
    const uint32_t row = in_tile / kPerRow, chunk = tc * kPerRow + in_tile % kPerRow;
    const uint32_t t = tr * kTile + row;
    if (tr >= a.tile_rows || chunk >= a.chunks || t >= a.positions.cols) return;
    const int32_t position = a.positions.at(t);
    if (position < 0) return;
    float sine[kElems], cosine[kElems];
#pragma unroll
    for (uint32_t i = 0; i < kElems; ++i) {
        const double turns = (double)position * a.revolutions[chunk * kElems + i];
        turn<DT>((float)(turns - __builtin_rint(turns)), &sine[i], &cosine[i]);
    }
    const uint32_t partner = chunk + a.chunks;
    const uint64_t first = ((uint64_t)tr * a.tile_cols + chunk / kPerRow) * kTileSize + row * (kTileSize / kTile)
            + (chunk % kPerRow) * 16;
    const uint64_t second = ((uint64_t)tr * a.tile_cols + partner / kPerRow) * kTileSize + row * (kTileSize / kTile)
            + (partner % kPerRow) * 16;
    const uint8_t* xb = a.x + blockIdx.y * a.x_head;
    uint8_t* ob = a.out + blockIdx.y * a.out_head;
    float lo[kElems], hi[kElems], r0[kElems], r1[kElems];
    unpack<DT>(*reinterpret_cast<const u32x4*>(xb + first), lo);
    unpack<DT>(*reinterpret_cast<const u32x4*>(xb + second), hi);
#pragma unroll
    for (uint32_t i = 0; i < kElems; ++i) {
        r0[i] = lo[i] * cosine[i] - hi[i] * sine[i];
        r1[i] = hi[i] * cosine[i] + lo[i] * sine[i];
    }
    *reinterpret_cast<u32x4*>(ob + first) = pack<DT>(r0);
    *reinterpret_cast<u32x4*>(ob + second) = pack<DT>(r1);
}

// ---------------------------------------------------------------------------
// cache_append_packed
// ---------------------------------------------------------------------------

struct AppendPackedArgs {
    const uint8_t* from[2];               // k, v
    uint8_t* to[2];                       // their pools
    uint64_t from_head[2], to_page[2], to_head[2];   // bytes
    IndexMatrix starts, table, lengths, rows;        // rows.base null: entry e is row e
    uint32_t entries, sequences, heads, T, pages, page_rows;
    uint32_t tile_cols, tile_bytes, row_bytes, units;  // units: chunks of a tile row
    uint32_t lanes_per_head;              // of a band of sixteen entries
    FastDiv div_page_rows;
};

// The sequence of each of the sixteen entries e0 .. e0 + 15: the first one s with starts[s] <= e < starts[s + 1],
// or `sequences`.  The wave reads the starts 64 at a time, a word per lane; a ballot tells which are at or below an
// entry, and a sequence holds it whose start is and whose end is not: one trip to memory for up to 63
// sequences, where a search would be a chain of them (and would need starts that do not fall).
__device__ __forceinline__ uint32_t sequence_of(const IndexMatrix& starts, uint32_t sequences, uint32_t e0,
                                                uint32_t which) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t found = sequences;
    for (uint32_t s0 = 0; s0 < sequences; s0 += 63) {
        const uint32_t s = s0 + lane;
        const int32_t start = s <= sequences ? starts.at(s) : 0;
        const uint32_t count = sequences - s0 < 63 ? sequences - s0 : 63;
        uint64_t holds = 0;                      // bit: a sequence of these that holds the lane's entry
#pragma unroll
        for (uint32_t i = 0; i < kTile; ++i) {
            const uint64_t below = __ballot(start <= (int32_t)(e0 + i));
            const uint64_t here = below & ~(below >> 1) & ((1ull << count) - 1);
            holds = which == i ? here : holds;
        }
        if (found == sequences && holds) found = s0 + (uint32_t)__ffsll((unsigned long long)holds) - 1u;
    }
    return found;
}

// blockIdx.y = a band of sixteen entries; lanes follow the tiles of a head as in rope_packed, a chunk of
// K and of V each.  Bound by memory: 14 thousand rows of 24 prompts (8 KV heads of 128 F16, 115 MB with
// the writes) take 19.8 us in the kernel; a few accepted rows 3.9 us, the chain start, length, page, row.
template <class Unit>
__global__ __launch_bounds__(256) void cache_append_packed_kernel(const AppendPackedArgs a) {
    const uint32_t lane = blockIdx.x * 256 + threadIdx.x;
    const uint32_t per_tile = kTile * a.units;
    const uint32_t head = lane / a.lanes_per_head, in_head = lane - head * a.lanes_per_head;
    const uint32_t tc = in_head / per_tile, in_tile = in_head - tc * per_tile;
    const uint32_t which = in_tile / a.units, unit = in_tile - which * a.units;
    for (uint32_t band = blockIdx.y; band * kTile < a.entries; band += gridDim.y) {
        const uint32_t e = band * kTile + which;
        const uint32_t s = sequence_of(a.starts, a.sequences, band * kTile, which);
        if (head >= a.heads || e >= a.entries || s >= a.sequences) continue;
        const int32_t first = a.starts.at(s);
        const uint32_t start = first < 0 ? 0u : (uint32_t)first;
        const uint32_t row = a.rows.base ? (uint32_t)a.rows.at(e) : e;
        if (row >= a.T) continue;
        const uint64_t capacity = (uint64_t)a.table.cols * a.page_rows;
        const int32_t length = a.lengths.at(s);
        const uint64_t token = (uint64_t)(length < 0 ? 0 : length) + (e - start);
        if (token >= capacity) continue;
        const uint32_t slot = divided((uint32_t)token, a.page_rows, a.div_page_rows);
        const uint32_t page = (uint32_t)a.table.at(s, slot);
        if (page >= a.pages) continue;
        const uint32_t pr = (uint32_t)token - slot * a.page_rows;
        const uint64_t from = ((uint64_t)(row >> 4) * a.tile_cols + tc) * a.tile_bytes + (row & 15u) * a.row_bytes
                + unit * sizeof(Unit);
        const uint64_t to = ((uint64_t)(pr >> 4) * a.tile_cols + tc) * a.tile_bytes + (pr & 15u) * a.row_bytes
                + unit * sizeof(Unit);
        const Unit kw = *reinterpret_cast<const Unit*>(a.from[0] + head * a.from_head[0] + from);
        const Unit vw = *reinterpret_cast<const Unit*>(a.from[1] + head * a.from_head[1] + from);
        *reinterpret_cast<Unit*>(a.to[0] + page * a.to_page[0] + head * a.to_head[0] + to) = kw;
        *reinterpret_cast<Unit*>(a.to[1] + page * a.to_page[1] + head * a.to_head[1] + to) = vw;
    }
}

}  // namespace iomx

using namespace iomx;

extern "C" int iomx_launch_rope_packed(int dtype, const iomx_view* x, const iomx_view* out,
                                       const iomx_view* positions, double theta, iomx_stream_t stream) {
    const uint32_t bits = leaf_bits(dtype);
    if (!bits) return IOMX_ERR_UNSUPPORTED;
    IOMX_TRY(check_view(x, bits));
    IOMX_TRY(check_view(out, bits));
    RopePackedArgs a = {};
    IOMX_TRY(index_matrix(positions, &a.positions));
    if (x->rank != 3 || !same_extents(*x, *out) || out->base == x->base || out->base == positions->base)
        return IOMX_ERR_INVALID;
    const Matrix m = matrix_of(*x);
    if (a.positions.rows != 1 || a.positions.cols != m.rows) return IOMX_ERR_INVALID;
    if (!(theta >= 1.0) || theta > 3.4028234663852886e38) return IOMX_ERR_INVALID;
    if (dtype != IOMX_DT_BF16 && dtype != IOMX_DT_F16 && dtype != IOMX_DT_F32) return IOMX_ERR_UNSUPPORTED;
    if (m.cols % kTile != 0 || m.cols > kMaxRopeWidth) return IOMX_ERR_UNSUPPORTED;
    uint8_t* base = nullptr;
    plane_bytes_of(*x, bits, &base, &a.x_head);
    a.x = base;
    plane_bytes_of(*out, bits, &a.out, &a.out_head);
    const uint32_t elems = 128 / bits, per_row = kTile / elems;
    a.width = (uint32_t)m.cols;
    a.tile_cols = (uint32_t)m.tile_cols;
    a.tile_rows = (uint32_t)m.tile_rows;
    a.chunks = a.width / 2 / elems;
    a.chunk_tiles = (a.chunks + per_row - 1) / per_row;
    a.div_chunk_tiles = make_fast_div(a.chunk_tiles);
    for (uint32_t c = 0; c < a.width / 2; ++c)
        a.revolutions[c] = std::pow(theta, -2.0 * c / a.width) / 6.283185307179586476925286766559;
    const uint64_t lanes = (uint64_t)a.tile_rows * a.chunk_tiles * kTile * per_row;
    if (lanes > 0x7FFFFF00ull) return IOMX_ERR_OVERFLOW;
    if (x->dims[0] > 65535) return IOMX_ERR_OVERFLOW;
    const dim3 grid((uint32_t)((lanes + 255) / 256), (uint32_t)x->dims[0]);
    const hipStream_t st = native(stream);
    if (dtype == IOMX_DT_BF16) hipLaunchKernelGGL(rope_packed_kernel<IOMX_DT_BF16>, grid, dim3(256), 0, st, a);
    else if (dtype == IOMX_DT_F16) hipLaunchKernelGGL(rope_packed_kernel<IOMX_DT_F16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(rope_packed_kernel<IOMX_DT_F32>, grid, dim3(256), 0, st, a);
    record_launch("rope_packed", grid.x * grid.y, 256, lanes * grid.y);
    IOMX_HIP(hipGetLastError());
    return IOMX_OK;
}

extern "C" int iomx_launch_cache_append_packed(int dtype, const iomx_view* k, const iomx_view* v,
                                               const iomx_view* k_pages, const iomx_view* v_pages,
                                               const iomx_view* starts, const iomx_view* table,
                                               const iomx_view* lengths, const iomx_view* rows,
                                               iomx_stream_t stream) {
    const uint32_t bits = leaf_bits(dtype);
    if (!bits) return IOMX_ERR_UNSUPPORTED;
    IOMX_TRY(check_view(k, bits));
    IOMX_TRY(check_view(v, bits));
    if (k->rank != 3 || !same_extents(*k, *v)) return IOMX_ERR_INVALID;
    IOMX_TRY(check_pools(k, k_pages, v_pages, bits));
    AppendPackedArgs a = {};
    IOMX_TRY(sequence_operands(starts, table, lengths, &a.starts, &a.table, &a.lengths));
    if (rows) {
        IOMX_TRY(index_matrix(rows, &a.rows));
        if (a.rows.rows != 1) return IOMX_ERR_INVALID;
    }
    for (const iomx_view* pool : {k_pages, v_pages})
        for (const iomx_view* in : {k, v, starts, table, lengths, rows})
            if (in && in->base == pool->base) return IOMX_ERR_INVALID;
    const Matrix m = matrix_of(*k);
    if (m.rows > 0x7FFFFFF0ull || k->dims[0] > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    if ((uint64_t)a.table.cols * k_pages->dims[2] > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    if (m.cols % kTile != 0) return IOMX_ERR_UNSUPPORTED;
    uint8_t* base = nullptr;
    uint64_t page_strides[2];
    plane_bytes_of(*k, bits, &base, &a.from_head[0]);
    a.from[0] = base;
    plane_bytes_of(*v, bits, &base, &a.from_head[1]);
    a.from[1] = base;
    plane_bytes_of(*k_pages, bits, &a.to[0], page_strides);
    a.to_page[0] = page_strides[0]; a.to_head[0] = page_strides[1];
    plane_bytes_of(*v_pages, bits, &a.to[1], page_strides);
    a.to_page[1] = page_strides[0]; a.to_head[1] = page_strides[1];
    a.entries = rows ? a.rows.cols : (uint32_t)m.rows;
    a.sequences = a.starts.cols - 1;
    a.heads = (uint32_t)k->dims[0];
    a.T = (uint32_t)m.rows;
    a.pages = (uint32_t)k_pages->dims[0];
    a.page_rows = (uint32_t)k_pages->dims[2];
    a.div_page_rows = make_fast_div(a.page_rows);
    a.tile_cols = (uint32_t)m.tile_cols;
    a.tile_bytes = kTileSlots * bits / 8;
    a.row_bytes = kTile * bits / 8;
    const bool wide = a.row_bytes % 16 == 0;      // else 32-bit words: leaves below 8 bits
    a.units = a.row_bytes / (wide ? 16 : 4);
    const uint64_t per_head = (uint64_t)a.tile_cols * kTile * a.units, lanes = per_head * a.heads;
    if (lanes > 0x7FFFFF00ull) return IOMX_ERR_OVERFLOW;
    a.lanes_per_head = (uint32_t)per_head;
    const uint32_t bands = (a.entries + kTile - 1) / kTile;
    const dim3 grid((uint32_t)((lanes + 255) / 256), bands < 65535 ? bands : 65535);
    if (wide) hipLaunchKernelGGL(cache_append_packed_kernel<u32x4>, grid, dim3(256), 0, native(stream), a);
    else hipLaunchKernelGGL(cache_append_packed_kernel<uint32_t>, grid, dim3(256), 0, native(stream), a);
    record_launch("cache_append_packed", grid.x * grid.y, 256, lanes * bands);
    IOMX_HIP(hipGetLastError());
    return IOMX_OK;
}
