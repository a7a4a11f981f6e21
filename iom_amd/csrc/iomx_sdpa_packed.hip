// Attention of packed rows: the rows of S sequences of different lengths share one axis, each
// sees the cached tokens of its sequence (in pages) and rows of its own sequence.
//
//   sdpa_packed_mfma   matrix cores: a workgroup takes a block of rows of all heads of one KV head
//   sdpa_packed_join   joins the parts of a row block whose tokens several workgroups shared out
//   sdpa_packed_rows   one wave per row and head, any head size up to 256 and any page size
#include <cmath>

#include "iomx_mfma.hpp"
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
    // the matrix-core kernel
    uint32_t row_blocks, splits;
    uint32_t page_tiles;                                      // page_rows / 16
    FastDiv div_page_tiles, div_units, div_splits, div_hkv;
    float scale_log2;                                         // log2(e) / sqrt(D)
    float* parts;                                             // [unit][row block][split][rows][D] unnormalised sums
    float* part_stats;                                        // ... [rows][2] reference exponent and sum
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

// ---------------------------------------------------------------------------
// The matrix-core kernel.
//
// Rows m = i * group + g (row i of the sequence, head g of the KV head's group) are the columns of
// the matrix products: S^T = K Q^T puts into lane (q = lane % 16, kg = lane / 16) the scores of
// tokens 4 kg + j of a tile for column q, and in that order they are the second operand of
// O^T = V^T P^T, whose first operand ds_read_b64_tr_b16 reads out of a V tile as it lies (the
// sixteen lanes of quarter kg supply rows 4 kg .. 4 kg + 3 and receive a column each).  So scores
// and probabilities never leave their lane's registers, a row's statistics are one value per lane,
// and K and V go to LDS as they lie in memory, by the direct loader.
//
// Softmax in one pass: p = 2^(s * scale_log2 - ref), with a reference exponent per row that is moved
// (and the sums with it) only when a score exceeds it by more than kSlack: the sums may be up to
// 2^kSlack times larger than with the true maximum, which F32 does not notice, and most blocks of
// tokens need neither the maximum over lanes nor a pass over the sums.  p is rounded to the leaf for
// the second product (its error is half a step of each probability, as much as a value's own); the
// sum is taken of the unrounded ones.  F16 lifts p by 2^kLift so that small probabilities keep their
// bits: they are at most 2^(kLift + kSlack), and subnormal below 2^-22 of the largest.
//
// Only blocks that a row does not see in full (the ends of the cached prefix, the diagonal, trees,
// absent pages) form masks.  There V is cleared where no row may see it, and where a value left
// is not finite the products are formed one token at a time: 0 times infinity must not reach a row
// that does not see it.
// ---------------------------------------------------------------------------

constexpr float kLowest = -3.4028234663852886e38f;

template <int DT> struct PackedLeaf;
template <> struct PackedLeaf<IOMX_DT_BF16> {
    static constexpr float kSlack = 8.0f, kLift = 0.0f;
    static constexpr uint32_t kExponent = 0x7F80u;
    static __device__ __forceinline__ f32x4_t mfma(u32x4 a, u32x4 b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
    }
};
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
template <> struct PackedLeaf<IOMX_DT_F16> {
    static constexpr float kSlack = 6.0f, kLift = 8.0f;
    static constexpr uint32_t kExponent = 0x7C00u;
    static __device__ __forceinline__ f32x4_t mfma(u32x4 a, u32x4 b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2));
    }
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t* tr_ptr_t;

// column lane % 16 of rows 4 (lane / 16) .. + 3 of a 16 x 16 tile of 16-bit elements in LDS
__device__ __forceinline__ u32x2 read_transposed(const uint8_t* tile, uint32_t lane) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(lptr_t)(tile + lane * 8)));
}

// Where the tokens of a row block lie: `prefix` tiles of the cache, then tiles of the packed rows.
struct PackedTiles {
    uint32_t cached, prefix;      // cached tokens, their tiles
    uint32_t first;               // first tile of the packed rows
    uint32_t count;               // all tiles
};

constexpr uint32_t packed_stage_bytes(int KS, int NT) { return (uint32_t)(NT * KS * 1024); }   // of K, and of V

// WQ of the four waves share out the rows of the block and read the same tokens from LDS; the
// 4 / WQ teams of them share out the tokens.  A wave has QT columns tiles of 16 rows; NT token
// tiles are in LDS per team and stage.
template <int DT, int KS, int QT, int WQ>
__global__ __launch_bounds__(256, 2) void sdpa_packed_mfma_kernel(const SdpaPackedArgs a) {
    using Leaf = PackedLeaf<DT>;
    constexpr int WK = 4 / WQ, NT = WQ == 4 ? 4 : 2, DTL = 2 * KS;
    constexpr uint32_t BM = 16 * QT * WQ, kStage = packed_stage_bytes(KS, NT);
    __shared__ __attribute__((aligned(1024))) uint8_t k_lds[2][WK][kStage];
    __shared__ __attribute__((aligned(1024))) uint8_t v_lds[2][WK][kStage];
    const uint32_t lane = threadIdx.x & 63u, l16 = lane & 15u, kg = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t team = WQ == 4 ? 0 : wave, member = WQ == 4 ? wave : 0;

    // unit (sequence, KV head) fastest: consecutive workgroups go to different dies, a unit's row
    // blocks to the same one where the units are a multiple of eight.  Late rows, which see the most,
    // go first.
    const uint32_t units = a.sequences * a.Hkv;
    const uint32_t rest = divided(blockIdx.x, units, a.div_units), unit = blockIdx.x - rest * units;
    const uint32_t rb_up = divided(rest, a.splits, a.div_splits), split = rest - rb_up * a.splits;
    const uint32_t rb = a.row_blocks - 1 - rb_up;
    const uint32_t s = divided(unit, a.Hkv, a.div_hkv), hkv = unit - s * a.Hkv;
    const PackedSequence seq = packed_sequence(a, s);
    const uint32_t rows = seq.rows < a.max_rows ? seq.rows : a.max_rows;
    const uint32_t m_end = rows * a.group, m_block = rb * BM;
    if (m_block >= m_end) return;

    // own rows that some row of the block sees
    uint32_t own;
    if (a.tree.base) own = a.tree.cols * 32 < seq.rows ? a.tree.cols * 32 : seq.rows;
    else {
        const uint32_t m_last = m_block + BM < m_end ? m_block + BM - 1 : m_end - 1;
        own = divided(m_last, a.group, a.div_group) + 1;
    }
    PackedTiles tiles;
    tiles.cached = seq.cached;
    tiles.prefix = (seq.cached + 15) >> 4;
    tiles.first = seq.start >> 4;
    tiles.count = tiles.prefix + ((seq.start + own + 15) >> 4) - tiles.first;
    const uint32_t blocks = (tiles.count + NT - 1) / NT;
    const uint32_t per_split = (blocks + a.splits - 1) / a.splits;
    const uint32_t b_begin = split * per_split + team;
    const uint32_t b_end = (split + 1) * per_split < blocks ? (split + 1) * per_split : blocks;

    // this wave's columns: rows of the sequence, and the wave's range of them
    const uint32_t m_wave = m_block + member * 16 * QT;
    uint32_t row_of[QT];
#pragma unroll
    for (int q = 0; q < QT; ++q) row_of[q] = divided(m_wave + 16 * q + l16, a.group, a.div_group);
    const bool idle = m_wave >= m_end;
    const uint32_t i_first = divided(m_wave, a.group, a.div_group);
    const uint32_t i_last = divided(m_wave + 16 * QT - 1, a.group, a.div_group);
    const uint32_t row_tiles = a.d_tiles * kTile16;

    u32x4 qf[QT][KS];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        const uint32_t m = m_wave + 16 * q + l16, t = seq.start + row_of[q];
        const uint32_t head = hkv * a.group + (m - row_of[q] * a.group);
        const uint8_t* qr = a.q + head * a.q_head + (uint64_t)(t >> 4) * row_tiles + (t & 15u) * 32 + (kg & 1u) * 16;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            const uint32_t tile = 2 * c + (kg >> 1);
            qf[q][c] = u32x4{0, 0, 0, 0};
            if (m < m_end && tile < a.d_tiles) qf[q][c] = *reinterpret_cast<const u32x4*>(qr + tile * kTile16);
        }
    }
    // with an odd number of feature tiles the last one of a token tile's stage is not loaded: it
    // meets zeros of Q and has to be finite
    if (a.d_tiles < (uint32_t)DTL) {
        for (uint32_t i = threadIdx.x; i < 2 * WK * NT * 32; i += 256)
            *reinterpret_cast<u32x4*>(&k_lds[0][0][0] + (i >> 5) * (KS * 1024) + (DTL - 1) * kTile16 + (i & 31u) * 16) = u32x4{0, 0, 0, 0};
        __syncthreads();
    }

    // page numbers of a block's tiles, one per lane below NT; ~0 where there is nothing to load
    auto block_pages = [&](uint32_t b) -> uint32_t {
        const uint32_t x = b * NT + lane;
        if (lane >= NT || b >= b_end || x >= tiles.count) return ~0u;
        if (x >= tiles.prefix) return 0u;
        const uint32_t slot = divided(x, a.page_tiles, a.div_page_tiles);
        const uint32_t page = (uint32_t)a.table.at(s, slot);
        return page < a.pages ? page : ~0u;
    };
    const bool odd = a.d_tiles < (uint32_t)DTL;
    // brings the tiles of block b to a stage: wave `member` of a team of four takes tile `member`
    auto fetch = [&](uint32_t b, uint32_t pages, uint8_t* ks, uint8_t* vs) {
#pragma unroll
        for (int n = 0; n < NT / WQ; ++n) {
            const uint32_t at = member + n;
            const uint32_t x = b * NT + at;
            const uint32_t page = __builtin_amdgcn_readlane(pages, at);
            if (page == ~0u) continue;
            const uint8_t *kt, *vt;
            if (x < tiles.prefix) {
                const uint32_t slot = divided(x, a.page_tiles, a.div_page_tiles);
                const uint64_t in_page = (uint64_t)(x - slot * a.page_tiles) * row_tiles;
                kt = a.k_pages + page * a.k_page + hkv * a.k_page_head + in_page;
                vt = a.v_pages + page * a.v_page + hkv * a.v_page_head + in_page;
            } else {
                const uint64_t row_at = (uint64_t)(tiles.first + x - tiles.prefix) * row_tiles;
                kt = a.k + hkv * a.k_head + row_at;
                vt = a.v + hkv * a.v_head + row_at;
            }
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                if (c == KS - 1 && odd && lane >= 32) break;
                __builtin_amdgcn_global_load_lds((gptr_t)(kt + c * 1024 + lane * 16), (lptr_t)(ks + at * (KS * 1024) + c * 1024), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((gptr_t)(vt + c * 1024 + lane * 16), (lptr_t)(vs + at * (KS * 1024) + c * 1024), 16, 0, 0);
            }
        }
    };

    f32x4_t acc[DTL][QT];
    float ref[QT], sum[QT];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        ref[q] = kLowest;
        sum[q] = 0.0f;
#pragma unroll
        for (int d = 0; d < DTL; ++d) acc[d][q] = f32x4_t{0, 0, 0, 0};
    }
    // tiles that every row of this wave sees in full
    const uint32_t whole_prefix = tiles.cached >> 4;
    const uint32_t whole_first = tiles.prefix + ((seq.start + 15) >> 4) - tiles.first;
    const uint32_t whole_end = a.tree.base ? 0 : tiles.prefix + ((seq.start + i_first + 1) >> 4) - tiles.first;
    const uint32_t k_lane = (kg >> 1) * kTile16 + l16 * 32 + (kg & 1u) * 16;

    // Two token tiles (x, x + 1) of the stage: scores, probabilities, sums.
    auto two_tiles = [&](uint32_t x, uint32_t present, const uint8_t* ks, const uint8_t* vs) {
        if (idle || !present) return;
        // the wave's rows are all before these tokens
        if (!a.tree.base && x >= tiles.prefix && ((tiles.first + x - tiles.prefix) << 4) > seq.start + i_last) return;
        f32x4_t sc[2][QT];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int q = 0; q < QT; ++q) sc[t][q] = f32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(ks + t * (KS * 1024) + c * 1024 + k_lane);
#pragma unroll
                for (int q = 0; q < QT; ++q) sc[t][q] = Leaf::mfma(kf, qf[q][c], sc[t][q]);
            }
        }
        auto whole = [&](uint32_t y) { return y < whole_prefix || (y >= whole_first && y < whole_end); };
        const bool masked = present != 3u || !whole(x) || !whole(x + 1);
        uint32_t seen[QT];                  // bit 4 t + j: the column sees token 4 kg + j of tile t
        uint32_t keep[2][2];                // V words (two tokens each) that some row may see
        if (masked) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t y = x + t;
                uint32_t any = 0;
                if (!((present >> t) & 1u)) {
#pragma unroll
                    for (int q = 0; q < QT; ++q) seen[q] = t ? seen[q] : 0u;
                } else if (y < tiles.prefix) {
                    const uint32_t token = y * 16 + 4 * kg;
                    const uint32_t n = token >= tiles.cached ? 0 : tiles.cached - token < 4 ? tiles.cached - token : 4;
                    any = (1u << n) - 1u;
#pragma unroll
                    for (int q = 0; q < QT; ++q) seen[q] = t ? seen[q] | any << 4 : any;
                } else {
                    // own rows j .. j + 3 of the sequence
                    const int32_t j = (int32_t)((tiles.first + y - tiles.prefix) * 16 + 4 * kg) - (int32_t)seq.start;
#pragma unroll
                    for (int i = 0; i < 4; ++i) any |= (uint32_t)(j + i >= 0 && j + i < (int32_t)seq.rows) << i;
#pragma unroll
                    for (int q = 0; q < QT; ++q) {
                        uint32_t bits = 0;
                        if (a.tree.base) {
                            if (any && m_wave + 16 * q + l16 < m_end) {
                                const uint32_t row = seq.start + row_of[q];
                                const int32_t w = j >> 5;              // -1 for the rows before the first
                                const uint32_t lo = w >= 0 && w < (int32_t)a.tree.cols ? (uint32_t)a.tree.at(row, w) : 0u;
                                const uint32_t hi = w + 1 < (int32_t)a.tree.cols ? (uint32_t)a.tree.at(row, w + 1) : 0u;
                                bits = (uint32_t)((((uint64_t)hi << 32) | lo) >> (j & 31));
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i) bits |= (uint32_t)(j + i <= (int32_t)row_of[q]) << i;
                        }
                        bits &= any;
                        seen[q] = t ? seen[q] | bits << 4 : bits;
                    }
                }
                keep[t][0] = ((any & 1u) ? 0xFFFFu : 0u) | ((any & 2u) ? 0xFFFF0000u : 0u);
                keep[t][1] = ((any & 4u) ? 0xFFFFu : 0u) | ((any & 8u) ? 0xFFFF0000u : 0u);
            }
#pragma unroll
            for (int q = 0; q < QT; ++q)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        sc[t][q][j] = (seen[q] >> (4 * t + j)) & 1u ? sc[t][q][j] : -__builtin_inff();
        }
        // scores beyond the reference move it
        float top[QT];
        bool beyond = false;
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            top[q] = fmaxf(fmaxf(fmaxf(sc[0][q][0], sc[0][q][1]), fmaxf(sc[0][q][2], sc[0][q][3])),
                           fmaxf(fmaxf(sc[1][q][0], sc[1][q][1]), fmaxf(sc[1][q][2], sc[1][q][3]))) * a.scale_log2;
            beyond = beyond || top[q] > ref[q] + Leaf::kSlack;
        }
        if (__any(beyond)) {
#pragma unroll
            for (int q = 0; q < QT; ++q) {
                float r = fmaxf(top[q], __shfl_xor(top[q], 16));
                r = fmaxf(r, __shfl_xor(r, 32));
                r = fmaxf(r, ref[q]);
                const float factor = __builtin_amdgcn_exp2f(ref[q] - r);
                ref[q] = r;
                sum[q] *= factor;
#pragma unroll
                for (int d = 0; d < DTL; ++d) acc[d][q] *= factor;
            }
        }
        u32x4 pf[QT];
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const float minus = Leaf::kLift - ref[q];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int j = 0; j < 4; ++j) sc[t][q][j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][q][j], a.scale_log2, minus));
                sum[q] += (sc[t][q][0] + sc[t][q][1]) + (sc[t][q][2] + sc[t][q][3]);
            }
            pf[q] = u32x4{Leaf::pair(sc[0][q][0], sc[0][q][1]), Leaf::pair(sc[0][q][2], sc[0][q][3]),
                          Leaf::pair(sc[1][q][0], sc[1][q][1]), Leaf::pair(sc[1][q][2], sc[1][q][3])};
        }
        auto values = [&](int d) {
            const u32x2 lo = read_transposed(vs + d * kTile16, lane), hi = read_transposed(vs + KS * 1024 + d * kTile16, lane);
            return u32x4{lo.x, lo.y, hi.x, hi.y};
        };
        if (!masked) {
#pragma unroll
            for (int d = 0; d < DTL; ++d) {
                const u32x4 vf = values(d);
#pragma unroll
                for (int q = 0; q < QT; ++q) acc[d][q] = Leaf::mfma(vf, pf[q], acc[d][q]);
            }
            return;
        }
        auto kept = [&](int d) {
            u32x4 vf = values(d);
            vf[0] &= keep[0][0]; vf[1] &= keep[0][1]; vf[2] &= keep[1][0]; vf[3] &= keep[1][1];
            return vf;
        };
        constexpr uint32_t lo_exp = Leaf::kExponent, hi_exp = Leaf::kExponent << 16;
        bool special = false;
#pragma unroll
        for (int d = 0; d < DTL; ++d) {
            if (d == DTL - 1 && odd) continue;        // not loaded, and its sums are not used
            const u32x4 vf = kept(d);
#pragma unroll
            for (int w = 0; w < 4; ++w) special = special || (vf[w] & lo_exp) == lo_exp || (vf[w] & hi_exp) == hi_exp;
        }
        if (!__any(special)) {
#pragma unroll
            for (int d = 0; d < DTL; ++d) {
                const u32x4 vf = kept(d);
#pragma unroll
                for (int q = 0; q < QT; ++q) acc[d][q] = Leaf::mfma(vf, pf[q], acc[d][q]);
            }
            return;
        }
        // one token at a time: lane (q, kg) adds features 4 kg .. 4 kg + 3 of every feature tile
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
#pragma clang loop unroll(disable)
                for (uint32_t from = 0; from < 4; ++from) {
                    const uint8_t* vr = vs + t * (KS * 1024) + (4 * from + j) * 32 + kg * 8;
#pragma unroll
                    for (int q = 0; q < QT; ++q) {
                        const float p = __shfl(sc[t][q][j], from * 16 + l16);
                        const uint32_t bits = __shfl(seen[q], from * 16 + l16);
                        if ((bits >> (4 * t + j)) & 1u) {
#pragma unroll
                            for (int d = 0; d < DTL; ++d) {
                                const u32x2 w = *reinterpret_cast<const u32x2*>(vr + d * kTile16);
                                acc[d][q][0] = __builtin_fmaf(p, wide16<DT>(w.x & 0xFFFFu), acc[d][q][0]);
                                acc[d][q][1] = __builtin_fmaf(p, wide16<DT>(w.x >> 16), acc[d][q][1]);
                                acc[d][q][2] = __builtin_fmaf(p, wide16<DT>(w.y & 0xFFFFu), acc[d][q][2]);
                                acc[d][q][3] = __builtin_fmaf(p, wide16<DT>(w.y >> 16), acc[d][q][3]);
                            }
                        }
                    }
                }
            }
        }
    };

    // Two stages: while a block is computed, the direct loader fills the other one.  The wait and
    // the barrier at the top make the block's tiles visible to the team and the other stage free.
    uint32_t pages = block_pages(b_begin);
    uint32_t next_pages = block_pages(b_begin + WK);
    if (b_begin < b_end) fetch(b_begin, pages, k_lds[0][team], v_lds[0][team]);
    auto step = [&](uint32_t b, int stage) {
        const uint32_t present = (uint32_t)__ballot(pages != ~0u);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);        // vmcnt(0), lgkmcnt(0)
        if constexpr (WQ == 4) __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        pages = next_pages;
        if (b + WK < b_end) fetch(b + WK, pages, k_lds[stage ^ 1][team], v_lds[stage ^ 1][team]);
        next_pages = block_pages(b + 2 * WK);
#pragma unroll
        for (int h = 0; h < NT / 2; ++h)
            two_tiles(b * NT + 2 * h, (present >> (2 * h)) & 3u, &k_lds[stage][team][h * 2 * KS * 1024],
                      &v_lds[stage][team][h * 2 * KS * 1024]);
    };
    for (uint32_t b = b_begin; b < b_end; b += 2 * WK) {
        step(b, 0);
        if (b + WK >= b_end) break;
        step(b + WK, 1);
    }
    // the columns' sums over the four token quarters
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        sum[q] += __shfl_xor(sum[q], 16);
        sum[q] += __shfl_xor(sum[q], 32);
    }

    const uint64_t part = ((uint64_t)unit * a.row_blocks + rb) * a.splits + split;
    auto emit = [&](uint32_t m_in_block, uint32_t feature, f32x4_t o, float r, float l) {
        const uint32_t m = m_block + m_in_block;
        if (m >= m_end || feature >= a.D) return;
        if (a.splits > 1) {
            *reinterpret_cast<f32x4_t*>(a.parts + (part * BM + m_in_block) * a.D + feature) = o;
            if (feature == 0) {
                a.part_stats[(part * BM + m_in_block) * 2] = r;
                a.part_stats[(part * BM + m_in_block) * 2 + 1] = l;
            }
            return;
        }
        const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
        const uint32_t i = divided(m, a.group, a.div_group), t = seq.start + i;
        const uint32_t col = (hkv * a.group + (m - i * a.group)) * a.D + feature;
        u32x2 w = {narrow2<DT>(o[0] * inverse, o[1] * inverse), narrow2<DT>(o[2] * inverse, o[3] * inverse)};
        if (l == 0.0f) w = u32x2{0, 0};
        *reinterpret_cast<u32x2*>(a.out + ((uint64_t)(t >> 4) * a.out_tile_cols + (col >> 4)) * kTile16 + (t & 15u) * 32
                                  + (col & 15u) * 2) = w;
    };
    if constexpr (WK == 1) {
        if (idle) return;
#pragma unroll
        for (int q = 0; q < QT; ++q)
#pragma unroll
            for (int d = 0; d < DTL; ++d) emit(member * 16 * QT + 16 * q + l16, 16 * d + 4 * kg, acc[d][q], ref[q], sum[q]);
    } else {
        // the teams meet in LDS: a wave leaves its sums scaled to the largest reference of all
        constexpr uint32_t kRows = 16 * QT, kFeatures = 32 * KS;
        __shared__ float meet_ref[WK][kRows], meet_sum[WK][kRows];
        static_assert(WK * kRows * kFeatures * 4 <= 2 * WK * kStage, "the teams' sums fit K's stages");
        float* meet = reinterpret_cast<float*>(&k_lds[0][0][0]);     // [team][row][feature]
        if (kg == 0) {
#pragma unroll
            for (int q = 0; q < QT; ++q) { meet_ref[team][16 * q + l16] = ref[q]; meet_sum[team][16 * q + l16] = sum[q]; }
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            float r = kLowest;
#pragma unroll
            for (int w = 0; w < WK; ++w) r = fmaxf(r, meet_ref[w][16 * q + l16]);
            const float factor = __builtin_amdgcn_exp2f(ref[q] - r);
#pragma unroll
            for (int d = 0; d < DTL; ++d)
                *reinterpret_cast<f32x4_t*>(meet + ((team * kRows + 16 * q + l16) * kFeatures) + 16 * d + 4 * kg) = acc[d][q] * factor;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < kRows * kFeatures / 4; i += 256) {
            const uint32_t row = i / (kFeatures / 4), feature = i % (kFeatures / 4) * 4;
            float r = kLowest, l = 0.0f;
#pragma unroll
            for (int w = 0; w < WK; ++w) r = fmaxf(r, meet_ref[w][row]);
            f32x4_t o = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                l += meet_sum[w][row] * __builtin_amdgcn_exp2f(meet_ref[w][row] - r);
                o += *reinterpret_cast<const f32x4_t*>(meet + (w * kRows + row) * kFeatures + feature);
            }
            emit(row, feature, o, r, l);
        }
    }
}

// Four features of a row: the parts of its row block, each scaled from its own reference.
template <int DT>
__global__ __launch_bounds__(256) void sdpa_packed_join_kernel(const SdpaPackedArgs a, uint32_t block_rows) {
    const uint32_t chunks = a.D / 4;
    const uint32_t unit = blockIdx.y + blockIdx.z * 65535u;
    if (unit >= a.sequences * a.Hkv) return;
    const uint32_t s = divided(unit, a.Hkv, a.div_hkv), hkv = unit - s * a.Hkv;
    const PackedSequence seq = packed_sequence(a, s);
    const uint32_t rows = seq.rows < a.max_rows ? seq.rows : a.max_rows;
    const uint32_t at = blockIdx.x * 256 + threadIdx.x, m = at / chunks, feature = at % chunks * 4;
    if (m >= rows * a.group) return;
    const uint64_t first = ((uint64_t)unit * a.row_blocks + m / block_rows) * a.splits * block_rows + m % block_rows;
    float r = kLowest;
    for (uint32_t p = 0; p < a.splits; ++p) r = fmaxf(r, a.part_stats[(first + (uint64_t)p * block_rows) * 2]);
    float l = 0.0f;
    f32x4_t o = {0, 0, 0, 0};
    for (uint32_t p = 0; p < a.splits; ++p) {
        const uint64_t row = first + (uint64_t)p * block_rows;
        const float factor = __builtin_amdgcn_exp2f(a.part_stats[row * 2] - r);
        l += a.part_stats[row * 2 + 1] * factor;
        o += *reinterpret_cast<const f32x4_t*>(a.parts + row * a.D + feature) * factor;
    }
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
    const uint32_t i = divided(m, a.group, a.div_group), t = seq.start + i;
    const uint32_t col = (hkv * a.group + (m - i * a.group)) * a.D + feature;
    u32x2 w = {narrow2<DT>(o[0] * inverse, o[1] * inverse), narrow2<DT>(o[2] * inverse, o[3] * inverse)};
    if (l == 0.0f) w = u32x2{0, 0};
    *reinterpret_cast<u32x2*>(a.out + ((uint64_t)(t >> 4) * a.out_tile_cols + (col >> 4)) * kTile16 + (t & 15u) * 32
                              + (col & 15u) * 2) = w;
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

// How a request runs on the matrix cores: rows of a block, workgroups that share a block's tokens,
// and the workspace their parts need.
struct PackedPlan {
    bool mfma;
    int tiles_per_wave;      // QT
    int row_waves;           // WQ
    uint32_t block_rows, row_blocks, splits;
    uint64_t parts_floats, stats_floats;
};

int packed_plan(const SdpaPackedArgs& a, int path, PackedPlan* p) {
    *p = {};
    p->mfma = path != 1 && a.D % kTile == 0 && a.D <= 128 && (!a.table.base || a.page_rows % kTile == 0);
    if (!p->mfma) return IOMX_OK;
    const uint64_t m = (uint64_t)a.max_rows * a.group;       // rows of the longest sequence, per KV head
    if (m <= 16) { p->row_waves = 1; p->tiles_per_wave = 1; }
    else if (m <= 32) { p->row_waves = 1; p->tiles_per_wave = 2; }
    else if (m <= 64) { p->row_waves = 4; p->tiles_per_wave = 1; }
    else { p->row_waves = 4; p->tiles_per_wave = 2; }
    p->block_rows = 16u * p->row_waves * p->tiles_per_wave;
    p->row_blocks = (uint32_t)((m + p->block_rows - 1) / p->block_rows);
    const uint64_t units = (uint64_t)a.sequences * a.Hkv, groups = units * p->row_blocks;
    // enough workgroups for two per CU; at least four blocks of tokens for each
    const uint64_t capacity = (uint64_t)a.table.cols * a.page_rows + a.max_rows;
    const uint64_t step = p->row_waves == 4 ? 64 : 128;
    uint64_t splits = groups >= 512 ? 1 : 512 / groups;
    const uint64_t most = capacity / (4 * step);
    if (splits > most) splits = most;
    if (splits > 64) splits = 64;
    p->splits = (uint32_t)(splits ? splits : 1);
    if (groups * p->splits > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    if (p->splits > 1) {
        p->stats_floats = (groups * p->splits * p->block_rows * 2 + 63) / 64 * 64;
        p->parts_floats = groups * p->splits * p->block_rows * a.D;
    }
    return IOMX_OK;
}

template <int DT, int KS>
void launch_packed(const SdpaPackedArgs& a, const PackedPlan& p, dim3 grid, hipStream_t st) {
    if (p.row_waves == 1 && p.tiles_per_wave == 1)
        hipLaunchKernelGGL((sdpa_packed_mfma_kernel<DT, KS, 1, 1>), grid, dim3(256), 0, st, a);
    else if (p.row_waves == 1)
        hipLaunchKernelGGL((sdpa_packed_mfma_kernel<DT, KS, 2, 1>), grid, dim3(256), 0, st, a);
    else if (p.tiles_per_wave == 1)
        hipLaunchKernelGGL((sdpa_packed_mfma_kernel<DT, KS, 1, 4>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((sdpa_packed_mfma_kernel<DT, KS, 2, 4>), grid, dim3(256), 0, st, a);
}

template <int DT>
void launch_packed(const SdpaPackedArgs& a, const PackedPlan& p, dim3 grid, hipStream_t st) {
    switch ((a.D + 31) / 32) {
        case 1: launch_packed<DT, 1>(a, p, grid, st); break;
        case 2: launch_packed<DT, 2>(a, p, grid, st); break;
        case 3: launch_packed<DT, 3>(a, p, grid, st); break;
        default: launch_packed<DT, 4>(a, p, grid, st); break;
    }
    if (p.splits > 1) {
        const uint64_t lanes = (uint64_t)a.max_rows * a.group * (a.D / 4);
        const uint64_t units = (uint64_t)a.sequences * a.Hkv;
        const dim3 joins((uint32_t)((lanes + 255) / 256), (uint32_t)(units < 65535 ? units : 65535), (uint32_t)((units + 65534) / 65535));
        hipLaunchKernelGGL(sdpa_packed_join_kernel<DT>, joins, dim3(256), 0, st, a, p.block_rows);
    }
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
    PackedPlan p;
    IOMX_TRY(packed_plan(a, 0, &p));
    *bytes = (p.stats_floats + p.parts_floats) * 4;
    *alignment = *bytes ? 256 : 1;
    return IOMX_OK;
}

extern "C" int iomx_launch_sdpa_packed(int dtype, const iomx_view* q, const iomx_view* k, const iomx_view* v,
                                       const iomx_view* out, const iomx_view* starts, const iomx_view* k_pages,
                                       const iomx_view* v_pages, const iomx_view* table, const iomx_view* lengths,
                                       const iomx_view* tree, uint64_t max_rows, void* workspace,
                                       uint64_t workspace_bytes, int path, iomx_stream_t stream) {
    SdpaPackedArgs a = {};
    IOMX_TRY(sdpa_packed_request(dtype, q, k, v, out, starts, k_pages, v_pages, table, lengths, tree, max_rows, &a));
    if (path < 0 || path > 1) return IOMX_ERR_INVALID;
    PackedPlan p;
    IOMX_TRY(packed_plan(a, path, &p));
    const hipStream_t st = native(stream);
    if (p.mfma) {
        const uint64_t bytes = (p.stats_floats + p.parts_floats) * 4;
        if (bytes && (!workspace || workspace_bytes < bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
            return IOMX_ERR_INVALID;
        a.row_blocks = p.row_blocks;
        a.splits = p.splits;
        a.page_tiles = a.page_rows / kTile;
        a.div_page_tiles = make_fast_div(a.page_tiles);
        a.div_units = make_fast_div(a.sequences * a.Hkv);
        a.div_splits = make_fast_div(a.splits);
        a.div_hkv = make_fast_div(a.Hkv);
        a.scale_log2 = 1.44269504088896340736f * a.scale;
        a.part_stats = static_cast<float*>(workspace);
        a.parts = a.part_stats + p.stats_floats;
        const dim3 grid(a.sequences * a.Hkv * p.row_blocks * p.splits);
        if (dtype == IOMX_DT_BF16) launch_packed<IOMX_DT_BF16>(a, p, grid, st);
        else launch_packed<IOMX_DT_F16>(a, p, grid, st);
        record_launch(p.row_waves == 1 ? "sdpa_packed_few" : "sdpa_packed_mfma", grid.x, 256, (uint64_t)a.T * a.Hq);
        IOMX_HIP(hipGetLastError());
        return IOMX_OK;
    }
    if (a.Hq > 65535 || a.sequences > 65535) return IOMX_ERR_OVERFLOW;
    const uint32_t blocks = (a.max_rows + 3) / 4;
    const dim3 grid(blocks < 65535 ? blocks : 65535, a.Hq, a.sequences);
    if (dtype == IOMX_DT_BF16)
        hipLaunchKernelGGL(sdpa_packed_rows_kernel<IOMX_DT_BF16>, grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(sdpa_packed_rows_kernel<IOMX_DT_F16>, grid, dim3(256), 0, st, a);
    record_launch("sdpa_packed_rows", grid.x * grid.y * grid.z, 256, (uint64_t)a.T * a.Hq);
    IOMX_HIP(hipGetLastError());
    return IOMX_OK;
}
