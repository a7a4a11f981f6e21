// Attention of packed rows: the rows of S sequences of different lengths share one axis, each
// sees the cached tokens of its sequence (in pages) and rows of its own sequence.
//
//   sdpa_packed_mfma   matrix cores: a workgroup takes a block of rows of all heads of one KV head
//   sdpa_packed_join   joins the parts of row blocks whose tokens were shared out
//   sdpa_packed_rows   one wave per row and head, any head size up to 256 and any page size
#include <cmath>
#include <type_traits>

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
    uint32_t row_blocks;
    uint32_t places;                                          // for the pieces of a KV head (PackedShare); 0: not shared out
    uint32_t page_tiles;                                      // page_rows / 16
    FastDiv div_page_tiles, div_units, div_hkv;
    float scale_log2;                                         // log2(e) / sqrt(D)
    float* parts;                                             // [workgroup][rows][D] unnormalised sums
    float* part_stats;                                        // [workgroup][rows][2] reference exponent and sum
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

template <int DT>
__device__ __forceinline__ float packed_element(const uint8_t* row, uint32_t d) {
    return wide16<DT>(*reinterpret_cast<const uint16_t*>(row + (d >> 4) * kTile16 + (d & 15u) * 2));
}

// What a wave found out about one row of one head over some tokens: the largest score, the sum of e^(score - most),
// and the mean of the values by these weights, feature lane + 64 c in mean[c].
struct PackedRow {
    float most, sum, mean[4];
};

// One row: 64 tokens at a time, a lane forms the score of one token, then the lanes take the features, four
// tokens' values on their way together (with eight, 15.4 ms instead of 13.1 for the prompts below).  Running maximum,
// sum and mean (a sum of values may pass F32's range where their mean does not); everything in F32.  `apart` keeps the
// values apart that are not finite: an infinity shows however small its probability, also where that is zero in F32
// (not done before a mean has come out that is not finite: 4 prompts of up to 300 rows, 8 / 2 heads of 40, would take
// 184 us instead of 131).
// `q` is the row times 1 / sqrt(D), in LDS.  locate(n, &k_row, &v_row) says whether the row sees token n and where
// it lies; `there` is the address of any row (read, and not used, for a token that is not seen).
template <int DT, class Locate>
__device__ __forceinline__ PackedRow packed_row(uint32_t D, const float* q, uint32_t tokens, const uint8_t* there,
                                                bool apart, const Locate& locate) {
    const float inf = __builtin_inff();
    const uint32_t lane = threadIdx.x & 63u;
    PackedRow row = {-inf, 0.0f, {0, 0, 0, 0}};
    float wild[4] = {0, 0, 0, 0};
    for (uint32_t n0 = 0; n0 < tokens; n0 += 64) {
        const uint8_t *kr = nullptr, *vr = there;
        const bool seen = n0 + lane < tokens && locate(n0 + lane, &kr, &vr);
        float score = -inf;
        if (seen) {
            score = 0.0f;
            uint32_t d = 0;
            for (; d + 8 <= D; d += 8) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(kr + (d >> 4) * kTile16 + (d & 15u) * 2);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    score = __builtin_fmaf(q[d + j], wide16<DT>(w[j >> 1] >> (16 * (j & 1)) & 0xFFFFu), score);
            }
            for (; d < D; ++d) score = __builtin_fmaf(q[d], packed_element<DT>(kr, d), score);
        }
        float top = score;
        for (int off = 1; off < 64; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
        const float m2 = fmaxf(row.most, top);
        const float base = m2 == -inf ? 0.0f : m2;
        const float p = seen ? expf(score - base) : 0.0f;   // a NaN score stays one
        const float keep = row.most == -inf ? 0.0f : expf(row.most - base);
        float part = p;
        for (int off = 1; off < 64; off *= 2) part += __shfl_xor(part, off);
        const float kept = row.sum * keep;
        row.sum = kept + part;
        row.most = m2;
        const float inverse = row.sum == 0.0f ? 0.0f : 1.0f / row.sum, weight = p * inverse;
#pragma unroll
        for (int c = 0; c < 4; ++c) row.mean[c] *= kept * inverse;
        const uint64_t any = __ballot(seen);
        const uint64_t at = reinterpret_cast<uint64_t>(vr);
        for (uint32_t y0 = 0; y0 < 64; y0 += 4) {
            if (!((any >> y0) & 15u)) continue;
            float value[4][4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const uint8_t* of = reinterpret_cast<const uint8_t*>(
                        (uint64_t)__builtin_amdgcn_readlane((uint32_t)(at >> 32), y0 + y) << 32
                        | (uint32_t)__builtin_amdgcn_readlane((uint32_t)at, y0 + y));
#pragma unroll
                for (int c = 0; c < 4; ++c) value[y][c] = lane + 64 * c < D ? packed_element<DT>(of, lane + 64 * c) : 0.0f;
            }
            if (apart) {
#pragma unroll
                for (int y = 0; y < 4; ++y)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (fabsf(value[y][c]) < inf) continue;
                        if ((any >> (y0 + y)) & 1u) wild[c] += value[y][c];
                        value[y][c] = 0.0f;
                    }
            }
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                if (!((any >> (y0 + y)) & 1u)) continue;
                const float of_all = as_f32(__builtin_amdgcn_readlane(as_u32(weight), y0 + y));
#pragma unroll
                for (int c = 0; c < 4; ++c) row.mean[c] = __builtin_fmaf(of_all, value[y][c], row.mean[c]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (wild[c] != 0.0f) row.mean[c] += wild[c];
    return row;
}

// One wave = one row of one head.  For head sizes of no whole tiles, pages of another size than whole tiles, and
// as a check of the matrix cores' kernel: every row reads K and V for itself, bound by the latency of these reads
// and by F32 arithmetic (24 prompts of up to 1201 rows, 32 / 4 heads of 64: 13 ms, 5 TFLOP/s, where the matrix cores
// take 0.17 ms).
template <int DT>
__global__ __launch_bounds__(256) void sdpa_packed_rows_kernel(const SdpaPackedArgs a) {
    __shared__ float q_rows[4][kMaxPackedWidth];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t s = blockIdx.z;
    const PackedSequence seq = packed_sequence(a, s);
    const uint32_t rows = seq.rows < a.max_rows ? seq.rows : a.max_rows;
    const uint32_t head = blockIdx.y, hkv = divided(head, a.group, a.div_group);
    const uint8_t* kb = a.k + hkv * a.k_head;
    const uint8_t* vb = a.v + hkv * a.v_head;
    const int32_t* pages = a.table.base ? a.table.row(s) : nullptr;
    const uint32_t row_tiles = a.d_tiles * kTile16;
    for (uint32_t i = blockIdx.x * 4 + wave; i < rows; i += gridDim.x * 4) {
        const uint32_t t = seq.start + i;
        const uint64_t row_at = (uint64_t)(t >> 4) * row_tiles + (t & 15u) * 32;
        const uint8_t* qr = a.q + head * a.q_head + row_at;
        for (uint32_t d = lane; d < a.D; d += 64) q_rows[wave][d] = packed_element<DT>(qr, d) * a.scale;
        __builtin_amdgcn_wave_barrier();
        const uint32_t own = a.tree.base ? (a.tree.cols * 32 < seq.rows ? a.tree.cols * 32 : seq.rows) : i + 1;
        auto locate = [&](uint32_t x, const uint8_t** kr, const uint8_t** vr) -> bool {
            if (x >= seq.cached) {
                const uint32_t j = x - seq.cached, own_t = seq.start + j;
                if (a.tree.base && !(((uint32_t)a.tree.at(t, j >> 5) >> (j & 31u)) & 1u)) return false;
                const uint64_t at = (uint64_t)(own_t >> 4) * row_tiles + (own_t & 15u) * 32;
                *kr = kb + at;
                *vr = vb + at;
                return true;
            }
            const uint32_t slot = divided(x, a.page_rows, a.div_page_rows);
            const uint32_t page = (uint32_t)pages[(uint64_t)(slot >> 4) * kTileSlots + (slot & 15u)];
            if (page >= a.pages) return false;
            const uint32_t r = x - slot * a.page_rows;
            const uint64_t at = (uint64_t)(r >> 4) * row_tiles + (r & 15u) * 32;
            *kr = a.k_pages + page * a.k_page + hkv * a.k_page_head + at;
            *vr = a.v_pages + page * a.v_page + hkv * a.v_page_head + at;
            return true;
        };
        PackedRow row;
        for (bool apart = false;; apart = true) {
            row = packed_row<DT>(a.D, q_rows[wave], seq.cached + own, vb + row_at, apart, locate);
            bool finite = true;
#pragma unroll
            for (int c = 0; c < 4; ++c) finite = finite && fabsf(row.mean[c]) < __builtin_inff();
            if (apart || row.sum != row.sum || __all(finite)) break;
        }
        uint8_t* ob = a.out + (uint64_t)(t >> 4) * a.out_tile_cols * kTile16 + (t & 15u) * 32;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const uint32_t d = lane + 64 * c;
            if (d >= a.D) continue;
            const uint32_t col = head * a.D + d;
            *reinterpret_cast<uint16_t*>(ob + (uint64_t)(col >> 4) * kTile16 + (col & 15u) * 2) =
                    (uint16_t)narrow2<DT>(row.sum == 0.0f ? 0.0f : row.mean[c], 0.0f);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ---------------------------------------------------------------------------
// The matrix-core kernel.
//
// Rows m = i * group + g (row i of the sequence, head g of the KV head's group) are the columns of
// the matrix products.  S^T = K Q^T leaves in a lane scores of one column for runs of four
// consecutive tokens, and in that order they are the second operand of O^T = V^T P^T, whose first
// operand ds_read_b64_tr_b16 reads out of a V tile as it lies (sixteen lanes supply four token rows
// of a tile, 128 bytes, and receive a feature column each).  So scores and probabilities never leave
// their lane's registers, a column's statistics are one value per lane, and K and V go to LDS as
// they lie in memory, by the direct loader.
//
// Softmax in one pass: p = 2^(s * scale_log2 - ref), with a reference exponent per row that is moved
// (and the sums with it) only when a score exceeds it by more than kSlack: the sums may be up to
// 2^kSlack times larger than with the true maximum, which F32 does not notice, and most blocks of
// tokens need neither the maximum over lanes nor a pass over the sums.  p is rounded to the leaf for
// the second product (its error is half a step of each probability, as much as a value's own); the
// sum is taken of the unrounded ones.  F16 lifts p by 2^kLift so that small probabilities keep their
// bits: they are at most 2^(kLift + kSlack), and subnormal below 2^-22 of the largest.
//
// The sums may pass F32's range where their mean does not (BF16's range is as wide), and an infinite value meets
// probabilities of zero: a row with a sum near the range's end or past it is taken again, as the other kernel does
// (near_end).
//
// Long prompts are bound by the matrix and the vector units, busy for 0.43 and 0.44 of the cycles (8191 rows,
// 32 / 8 heads of 128 BF16: 565 to 610 us on different cards, 900 to 970 TFLOP/s, where library products of 4096^3
// to 16384^3 reach 1163 to 1337); shorter ones wait more (24 prompts of up to 1201 rows of 64: 170 us, 400
// TFLOP/s); single tokens are bound by memory (32 tokens over 700 to 15001 cached ones, 8 KV heads of 128: 195 us,
// 5.2 TB/s, where a bare read reaches 6.6).
//
// Only blocks that a row does not see in full (the ends of the cached prefix, the diagonal, trees,
// absent pages) form masks.  There V is cleared where no row may see it, and a value left that is
// not finite is taken out of the product (0 times infinity must not reach a row that does not see
// it): two more products count, for every row and feature, the infinities of either sign that the
// row sees, a NaN as both.
// ---------------------------------------------------------------------------

constexpr float kLowest = -3.4028234663852886e38f;
// 2^115, as bits: four teams' sums of this size and those of 1536 pieces (three for each of fewer than kPackedGroups
// row blocks at the most, see packed_room) add up to less than 2^127.6.
constexpr uint32_t kNearEnd = (127u + 115u) << 23;

typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

template <int DT> struct PackedLeaf;
template <> struct PackedLeaf<IOMX_DT_BF16> {
    static constexpr float kSlack = 8.0f, kLift = 0.0f;
    static constexpr uint32_t kExponent = 0x7F80u, kCarry = 0x0080u, kOne = 0x3F80u;
    static __device__ __forceinline__ f32x4_t mfma(u32x4 a, u32x4 b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16_t mfma(u32x4 a, u32x4 b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
    }
};
template <> struct PackedLeaf<IOMX_DT_F16> {
    static constexpr float kSlack = 6.0f, kLift = 8.0f;
    static constexpr uint32_t kExponent = 0x7C00u, kCarry = 0x0400u, kOne = 0x3C00u;
    static __device__ __forceinline__ f32x4_t mfma(u32x4 a, u32x4 b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16_t mfma(u32x4 a, u32x4 b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pair(float lo, float hi) {
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2));
    }
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4_t* tr_ptr_t;

// Sixteen lanes read 128 consecutive bytes, four rows of a tile of 16-bit elements; lane i of them
// receives column i.
__device__ __forceinline__ u32x2 read_transposed(const uint8_t* at) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr_t)(lptr_t)at));
}

// How a lane's values lie for products of W columns, KS = ceil(D / 32).  A "pair" is two token tiles
// (32 tokens); a lane holds kQuads runs of four tokens of it.
template <int DT, int KS, int W> struct PackedShape;

// v_mfma_f32_16x16x32: lane = column lane % 16, quarter lane / 16.
template <int DT, int KS> struct PackedShape<DT, KS, 16> {
    using Acc = f32x4_t;
    static constexpr int kSteps = KS;               // of the first product, 32 features each
    static constexpr int kScores = 2, kAccs = 2 * KS, kQuads = 2, kHalves = 1;
    static __device__ __forceinline__ uint32_t column(uint32_t lane) { return lane & 15u; }
    // feature tile and byte within its row that a lane supplies in step c
    static __device__ __forceinline__ uint32_t operand_tile(int c, uint32_t lane) { return 2 * c + (lane >> 5); }
    static __device__ __forceinline__ uint32_t operand_byte(uint32_t lane) { return ((lane >> 4) & 1u) * 16; }
    // sixteen-byte piece of a kilobyte that a lane of the loader brings
    static __device__ __forceinline__ uint32_t k_source(uint32_t lane, uint32_t) { return lane; }
    static __device__ __forceinline__ uint32_t v_source(uint32_t lane) { return lane; }
    // first operand of S^T: byte within the pair's stage, score tile t, step c
    static __device__ __forceinline__ uint32_t k_lane(uint32_t lane) { return (lane >> 5) * kTile16 + (lane & 15u) * 32 + operand_byte(lane); }
    static constexpr int k_at(int t, int c) { return t * KS * 1024 + c * 1024; }
    // tile of quad u, and which run of four tokens of it
    static constexpr int quad_tile(int u) { return u; }
    static __device__ __forceinline__ uint32_t quad_run(int, uint32_t lane) { return lane >> 4; }
    // first operand of O^T: 32 tokens of feature tile d
    static __device__ __forceinline__ uint32_t v_lane(uint32_t lane) { return lane * 8; }
    static constexpr int v_at(int d, int, int part) { return part * KS * 1024 + d * 512; }
    static constexpr int v_quad(int, int part) { return part; }
    // first feature of quad u of accumulator d
    static __device__ __forceinline__ uint32_t feature(int d, int, uint32_t lane) { return 16 * d + 4 * (lane >> 4); }
    static constexpr int kAccQuads = 1;
    static __device__ __forceinline__ float join(float x) { x = fmaxf(x, __shfl_xor(x, 16)); return fmaxf(x, __shfl_xor(x, 32)); }
    static __device__ __forceinline__ float add(float x) { x += __shfl_xor(x, 16); return x + __shfl_xor(x, 32); }
};

// v_mfma_f32_32x32x16: lane = column lane % 32, half lane / 32.
template <int DT, int KS> struct PackedShape<DT, KS, 32> {
    using Acc = f32x16_t;
    static constexpr int kSteps = 2 * KS;           // 16 features each
    static constexpr int kScores = 1, kAccs = KS, kQuads = 4, kHalves = 2;
    static __device__ __forceinline__ uint32_t column(uint32_t lane) { return lane & 31u; }
    static __device__ __forceinline__ uint32_t operand_tile(int c, uint32_t) { return c; }
    static __device__ __forceinline__ uint32_t operand_byte(uint32_t lane) { return (lane >> 5) * 16; }
    // The two token tiles of a pair would be read from the same banks at once, as would two feature
    // tiles of V: the second of either lies in LDS with its rows' halves, or its runs of four rows,
    // exchanged (a lane of the loader may take its sixteen bytes from anywhere).
    static __device__ __forceinline__ uint32_t k_source(uint32_t lane, uint32_t token_tile) { return lane ^ (token_tile & 1u); }
    static __device__ __forceinline__ uint32_t v_source(uint32_t lane) { return lane ^ (lane >> 5) * 8; }
    static __device__ __forceinline__ uint32_t k_lane(uint32_t lane) {
        const uint32_t second = (lane >> 4) & 1u;
        return second * (KS * 1024) + (lane & 15u) * 32 + ((lane >> 5) ^ second) * 16;
    }
    static constexpr int k_at(int, int c) { return c * 512; }
    static constexpr int quad_tile(int u) { return u >> 1; }
    static __device__ __forceinline__ uint32_t quad_run(int u, uint32_t lane) { return 2 * (u & 1) + (lane >> 5); }
    // sixteen tokens (tile h) of feature tiles 2 d and 2 d + 1
    static __device__ __forceinline__ uint32_t v_lane(uint32_t lane) {
        const uint32_t second = (lane >> 4) & 1u;
        return second * 512 + ((lane >> 5) ^ second) * 128 + (lane & 15u) * 8;
    }
    static constexpr int v_at(int d, int h, int part) { return h * KS * 1024 + d * 1024 + part * 256; }
    static constexpr int v_quad(int h, int part) { return 2 * h + part; }
    static __device__ __forceinline__ uint32_t feature(int d, int u, uint32_t lane) { return 32 * d + 8 * u + 4 * (lane >> 5); }
    static constexpr int kAccQuads = 4;
    static __device__ __forceinline__ float join(float x) { return fmaxf(x, __shfl_xor(x, 32)); }
    static __device__ __forceinline__ float add(float x) { return x + __shfl_xor(x, 32); }
};

// Where the tokens of a row block lie: `prefix` tiles of the cache, then tiles of the packed rows.
struct PackedTiles {
    uint32_t cached, prefix;      // cached tokens, their tiles
    uint32_t first;               // first tile of the packed rows
    uint32_t count;               // all tiles
};

// Where few row blocks meet long contexts, a row block's tokens are shared out among workgroups,
// every one of which takes the same number of token blocks: the lengths are on the device, so each
// wave adds up the work of all sequences (a sequence per lane), divides it by the workgroups there is
// room for, and looks up its own piece in the running count.  Pieces are rounded up, so there may be
// one more for every row block: where that is the lesser part, the size is chosen for all pieces to
// run at once (eight drafted trees: 544 pieces of 12 blocks take a second turn on 512 places), else
// the smaller size evens out the lengths over several turns.
constexpr uint32_t kPackedGroups = 512;   // two workgroups for each CU
// Tokens of a piece at the least.  A piece costs a second launch and its sums' way through memory:
// sixteen sequences of up to 509 cached tokens and one row each (4 KV heads of 64) take 9.3 us on 64
// workgroups and 12.3 us in pieces of 128.
constexpr uint32_t kPackedLeastTokens = 512;

// Pieces to divide the work of a KV head into, for `row_blocks` row blocks.  Blocks of many rows leave
// large parts behind, so they are not divided further than there is room.
template <uint32_t BM>
__host__ __device__ constexpr uint32_t packed_room(uint32_t places, uint32_t row_blocks) {
    return 2 * row_blocks <= places ? places - row_blocks : BM <= 32 ? 2 * row_blocks : places;
}

struct PackedShare {
    uint32_t s, row_block, piece, pieces, size;   // size: token blocks of a piece
    uint32_t first;                               // index of the sequence's first piece (per KV head)
    PackedSequence seq;
};

// The share of piece number `index`, or (find_sequence) of sequence `index`; s = ~0 if there is none.
template <uint32_t BM, uint32_t NT>
__device__ __forceinline__ PackedShare packed_share(const SdpaPackedArgs& a, uint32_t index, bool find_sequence) {
    const uint32_t lane = threadIdx.x & 63u;
    PackedSequence seq = {};
    auto work = [&](uint32_t s, uint32_t* blocks) __attribute__((always_inline)) -> uint32_t {
        *blocks = 0;
        if (s >= a.sequences) return 0;
        seq = packed_sequence(a, s);
        const uint32_t rows = seq.rows < a.max_rows ? seq.rows : a.max_rows;
        if (!rows) return 0;
        const uint32_t tiles = ((seq.cached + 15) >> 4) + ((seq.start + seq.rows + 15) >> 4) - (seq.start >> 4);
        *blocks = (tiles + NT - 1) / NT;
        return (rows * a.group + BM - 1) / BM;
    };
    uint32_t blocks, row_blocks = work(lane, &blocks);
    uint64_t total = (uint64_t)row_blocks * blocks;
    uint32_t all_rows = row_blocks;
    for (uint32_t s = 64 + lane; s - lane < a.sequences; s += 64) {
        uint32_t more;
        const uint32_t n = work(s, &more);
        total += (uint64_t)n * more;
        all_rows += n;
    }
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        total += __shfl_xor((unsigned long long)total, off);
        all_rows += __shfl_xor(all_rows, off);
    }
    PackedShare p = {};
    const uint32_t room = packed_room<BM>(a.places, all_rows);
    const uint64_t even = total >> 31 ? (total + room - 1) / room : ((uint32_t)total + room - 1) / room;
    constexpr uint32_t least = kPackedLeastTokens / (16 * NT);
    // (the same in every lane, and known to be: what is formed from it goes to the scalar unit)
    p.size = __builtin_amdgcn_readfirstlane(even > least ? (uint32_t)even : least);
    p.s = ~0u;
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < a.sequences; s0 += 64) {
        if (a.sequences > 64) row_blocks = work(s0 + lane, &blocks);
        const uint32_t pieces = (blocks + p.size - 1) / p.size, count = row_blocks * pieces;
        uint32_t upto = count;
#pragma unroll
        for (int off = 1; off < 64; off *= 2) {
            const uint32_t lower = __shfl_up(upto, off);
            if (lane >= (uint32_t)off) upto += lower;
        }
        const uint64_t here = __ballot(find_sequence ? s0 + lane == index : before + upto > index);
        if (here) {
            const int at = __ffsll((unsigned long long)here) - 1;
            p.s = s0 + at;
            p.pieces = __builtin_amdgcn_readlane(pieces, at);
            p.first = before + __builtin_amdgcn_readlane(upto - count, at);
            p.seq.start = __builtin_amdgcn_readlane(seq.start, at);
            p.seq.rows = __builtin_amdgcn_readlane(seq.rows, at);
            p.seq.cached = __builtin_amdgcn_readlane(seq.cached, at);
            if (!find_sequence) {
                p.row_block = (index - p.first) / p.pieces;
                p.piece = index - p.first - p.row_block * p.pieces;
            }
            return p;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return p;
}

// The block of rows that a workgroup takes (m_block .. of m_end rows times heads) and its token blocks.
struct PackedBlock {
    uint32_t s, hkv, pieces, m_block, m_end;
    uint32_t own;                 // own rows that some row of the block sees
    uint32_t begin, end;          // token blocks
    PackedSequence seq;
    PackedTiles tiles;
};
// false: there is none for this workgroup
template <uint32_t BM, uint32_t NT>
__device__ __forceinline__ bool packed_block(const SdpaPackedArgs& a, PackedBlock* p) {
    uint32_t rb, piece = 0, size = 0;
    p->pieces = 1;
    if (a.places) {
        const uint32_t index = divided(blockIdx.x, a.Hkv, a.div_hkv);
        p->hkv = blockIdx.x - index * a.Hkv;
        const PackedShare share = packed_share<BM, NT>(a, index, false);
        if (share.s == ~0u) return false;
        p->s = share.s; rb = share.row_block; piece = share.piece; p->pieces = share.pieces; size = share.size;
        p->seq = share.seq;
    } else {
        // unit (sequence, KV head) fastest: consecutive workgroups go to different dies, a unit's row
        // blocks to the same one where the units are a multiple of eight.  Late rows, which see the
        // most, go first.
        const uint32_t units = a.sequences * a.Hkv;
        const uint32_t rb_up = divided(blockIdx.x, units, a.div_units), unit = blockIdx.x - rb_up * units;
        rb = a.row_blocks - 1 - rb_up;
        p->s = divided(unit, a.Hkv, a.div_hkv);
        p->hkv = unit - p->s * a.Hkv;
        p->seq = packed_sequence(a, p->s);
    }
    const uint32_t rows = p->seq.rows < a.max_rows ? p->seq.rows : a.max_rows;
    p->m_end = rows * a.group;
    p->m_block = rb * BM;
    if (p->m_block >= p->m_end) return false;
    if (a.tree.base) p->own = a.tree.cols * 32 < p->seq.rows ? a.tree.cols * 32 : p->seq.rows;
    else {
        const uint32_t m_last = p->m_block + BM < p->m_end ? p->m_block + BM - 1 : p->m_end - 1;
        p->own = divided(m_last, a.group, a.div_group) + 1;
    }
    p->tiles.cached = p->seq.cached;
    p->tiles.prefix = (p->seq.cached + 15) >> 4;
    p->tiles.first = p->seq.start >> 4;
    p->tiles.count = p->tiles.prefix + ((p->seq.start + p->own + 15) >> 4) - p->tiles.first;
    const uint32_t blocks = (p->tiles.count + NT - 1) / NT;
    p->begin = 0;
    p->end = blocks;
    if (p->pieces > 1) {
        p->begin = piece * size;
        p->end = p->begin + size < blocks ? p->begin + size : blocks;
    }
    return true;
}

// A row of the workgroup's block over the block's tokens once more, by one wave, and to its place; `q` is LDS of the
// wave's own.  A function that is called, and finds out everything anew from the kernel's arguments: inlined, what this
// (hardly ever taken) path needs is kept in registers through the main loop (prompts of heads of 64: 181 us instead
// of 173).  It reads K and V for every row: where all values are 1e38, 4096 rows of 32 / 8 heads of 128 take 50 ms
// instead of 0.18, 32 single tokens over 700 to 15001 cached ones 5.8 ms instead of 0.2.
template <int DT, uint32_t BM, uint32_t NT>
static __device__ __attribute__((noinline, cold)) void packed_again(const SdpaPackedArgs* args, float* q, uint32_t row_in_block) {
    const SdpaPackedArgs& a = *args;
    PackedBlock b;
    if (!packed_block<BM, NT>(a, &b)) return;
    const uint32_t m = b.m_block + row_in_block;
    if (m >= b.m_end) return;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t i = divided(m, a.group, a.div_group), t = b.seq.start + i;
    const uint32_t head = b.hkv * a.group + (m - i * a.group);
    const uint32_t row_tiles = a.d_tiles * kTile16;
    const uint64_t row_at = (uint64_t)(t >> 4) * row_tiles + (t & 15u) * 32;
    const uint8_t* qr = a.q + head * a.q_head + row_at;
    __builtin_amdgcn_wave_barrier();
    for (uint32_t d = lane; d < a.D; d += 64) q[d] = packed_element<DT>(qr, d) * a.scale;
    __builtin_amdgcn_wave_barrier();
    const uint32_t visible = a.tree.base ? b.own : i + 1;
    const uint8_t *kb = a.k + b.hkv * a.k_head, *vb = a.v + b.hkv * a.v_head;
    const PackedRow row = packed_row<DT>(a.D, q, (b.end - b.begin) * NT * 16, vb + row_at, true,
                                         [&](uint32_t n, const uint8_t** kr, const uint8_t** vr) -> bool {
        const uint32_t x = b.begin * NT + (n >> 4), r = n & 15u;        // tile, row in it
        if (x >= b.tiles.prefix) {
            const uint32_t tile = b.tiles.first + x - b.tiles.prefix, j = tile * 16 + r - b.seq.start;
            if (j >= visible) return false;                             // (rows before the first one wrap)
            if (a.tree.base && !(((uint32_t)a.tree.at(t, j >> 5) >> (j & 31u)) & 1u)) return false;
            *kr = kb + (uint64_t)tile * row_tiles + r * 32;
            *vr = vb + (uint64_t)tile * row_tiles + r * 32;
            return true;
        }
        if (x * 16 + r >= b.tiles.cached) return false;
        const uint32_t slot = divided(x, a.page_tiles, a.div_page_tiles);
        const uint32_t page = (uint32_t)a.table.at(b.s, slot);
        if (page >= a.pages) return false;
        const uint64_t at = (uint64_t)(x - slot * a.page_tiles) * row_tiles + r * 32;
        *kr = a.k_pages + page * a.k_page + b.hkv * a.k_page_head + at;
        *vr = a.v_pages + page * a.v_page + b.hkv * a.v_page_head + at;
        return true;
    });
    // A part's sum of probabilities is brought to 2^-14 .. 2^-13 by a power of two, which its reference takes up (next to
    // the 2^kLift that the other parts' sums hold): the unnormalised sums are then far from the end.
    int32_t exponent = 0;
    if (row.sum > 0.0f) exponent = (int32_t)(as_u32(row.sum) >> 23) - 126 + 13;
    const float l = __builtin_ldexpf(row.sum, -exponent);
    uint8_t* to = a.out + ((uint64_t)(t >> 4) * a.out_tile_cols + head * a.d_tiles) * kTile16 + (t & 15u) * 32;
    const uint64_t part = (uint64_t)blockIdx.x * BM + row_in_block;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t d = lane + 64 * c;
        if (d >= a.D) continue;
        const float mean = row.mean[c];
        if (b.pieces > 1) a.parts[part * a.D + d] = row.sum == 0.0f ? mean : mean * l;
        else *reinterpret_cast<uint16_t*>(to + (d >> 4) * kTile16 + (d & 15u) * 2) = (uint16_t)narrow2<DT>(row.sum == 0.0f ? 0.0f : mean, 0.0f);
    }
    if (b.pieces > 1 && lane == 0) {
        a.part_stats[part * 2] = row.sum == 0.0f ? kLowest : row.most * 1.44269504088896340736f + (float)exponent + PackedLeaf<DT>::kLift;
        a.part_stats[part * 2 + 1] = l;
    }
}

// Waves per SIMD: as many workgroups as the stages leave room for in the LDS of a CU, up to two, or
// three where the registers last (packed prompts of heads of 64 take 169 us with three and 216 us
// with two).
constexpr int packed_waves(int KS, int WQ, int NT) {
    const int fit = 160 * 1024 / (4 * (4 / WQ) * NT * KS * 1024 + 2048), most = KS <= 2 && WQ == 4 ? 3 : 2;
    return fit < 1 ? 1 : fit < most ? fit : most;
}

// WQ of the four waves share out the rows of the block and read the same tokens from LDS; the
// 4 / WQ teams of them share out the tokens.  A wave has QT times W columns; NT token tiles are in
// LDS per team and stage.
template <int DT, int KS, int W, int QT, int WQ, int NT>
__global__ __launch_bounds__(256, packed_waves(KS, WQ, NT)) void sdpa_packed_mfma_kernel(const SdpaPackedArgs a) {
    using Leaf = PackedLeaf<DT>;
    using Shape = PackedShape<DT, KS, W>;
    using Acc = typename Shape::Acc;
    constexpr int WK = 4 / WQ, DTL = 2 * KS, QUADS = Shape::kQuads;
    constexpr bool kScarce = packed_waves(KS, WQ, NT) == 3 || (KS == 8 && W == 32);     // registers are
    constexpr uint32_t BM = W * QT * WQ, kStage = NT * KS * 1024;
    // Two stages of K and V, variables of their own and named where they are used: the compiler then
    // knows that a read of one need not wait for the loader's writes to the other.
    __shared__ __attribute__((aligned(1024))) uint8_t k_even[WK][kStage], k_odd[WK][kStage];
    __shared__ __attribute__((aligned(1024))) uint8_t v_even[WK][kStage], v_odd[WK][kStage];
    // For packed_again: the address of `a` (the one argument) waits in LDS, for where it is in registers the compiler reads
    // the arguments again and again in the main loop instead of keeping them.
    __shared__ float q_again[4][32 * KS];
    __shared__ const SdpaPackedArgs* args_at;
    args_at = (const SdpaPackedArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    const uint32_t lane = threadIdx.x & 63u, column = Shape::column(lane);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t team = wave / WQ, member = wave % WQ;

    PackedBlock block;
    if (!packed_block<BM, NT>(a, &block)) return;
    const uint32_t s = block.s, hkv = block.hkv, pieces = block.pieces, m_end = block.m_end, m_block = block.m_block;
    const uint32_t b_begin = block.begin, b_end = block.end;
    const PackedSequence seq = block.seq;
    const PackedTiles tiles = block.tiles;

    // this wave's columns: rows of the sequence, and the wave's range of them
    const uint32_t m_wave = m_block + member * W * QT;
    uint32_t row_of[QT];
#pragma unroll
    for (int q = 0; q < QT; ++q) row_of[q] = divided(m_wave + W * q + column, a.group, a.div_group);
    const bool idle = m_wave >= m_end;
    const uint32_t row_tiles = a.d_tiles * kTile16;
    // Feature tiles that a token tile's stage has room for and that there are none of (the last one; of
    // heads above 128 up to three) are not loaded: those of K meet zeros of Q and have to be
    // finite, those of V are in no output.
    constexpr uint32_t kSpare = KS > 4 ? 3 : 1;
    const uint32_t spare = DTL - a.d_tiles;

    u32x4 qf[QT][Shape::kSteps];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        const uint32_t m = m_wave + W * q + column, t = seq.start + row_of[q];
        const uint32_t head = hkv * a.group + (m - row_of[q] * a.group);
        const uint8_t* qr = a.q + head * a.q_head + (uint64_t)(t >> 4) * row_tiles + (t & 15u) * 32 + Shape::operand_byte(lane);
#pragma unroll
        for (int c = 0; c < Shape::kSteps; ++c) {
            const uint32_t tile = Shape::operand_tile(c, lane);
            qf[q][c] = u32x4{0, 0, 0, 0};
            if (m < m_end && tile < a.d_tiles) qf[q][c] = *reinterpret_cast<const u32x4*>(qr + tile * kTile16);
        }
    }
    if (spare) {
        for (uint32_t i = threadIdx.x; i < WK * NT * kSpare * 32; i += 256) {
            const uint32_t tile = DTL - kSpare + (i >> 5) % kSpare;
            if (tile < a.d_tiles) continue;
            const uint32_t at = i / (kSpare * 32) * (KS * 1024) + tile * kTile16 + (i & 31u) * 16;
            *reinterpret_cast<u32x4*>(&k_even[0][0] + at) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(&k_odd[0][0] + at) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(&v_even[0][0] + at) = u32x4{0, 0, 0, 0};
            *reinterpret_cast<u32x4*>(&v_odd[0][0] + at) = u32x4{0, 0, 0, 0};
        }
        __syncthreads();
    }

    // page numbers of a block's tiles, one per lane below NT.  The number is not looked at before the
    // block's turn (present_of): a comparison here would wait for the load, and with it for every
    // tile on its way to LDS.
    auto block_pages = [&](uint32_t b) __attribute__((always_inline)) -> uint32_t {
        if (b >= b_end || b * NT >= tiles.prefix) return 0u;
        const uint32_t x = b * NT + lane;
        if (lane >= NT || x >= tiles.prefix) return 0u;
        return (uint32_t)a.table.at(s, divided(x, a.page_tiles, a.div_page_tiles));
    };
    auto present_of = [&](uint32_t b, uint32_t pages) __attribute__((always_inline)) -> uint32_t {
        if (b >= b_end) return 0u;
        if (b * NT >= tiles.prefix) return tiles.count - b * NT >= NT ? (1u << NT) - 1u : (1u << (tiles.count - b * NT)) - 1u;
        const uint32_t x = b * NT + lane;
        return (uint32_t)__ballot(lane < NT && x < tiles.count && (x >= tiles.prefix || pages < a.pages));
    };
    // brings the tiles of block b that are present to a stage: a wave of the team takes every WQ-th
    auto fetch = [&](uint32_t b, uint32_t pages, uint32_t present, uint8_t* ks, uint8_t* vs) __attribute__((always_inline)) {
        // (where registers are scarce, not to be known as the same lane every time: the addresses formed
        // from it would be kept in registers throughout the loop)
        uint32_t own_lane = lane;
        if constexpr (kScarce) asm volatile("" : "+v"(own_lane));
#pragma unroll
        for (int n = 0; n < NT / WQ; ++n) {
            const uint32_t at = member + n * WQ;
            const uint32_t x = b * NT + at;
            const uint32_t page = __builtin_amdgcn_readlane(pages, at);
            if (!((present >> at) & 1u)) continue;
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
                if (2 * c + 2 > DTL - (int)kSpare && spare && 2 * c + (lane >> 5) >= a.d_tiles) break;
                __builtin_amdgcn_global_load_lds((gptr_t)(kt + c * 1024 + Shape::k_source(own_lane, at) * 16), (lptr_t)(ks + at * (KS * 1024) + c * 1024), 16, 0, 0);
                __builtin_amdgcn_global_load_lds((gptr_t)(vt + c * 1024 + Shape::v_source(own_lane) * 16), (lptr_t)(vs + at * (KS * 1024) + c * 1024), 16, 0, 0);
            }
        }
    };

    Acc acc[Shape::kAccs][QT];
    float ref[QT], sum[QT];
#pragma unroll
    for (int q = 0; q < QT; ++q) {
        ref[q] = kLowest;
        sum[q] = 0.0f;
#pragma unroll
        for (int d = 0; d < Shape::kAccs; ++d) acc[d][q] = Acc{};
    }
    // tiles that every row of this wave sees in full, and the first that none of them sees
    const uint32_t whole_prefix = tiles.cached >> 4;
    const uint32_t whole_first = tiles.prefix + ((seq.start + 15) >> 4) - tiles.first;
    uint32_t whole_end = 0, past = ~0u;
    if (!a.tree.base) {
        whole_end = tiles.prefix + ((seq.start + divided(m_wave, a.group, a.div_group) + 1) >> 4) - tiles.first;
        past = tiles.prefix + ((seq.start + divided(m_wave + W * QT - 1, a.group, a.div_group)) >> 4) + 1 - tiles.first;
    }
    const uint32_t k_lane = Shape::k_lane(lane), v_lane = Shape::v_lane(lane);

    // scores of a pair: [column tile][score tile]
    auto scores = [&](const uint8_t* ks, Acc (&sc)[QT][Shape::kScores]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < Shape::kScores; ++t) {
#pragma unroll
            for (int q = 0; q < QT; ++q) sc[q][t] = Acc{};
#pragma unroll
            for (int c = 0; c < Shape::kSteps; ++c) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(ks + Shape::k_at(t, c) + k_lane);
#pragma unroll
                for (int q = 0; q < QT; ++q) sc[q][t] = Leaf::mfma(kf, qf[q][c], sc[q][t]);
            }
        }
    };
    // largest score of each column over N pairs, as an exponent of two
    auto largest = [&](auto& sc, float (&top)[QT]) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            float most = -__builtin_inff();
#pragma unroll
            for (uint32_t n = 0; n < sizeof(sc) / sizeof(sc[0]); ++n)
#pragma unroll
                for (int t = 0; t < Shape::kScores; ++t)
#pragma unroll
                    for (int j = 0; j < 4 * QUADS / Shape::kScores; j += 2)
                        most = fmaxf(fmaxf(most, sc[n][q][t][j]), sc[n][q][t][j + 1]);
            top[q] = most * a.scale_log2;
        }
    };
    auto beyond = [&](float (&top)[QT]) __attribute__((always_inline)) -> bool {
        bool any = false;
#pragma unroll
        for (int q = 0; q < QT; ++q) any = any || top[q] > ref[q] + Leaf::kSlack;
        return __any(any);
    };
    // probabilities of a pair, as the second product takes them: words 2 u, 2 u + 1 of quad u
    auto probabilities = [&](Acc (&sc)[QT][Shape::kScores], uint32_t (&pw)[QT][2 * QUADS]) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const float minus = Leaf::kLift - ref[q];
#pragma unroll
            for (int u = 0; u < QUADS; ++u) {
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[q][W == 16 ? u : 0][W == 16 ? j : 4 * u + j], a.scale_log2, minus));
                sum[q] += (p[0] + p[1]) + (p[2] + p[3]);
                pw[q][2 * u] = Leaf::pair(p[0], p[1]);
                pw[q][2 * u + 1] = Leaf::pair(p[2], p[3]);
            }
        }
    };
    // V of a pair's tokens (half h of them), accumulator d, as the second product takes it
    auto values = [&](const uint8_t* vs, int d, int h) __attribute__((always_inline)) {
        const u32x2 lo = read_transposed(vs + Shape::v_at(d, h, 0) + v_lane), hi = read_transposed(vs + Shape::v_at(d, h, 1) + v_lane);
        return u32x4{lo.x, lo.y, hi.x, hi.y};
    };
    auto words = [&](uint32_t (&w)[2 * QUADS], int h) __attribute__((always_inline)) {
        return u32x4{w[4 * h], w[4 * h + 1], w[4 * h + 2], w[4 * h + 3]};
    };
    // (kYield: with two waves on a SIMD the one at its vector instructions goes first, since the other's matrix
    // instructions run on by themselves: 581 us instead of 591 for the long prompt, 51.5 instead of 53 for trees; with
    // three, short prompts take 176 us instead of 173.)
    constexpr bool kYield = packed_waves(KS, WQ, NT) == 2;
    // A block that every row of the wave sees in full and whose scores are below the references, which
    // the wave's first block sets; false if they are not (nothing is changed then: any_pair takes the
    // block, and the sums, which only it scales, keep their registers here).
    bool begun = false;
    auto whole_block = [&](const uint8_t* ks, const uint8_t* vs) __attribute__((always_inline)) -> bool {
        Acc sc[NT / 2][QT][Shape::kScores];
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) scores(ks + n * (2 * KS * 1024), sc[n]);
        if constexpr (kYield) __builtin_amdgcn_s_setprio(1);
        float top[QT];
        largest(sc, top);
        if (!begun) {
#pragma unroll
            for (int q = 0; q < QT; ++q) ref[q] = fmaxf(Shape::join(top[q]), kLowest);
        } else if (beyond(top)) {
            if constexpr (kYield) __builtin_amdgcn_s_setprio(0);
            return false;
        }
#pragma unroll
        for (int n = 0; n < NT / 2; ++n) {
            uint32_t pw[QT][2 * QUADS];
            if constexpr (kYield) __builtin_amdgcn_s_setprio(1);
            probabilities(sc[n], pw);
            if constexpr (kYield) __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int h = 0; h < Shape::kHalves; ++h)
#pragma unroll
                for (int d = 0; d < Shape::kAccs; ++d) {
                    const u32x4 vf = values(vs + n * (2 * KS * 1024), d, h);
#pragma unroll
                    for (int q = 0; q < QT; ++q) acc[d][q] = Leaf::mfma(vf, words(pw[q], h), acc[d][q]);
                }
        }
        return true;
    };
    // Two token tiles x, x + 1, with masks where the wave does not see both in full.
    auto any_pair = [&](uint32_t x, uint32_t present, const uint8_t* ks, const uint8_t* vs) __attribute__((always_inline)) {
        if (!present || x >= past) return;
        const bool whole = present == 3u && (x + 2 <= whole_prefix || (x >= whole_first && x + 2 <= whole_end));
        Acc sc[1][QT][Shape::kScores];
        scores(ks, sc[0]);
        uint32_t seen[QT];                  // bit 4 u + j: the column sees token j of quad u
        uint32_t keep[2 * QUADS];           // V words (two tokens each) that some row may see
        bool ragged = false;                // there are tokens that none may see
        if (!whole) {
#pragma unroll
            for (int q = 0; q < QT; ++q) seen[q] = 0;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const uint32_t y = x + t;
                uint32_t any = 0;               // bit: token of the tile
                uint32_t bits[QT];
#pragma unroll
                for (int q = 0; q < QT; ++q) bits[q] = 0;
                if ((present >> t) & 1u) {
                    if (y < tiles.prefix) {
                        const uint32_t left = tiles.cached - y * 16;
                        any = left < 16 ? (1u << left) - 1u : 0xFFFFu;
#pragma unroll
                        for (int q = 0; q < QT; ++q) bits[q] = any;
                    } else {
                        // own rows j .. j + 15 of the sequence (j < 0: rows before the first)
                        const int32_t j = (int32_t)((tiles.first + y - tiles.prefix) * 16) - (int32_t)seq.start;
                        any = j < 0 ? 0xFFFFu << -j & 0xFFFFu : 0xFFFFu;
                        const int32_t left = (int32_t)seq.rows - j;
                        if (left < 16) any &= (1u << left) - 1u;
#pragma unroll
                        for (int q = 0; q < QT; ++q) {
                            if (a.tree.base) {
                                if (m_wave + W * q + column < m_end) {
                                    uint32_t row = seq.start + row_of[q];
                                    if constexpr (kScarce) asm volatile("" : "+v"(row));   // (as in fetch)
                                    const int32_t w = j >> 5;              // -1 for the rows before the first
                                    const uint32_t lo = w >= 0 && w < (int32_t)a.tree.cols ? (uint32_t)a.tree.at(row, w) : 0u;
                                    const uint32_t hi = w + 1 < (int32_t)a.tree.cols ? (uint32_t)a.tree.at(row, w + 1) : 0u;
                                    bits[q] = (uint32_t)((((uint64_t)hi << 32) | lo) >> (j & 31)) & any;
                                }
                            } else {
                                const int32_t last = (int32_t)row_of[q] - j;   // the last one it sees
                                bits[q] = (last < 0 ? 0u : last < 15 ? (2u << last) - 1u : 0xFFFFu) & any;
                            }
                        }
                    }
                }
                ragged = ragged || any != 0xFFFFu;
#pragma unroll
                for (int u = 0; u < QUADS; ++u) {
                    if (Shape::quad_tile(u) != t) continue;
                    const uint32_t run = 4 * Shape::quad_run(u, lane);
                    const uint32_t k4 = any >> run;
                    keep[2 * u] = ((k4 & 1u) ? 0xFFFFu : 0u) | ((k4 & 2u) ? 0xFFFF0000u : 0u);
                    keep[2 * u + 1] = ((k4 & 4u) ? 0xFFFFu : 0u) | ((k4 & 8u) ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int q = 0; q < QT; ++q) seen[q] |= (bits[q] >> run & 15u) << (4 * u);
                }
            }
#pragma unroll
            for (int q = 0; q < QT; ++q)
#pragma unroll
                for (int u = 0; u < QUADS; ++u)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float now = sc[0][q][W == 16 ? u : 0][W == 16 ? j : 4 * u + j];
                        sc[0][q][W == 16 ? u : 0][W == 16 ? j : 4 * u + j] = (seen[q] >> (4 * u + j)) & 1u ? now : -__builtin_inff();
                    }
        }
        // scores beyond the references move them
        float top[QT];
        largest(sc, top);
        if (beyond(top)) {
#pragma unroll
            for (int q = 0; q < QT; ++q) {
                const float r = fmaxf(Shape::join(top[q]), ref[q]);
                const float factor = __builtin_amdgcn_exp2f(ref[q] - r);
                ref[q] = r;
                sum[q] *= factor;
#pragma unroll
                for (int d = 0; d < Shape::kAccs; ++d) acc[d][q] *= factor;
            }
        }
        uint32_t pw[QT][2 * QUADS];
        probabilities(sc[0], pw);
#pragma unroll
        for (int h = 0; h < Shape::kHalves; ++h) {
            u32x4 vf[Shape::kAccs];
#pragma unroll
            for (int d = 0; d < Shape::kAccs; ++d) vf[d] = values(vs, d, h);
            if (!whole) {
                if (ragged) {
#pragma unroll
                    for (int d = 0; d < Shape::kAccs; ++d)
#pragma unroll
                        for (int w = 0; w < 4; ++w) vf[d][w] &= keep[4 * h + w];
                }
                // the largest magnitude of each half: an exponent field of all ones is above every other
                u16x2_t wild = {0, 0};
#pragma unroll
                for (int d = 0; d < Shape::kAccs; ++d)
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        wild = __builtin_elementwise_max(wild, __builtin_bit_cast(u16x2_t, vf[d][w] & 0x7FFF7FFFu));
                if (__any(wild.x >= Leaf::kExponent || wild.y >= Leaf::kExponent)) {
#pragma unroll
                    for (int q = 0; q < QT; ++q) {
                        u32x4 ones;
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t two = seen[q] >> (2 * (4 * h + w));
                            ones[w] = ((two & 1u) ? Leaf::kOne : 0u) | ((two & 2u) ? Leaf::kOne << 16 : 0u);
                        }
#pragma unroll
                        for (int d = 0; d < Shape::kAccs; ++d) {
#pragma unroll 1
                            for (uint32_t sign = 0; sign < 2; ++sign) {
                                u32x4 special;
#pragma unroll
                                for (int w = 0; w < 4; ++w) {
                                    special[w] = 0;
#pragma unroll
                                    for (int half = 0; half < 32; half += 16) {
                                        const uint32_t e = vf[d][w] >> half & 0xFFFFu, size = e & 0x7FFFu;
                                        special[w] |= (size > Leaf::kExponent || (size == Leaf::kExponent && e >> 15 == sign) ? Leaf::kOne : 0u) << half;
                                    }
                                }
                                const Acc n = Leaf::mfma(special, ones, Acc{});
#pragma unroll
                                for (int j = 0; j < 4 * Shape::kAccQuads; ++j)
                                    if (n[j] > 0.0f) acc[d][q][j] += sign ? -__builtin_inff() : __builtin_inff();
                            }
                        }
                    }
#pragma unroll
                    for (int d = 0; d < Shape::kAccs; ++d)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t up = ((vf[d][w] & 0x7FFF7FFFu) + (Leaf::kCarry | Leaf::kCarry << 16)) & 0x80008000u;
                            vf[d][w] &= ~(up | (up - (up >> 15)));     // both halves' bits under an all-ones exponent
                        }
                }
            }
#pragma unroll
            for (int d = 0; d < Shape::kAccs; ++d)
#pragma unroll
                for (int q = 0; q < QT; ++q) acc[d][q] = Leaf::mfma(vf[d], words(pw[q], h), acc[d][q]);
        }
    };

    // Two stages: while a block is computed, the direct loader fills the other one.  The wait and
    // the barrier at the top make the block's tiles visible to the team and the other stage free.
    // The teams take turns at the blocks, and as many turns each.
    uint32_t next_pages = block_pages(b_begin + team);
    uint32_t present = present_of(b_begin + team, next_pages);
    fetch(b_begin + team, next_pages, present, k_even[team], v_even[team]);
    next_pages = block_pages(b_begin + team + WK);
    auto step = [&](uint32_t b, auto stage) __attribute__((always_inline)) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0070);        // vmcnt(0), lgkmcnt(0)
        if constexpr (WQ > 1) __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const uint32_t here = present;
        present = present_of(b + WK, next_pages);
        if constexpr (decltype(stage)::value) fetch(b + WK, next_pages, present, k_even[team], v_even[team]);
        else fetch(b + WK, next_pages, present, k_odd[team], v_odd[team]);
        next_pages = block_pages(b + 2 * WK);
        if (idle) return;
        const uint8_t *ks, *vs;
        if constexpr (decltype(stage)::value) { ks = &k_odd[team][0]; vs = &v_odd[team][0]; }
        else { ks = &k_even[team][0]; vs = &v_even[team][0]; }
        const uint32_t x = b * NT;
        if (here == (1u << NT) - 1u && (x + NT <= whole_prefix || (x >= whole_first && x + NT <= whole_end)) && whole_block(ks, vs)) {
            begun = true;
            return;
        }
        begun = true;
#pragma unroll 1
        for (uint32_t n = 0; n < NT / 2; ++n)
            any_pair(x + 2 * n, (here >> (2 * n)) & 3u, ks + n * 2 * KS * 1024, vs + n * 2 * KS * 1024);
    };
    for (uint32_t b = b_begin; b < b_end; b += 2 * WK) {
        step(b + team, std::false_type{});
        if (b + WK >= b_end) break;
        step(b + WK + team, std::true_type{});
    }
    // the columns' sums over the lanes that hold them
#pragma unroll
    for (int q = 0; q < QT; ++q) sum[q] = Shape::add(sum[q]);

    // Columns with a sum near the end of F32 or past it, a bit each (a row whose probabilities' sum is a NaN is one in
    // any case).
    auto near_end = [&](int q) __attribute__((always_inline)) -> uint32_t {
        uint32_t most = 0;               // magnitudes in the order of their bits, a NaN above all
#pragma unroll
        for (int d = 0; d < Shape::kAccs; ++d)
#pragma unroll
            for (int j = 0; j < 4 * Shape::kAccQuads; ++j) {
                const uint32_t size = as_u32(acc[d][q][j]) & 0x7FFFFFFFu;
                most = most > size ? most : size;
            }
        const uint64_t lanes = __ballot(most >= kNearEnd && sum[q] == sum[q]);
        const uint32_t columns = (uint32_t)lanes | (uint32_t)(lanes >> 32);
        return W == 32 ? columns : (columns | columns >> 16) & 0xFFFFu;
    };

    // A row's place: its parts, or its first feature tile in the output (features of a head are whole
    // tiles).
    const uint64_t part = (uint64_t)blockIdx.x * BM;
    auto result_of = [&](uint32_t m) __attribute__((always_inline)) -> uint8_t* {
        const uint32_t i = divided(m, a.group, a.div_group), t = seq.start + i;
        const uint32_t head = hkv * a.group + (m - i * a.group);
        return a.out + ((uint64_t)(t >> 4) * a.out_tile_cols + head * a.d_tiles) * kTile16 + (t & 15u) * 32;
    };
    auto finished = [&](f32x4_t o, float l) __attribute__((always_inline)) -> u32x2 {
        const float inverse = 1.0f / l;
        if (l == 0.0f) return u32x2{0, 0};
        return u32x2{narrow2<DT>(o[0] * inverse, o[1] * inverse), narrow2<DT>(o[2] * inverse, o[3] * inverse)};
    };
    auto quad_of = [&](const Acc& o, int u) __attribute__((always_inline)) { return f32x4_t{o[4 * u], o[4 * u + 1], o[4 * u + 2], o[4 * u + 3]}; };
    if constexpr (WK == 1) {
        if (idle) return;
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const uint32_t m = m_wave + W * q + column;
            if (m < m_end) {
                float* parts = pieces > 1 ? a.parts + (part + m - m_block) * a.D : nullptr;
                uint8_t* to = result_of(m);
#pragma unroll
                for (int d = 0; d < Shape::kAccs; ++d)
#pragma unroll
                    for (int u = 0; u < Shape::kAccQuads; ++u) {
                        const uint32_t feature = Shape::feature(d, u, lane);
                        if (feature >= a.D) continue;
                        const f32x4_t o = quad_of(acc[d][q], u);
                        if (parts) *reinterpret_cast<f32x4_t*>(parts + feature) = o;
                        else *reinterpret_cast<u32x2*>(to + (feature >> 4) * kTile16 + (feature & 15u) * 2) = finished(o, sum[q]);
                    }
                if (parts && lane < W) {
                    a.part_stats[(part + m - m_block) * 2] = ref[q];
                    a.part_stats[(part + m - m_block) * 2 + 1] = sum[q];
                }
            }
            // (over what was stored)
            const uint32_t near = near_end(q);
            if (near) __builtin_amdgcn_s_waitcnt(0);
            for (uint32_t rest = near; rest; rest &= rest - 1)
                packed_again<DT, BM, NT>(args_at, q_again[wave], member * W * QT + W * q + __ffs(rest) - 1);
        }
    } else {
        // The teams meet in LDS, a wave's columns at a time: a wave leaves its sums scaled to the
        // largest reference of all teams.
        constexpr uint32_t kFeatures = 32 * KS, kRows = 16;
        __shared__ float meet_ref[WK][BM], meet_sum[WK][BM];
        __shared__ uint32_t meet_near[WK][BM / W];
        static_assert(WK * kRows * kFeatures * 4 <= WK * kStage, "the teams' sums fit a stage of K");
        float* meet = reinterpret_cast<float*>(&k_even[0][0]);     // [team][row][feature]
#pragma unroll
        for (int q = 0; q < QT; ++q) {
            const uint32_t near = near_end(q);
            if (lane == 0) meet_near[team][member * QT + q] = near;
        }
        // (after the first barrier) a column tile's rows that are taken again
        auto near_of = [&](uint32_t column_tile) __attribute__((always_inline)) -> uint32_t {
            uint32_t near = 0;
#pragma unroll
            for (int w = 0; w < WK; ++w) near |= meet_near[w][column_tile];
            return near;
        };
        if (lane < W) {
#pragma unroll
            for (int q = 0; q < QT; ++q) {
                meet_ref[team][member * W * QT + W * q + column] = ref[q];
                meet_sum[team][member * W * QT + W * q + column] = sum[q];
            }
        }
#pragma unroll
        for (int turn = 0; turn < (int)(BM / kRows); ++turn) {
            __syncthreads();       // the stages, or the rows before, have been read
            // rows turn * 16 .. of the block: sixteen columns of one column tile of one member
            constexpr int kPerWave = W * QT / kRows;
            if ((int)member == turn / kPerWave) {
                const int q = (turn % kPerWave) * (int)kRows / W;
                if (W == 16 || (int)(column >> 4) == (turn & 1)) {
                    float r = kLowest;
#pragma unroll
                    for (int w = 0; w < WK; ++w) r = fmaxf(r, meet_ref[w][turn * kRows + (column & 15u)]);
                    const float factor = __builtin_amdgcn_exp2f(ref[q] - r);
#pragma unroll
                    for (int d = 0; d < Shape::kAccs; ++d)
#pragma unroll
                        for (int u = 0; u < Shape::kAccQuads; ++u)
                            *reinterpret_cast<f32x4_t*>(meet + (team * kRows + (column & 15u)) * kFeatures + Shape::feature(d, u, lane)) =
                                    quad_of(acc[d][q], u) * factor;
                }
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < kRows * kFeatures / 4; i += 256) {
                const uint32_t row = i / (kFeatures / 4), feature = i % (kFeatures / 4) * 4, m = turn * kRows + row;
                if (m_block + m >= m_end || feature >= a.D || ((near_of(m / W) >> (m % W)) & 1u)) continue;
                float top = kLowest, l = 0.0f;
#pragma unroll
                for (int w = 0; w < WK; ++w) top = fmaxf(top, meet_ref[w][m]);
                f32x4_t o = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < WK; ++w) {
                    l += meet_sum[w][m] * __builtin_amdgcn_exp2f(meet_ref[w][m] - top);
                    o += *reinterpret_cast<const f32x4_t*>(meet + (w * kRows + row) * kFeatures + feature);
                }
                if (pieces > 1) {
                    *reinterpret_cast<f32x4_t*>(a.parts + (part + m) * a.D + feature) = o;
                    if (feature == 0) {
                        a.part_stats[(part + m) * 2] = top;
                        a.part_stats[(part + m) * 2 + 1] = l;
                    }
                } else
                    *reinterpret_cast<u32x2*>(result_of(m_block + m) + (feature >> 4) * kTile16 + (feature & 15u) * 2) = finished(o, l);
            }
        }
        // the waves take these rows in turn
        uint32_t turn = 0;
        for (uint32_t n = 0; n < BM / W; ++n)
            for (uint32_t rest = near_of(n); rest; rest &= rest - 1)
                if (turn++ % 4 == wave) packed_again<DT, BM, NT>(args_at, q_again[wave], n * W + __ffs(rest) - 1);
    }
}

// Joins the rows of a sequence and KV head whose tokens were shared out: a lane takes four features of
// a row, and scales each part from its own reference.  Bound by the chain of reads that finds the
// shares and then the parts: 7.3 us for 32 tokens, 9.8 us for eight trees of up to 61 rows (32 / 8 heads of 128).
template <int DT, uint32_t BM, uint32_t NT>
__global__ __launch_bounds__(256) void sdpa_packed_join_kernel(const SdpaPackedArgs a) {
    const uint32_t chunks = a.D / 4;
    const uint32_t s = divided(blockIdx.y, a.Hkv, a.div_hkv), hkv = blockIdx.y - s * a.Hkv;
    const PackedShare share = packed_share<BM, NT>(a, s, true);
    if (share.pieces <= 1) return;
    const PackedSequence seq = share.seq;
    const uint32_t rows = seq.rows < a.max_rows ? seq.rows : a.max_rows;
    const uint32_t at = blockIdx.x * 256 + threadIdx.x, m = at / chunks, feature = at % chunks * 4;
    if (m >= rows * a.group) return;
    // the parts are Hkv workgroups apart; eight of them are on their way together (the last one again
    // in the place of those past it, with no weight)
    const uint64_t first = ((uint64_t)(share.first + m / BM * share.pieces) * a.Hkv + hkv) * BM + m % BM;
    const uint64_t step = (uint64_t)a.Hkv * BM;
    constexpr uint32_t kAhead = 8;
    auto row_of = [&](uint32_t p) { return first + (p < share.pieces ? p : share.pieces - 1) * step; };
    float r = kLowest;
    for (uint32_t p0 = 0; p0 < share.pieces; p0 += kAhead) {
        float part[kAhead];
#pragma unroll
        for (uint32_t n = 0; n < kAhead; ++n) part[n] = a.part_stats[row_of(p0 + n) * 2];
#pragma unroll
        for (uint32_t n = 0; n < kAhead; ++n) r = fmaxf(r, part[n]);
    }
    float l = 0.0f;
    f32x4_t o = {0, 0, 0, 0};
    for (uint32_t p0 = 0; p0 < share.pieces; p0 += kAhead) {
        float ref[kAhead], sum[kAhead];
        f32x4_t part[kAhead];
#pragma unroll
        for (uint32_t n = 0; n < kAhead; ++n) {
            const uint64_t row = row_of(p0 + n);
            ref[n] = a.part_stats[row * 2];
            sum[n] = a.part_stats[row * 2 + 1];
            part[n] = *reinterpret_cast<const f32x4_t*>(a.parts + row * a.D + feature);
        }
#pragma unroll
        for (uint32_t n = 0; n < kAhead; ++n) {
            if (p0 + n >= share.pieces) break;
            const float factor = __builtin_amdgcn_exp2f(ref[n] - r);
            l += sum[n] * factor;
            // (an infinite value shows whatever its part's weight)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[j] += fabsf(part[n][j]) < __builtin_inff() ? part[n][j] * factor : part[n][j];
        }
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
    // and the tokens of a sequence, 64 at a time
    if ((cached ? (uint64_t)a->table.cols * k_pages->dims[2] : 0) + qm.rows > 0xFFFFFF00ull) return IOMX_ERR_OVERFLOW;
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

// How a request runs on the matrix cores: the rows of a block, whether its tokens are shared out,
// and the workspace the parts need.
struct PackedPlan {
    bool mfma;
    uint32_t places;         // see SdpaPackedArgs
    int columns;             // W
    int row_waves;           // WQ
    uint32_t block_rows, row_blocks;
    uint64_t groups;         // workgroups
    uint64_t parts_floats, stats_floats;
};

int packed_plan(const SdpaPackedArgs& a, int path, PackedPlan* p) {
    *p = {};
    p->mfma = path != 1 && a.D % kTile == 0 && (!a.table.base || a.page_rows % kTile == 0);
    if (!p->mfma) return IOMX_OK;
    const uint64_t m = (uint64_t)a.max_rows * a.group;       // rows of the longest sequence, per KV head
    // (four teams' stages of heads above 128 do not fit the LDS of a CU)
    const bool wide = a.D > 128;
    p->columns = m <= (wide ? 32 : 16) ? 16 : 32;
    p->row_waves = m <= 32 ? wide ? 2 : 1 : m <= 64 ? 2 : 4;
    p->block_rows = (uint32_t)(p->columns * p->row_waves);
    p->row_blocks = (uint32_t)((m + p->block_rows - 1) / p->block_rows);
    p->groups = (uint64_t)a.sequences * a.Hkv * p->row_blocks;
    // Shared out where there are few row blocks and a sequence may have tokens for more than one piece:
    // fewer than two per CU, or than one where a block has many rows and leaves large parts behind (128
    // blocks of four trees of 128 rows: 58 us shared out, 119 us not; 376 blocks of a prompt of 1500 rows,
    // 4 KV heads of 64: 50 us shared out, 33 us not).
    const uint64_t capacity = (uint64_t)a.table.cols * a.page_rows + a.max_rows;
    if (p->groups < (p->block_rows <= 32 ? kPackedGroups : kPackedGroups / 2) && capacity > 2 * kPackedLeastTokens) {
        // (few rows of wide heads: a workgroup's stages fill the LDS of a CU)
        const uint32_t groups = wide || (p->row_waves == 1 && a.D > 64) ? kPackedGroups / 2 : kPackedGroups;
        p->places = (groups + (uint32_t)a.Hkv - 1) / (uint32_t)a.Hkv;
        // (the row blocks there may be and one more piece for each of packed_room's at the most)
        const uint64_t most = p->block_rows <= 32 ? 2 * p->groups / a.Hkv : 0;
        p->groups += (most > p->places ? most : p->places) * a.Hkv;
        p->stats_floats = (p->groups * p->block_rows * 2 + 63) / 64 * 64;
        p->parts_floats = p->groups * p->block_rows * a.D;
    }
    if (p->groups > 0xFFFFFFull) return IOMX_ERR_OVERFLOW;     // a grid has fewer than 2^32 lanes
    return IOMX_OK;
}

template <int DT, int KS, int W, int WQ, int NT>
void launch_packed(const SdpaPackedArgs& a, const PackedPlan& p, hipStream_t st) {
    hipLaunchKernelGGL((sdpa_packed_mfma_kernel<DT, KS, W, 1, WQ, NT>), dim3((uint32_t)p.groups), dim3(256), 0, st, a);
    if (!p.places) return;
    const uint64_t lanes = (uint64_t)a.max_rows * a.group * (a.D / 4);
    const dim3 joins((uint32_t)((lanes + 255) / 256), a.sequences * a.Hkv);     // fewer than kPackedGroups of them
    hipLaunchKernelGGL((sdpa_packed_join_kernel<DT, W * WQ, NT>), joins, dim3(256), 0, st, a);
}

template <int DT, int KS>
void launch_packed(const SdpaPackedArgs& a, const PackedPlan& p, hipStream_t st) {
    if constexpr (KS > 4) {
        if (p.columns == 16) launch_packed<DT, KS, 16, 2, 2>(a, p, st);
        else if (p.row_waves == 2) launch_packed<DT, KS, 32, 2, 2>(a, p, st);
        else launch_packed<DT, KS, 32, 4, 4>(a, p, st);
    } else if (p.columns == 16) launch_packed<DT, KS, 16, 1, 2>(a, p, st);
    else if (p.row_waves == 1) launch_packed<DT, KS, 32, 1, 2>(a, p, st);
    else if (p.row_waves == 2) launch_packed<DT, KS, 32, 2, 2>(a, p, st);
    else launch_packed<DT, KS, 32, 4, 4>(a, p, st);
}

template <int DT>
void launch_packed(const SdpaPackedArgs& a, const PackedPlan& p, hipStream_t st) {
    switch ((a.D + 31) / 32) {
        case 1: launch_packed<DT, 1>(a, p, st); break;
        case 2: launch_packed<DT, 2>(a, p, st); break;
        case 3: launch_packed<DT, 3>(a, p, st); break;
        case 4: launch_packed<DT, 4>(a, p, st); break;
        case 5: case 6: launch_packed<DT, 6>(a, p, st); break;
        default: launch_packed<DT, 8>(a, p, st); break;
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
        a.places = p.places;
        a.page_tiles = a.page_rows / kTile;
        a.div_page_tiles = make_fast_div(a.page_tiles);
        a.div_units = make_fast_div(a.sequences * a.Hkv);
        a.div_hkv = make_fast_div(a.Hkv);
        a.scale_log2 = 1.44269504088896340736f * a.scale;
        a.part_stats = static_cast<float*>(workspace);
        a.parts = a.part_stats + p.stats_floats;
        if (dtype == IOMX_DT_BF16) launch_packed<IOMX_DT_BF16>(a, p, st);
        else launch_packed<IOMX_DT_F16>(a, p, st);
        record_launch(p.columns == 16 ? "sdpa_packed_few" : "sdpa_packed_mfma", (uint32_t)p.groups, 256, (uint64_t)a.T * a.Hq);
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
