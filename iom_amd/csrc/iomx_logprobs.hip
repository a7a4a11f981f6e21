// Log probabilities of given tokens, entropy and the most likely tokens of vocabulary rows.
#include <type_traits>

#include "iomx_packed.hpp"

namespace iomx {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kMaxTop = 32;

struct LogprobsArgs {
    const uint8_t* logits;
    const int32_t* tokens;
    float* logprobs;
    float* entropy;
    int32_t* top_ids;
    float* top_logprobs;
    PlaneWalk<6> walk;              // the operands above, in their order
    uint64_t logits_plane, given_plane, entropy_plane, top_plane;   // elements
    uint32_t R, V, G, K;
    uint32_t tile_cols, given_tile_cols, top_tile_cols;
    FastDiv div_rows;
    FastDiv div_parts;               // pieces of sixteen tiles of a cell
    // how the scan is laid out
    uint32_t rows, bands;            // rows of all planes; tile rows of a plane
    uint32_t splits, cells_per_split, cells, cell_groups, group_tiles;
    FastDiv div_splits, div_bands;
    float* stats;                    // [plane][tile row][split][16 rows][4]: M, sum e^d, sum d e^d
    float* cell_max;                 // [plane][tile row][cell][16 rows], null where no top is asked for
};

// ---------------------------------------------------------------------------
// token_logprobs_scan reads the logits once.  A band (16 rows of a plane) lies in memory as one run
// of tiles, so a wave's loads are whole kilobytes and a lane meets one row only: lane (row, part of a
// tile row).  It keeps the row's maximum M, sum e^d and sum d e^d with d = x - M (a difference, not a
// product with log2 e taken from another: logits near the ends of the range stay finite), 64,
// 32 or 16 logits at a time with the maximum moved before each, and the maximum of every cell (a group
// of 64 to 256 columns, or a few groups) goes to the workspace.  2047 rows of 128256 BF16: 102 us, 5.1
// TB/s, where a bare read reaches 6.6; the vector units are busy for two thirds of it.
//
// token_logprobs_finish, one wave per row (or four), joins the sums and picks the most likely tokens without
// another pass: a value that K cells' maxima reach is reached by K logits, so only the cells that
// reach it are read again, and in them the logits that reach it are few; each counts those before it
// (larger, or equal with a lower id), which is its place.  Bound by that gather: 28 us for 2047 rows and
// their 20 most likely (112 MB in lines of 128 bytes, of which a row has a quarter), of which 2 us look
// for the bound; twice as many cells of half the size save 4 us here and cost the scan 10 us.  Few rows wait
// for three reads one after the other: 8.5 us for 16.
// ---------------------------------------------------------------------------

constexpr uint32_t kMostCells = 512;          // of a row: eight per lane
constexpr uint32_t kMostChosen = 256;         // cells that are read again
// Where a row has hardly more cells than places, nearly every logit is above the bound; its logits are then
// their own cells, and a wave holds them all, sixteen or 38 per lane (5 rows of 686 logits, their 20 most
// likely: 55 us by cells of 64, 14 us by logits; 2000 logits: 13 us by cells, 24 us by logits).
constexpr uint32_t kFewSlots = 16, kMoreSlots = 38;
constexpr uint32_t kTeamRows = 512;           // up to here four waves may pick from a row
constexpr uint32_t kMostCandidates = 128;     // of a row: two per lane

// d as a factor of e^d: from -200 on down e^d is 0 in F32, and its product with d is, too
__device__ __forceinline__ float at_least(float d) { return fmaxf(d, -200.0f); }
// e^d for d <= 0, to a few units in the last place for the d whose exponential is not tiny
__device__ __forceinline__ float exponential(float d) { return __builtin_amdgcn_exp2f(d * 1.44269504088896340736f); }

template <int DT>
__device__ __forceinline__ float logit_at(const uint8_t* row, uint32_t c) {
    const uint64_t slot = (uint64_t)(c >> 4) * kTileSlots + (c & 15u);
    if constexpr (DT == IOMX_DT_F32) return reinterpret_cast<const float*>(row)[slot];
    else if constexpr (DT == IOMX_DT_BF16) return as_f32((uint32_t)reinterpret_cast<const uint16_t*>(row)[slot] << 16);
    else return (float)reinterpret_cast<const _Float16*>(row)[slot];
}

// element i of a lane's 16 bytes
template <int DT>
__device__ __forceinline__ float logit_of(u32x4 w, int i) {
    if constexpr (DT == IOMX_DT_F32) return as_f32(w[i]);
    else if constexpr (DT == IOMX_DT_BF16) return (i & 1) ? bf16_hi(w[i >> 1]) : bf16_lo(w[i >> 1]);
    else { const f32x2 p = f16_pair(w[i >> 1]); return (i & 1) ? p.y : p.x; }
}

// A lane's value from another lane of its row of sixteen, by a move within the register file (a shuffle goes
// through LDS); and the other half of the wave's.
template <int CONTROL>
__device__ __forceinline__ float lane_moved(float v) {
    return as_f32(__builtin_amdgcn_update_dpp(as_u32(v), as_u32(v), CONTROL, 0xF, 0xF, false));
}
__device__ __forceinline__ float other_half(float v) {
    const auto both = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
    return as_f32((threadIdx.x & 32u) ? both[0] : both[1]);
}

// GT: tiles of a group, which a wave loads at once
template <int DT, int GT, bool ENTROPY>
__global__ __launch_bounds__(256) void token_logprobs_scan_kernel(const LogprobsArgs a) {
    constexpr int kSize = DT == IOMX_DT_F32 ? 4 : 2, kElems = 16 / kSize, kPerRow = kTile / kElems;
    constexpr int kLoads = GT * 256 * kSize / 1024;
    constexpr float inf = __builtin_inff();
    __shared__ float joined[3][4][kTile];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t band = divided(blockIdx.x, a.splits, a.div_splits), split = blockIdx.x - band * a.splits;
    const uint32_t plane_index = divided(band, a.bands, a.div_bands), tile_row = band - plane_index * a.bands;
    uint64_t plane[6];
    walk_planes(a.walk, plane_index, plane);
    const uint8_t* base = a.logits + (plane[0] * a.logits_plane + (uint64_t)tile_row * a.tile_cols * kTileSlots) * kSize;
    const uint32_t row = lane / kPerRow % kTile, part = lane % kPerRow;
    const bool there = tile_row * kTile + row < a.R;
    const uint32_t lane_tile = lane / (kPerRow * kTile);      // of a load: 1 in the upper half of a wave, 16-bit leaves

    float most = -inf, sum = 0.0f, weighted = 0.0f;           // M (-inf before the first finite logit)
    const uint32_t c_end = (split + 1) * a.cells_per_split < a.cells ? (split + 1) * a.cells_per_split : a.cells;
    auto load = [&](uint32_t g, u32x4 (&w)[kLoads]) {
        const uint8_t* at = base + (uint64_t)g * (GT * kTileSlots * kSize) + lane * 16;
        if ((g + 1) * GT <= a.tile_cols && there) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) w[i] = *reinterpret_cast<const u32x4*>(at + i * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                w[i] = u32x4{0, 0, 0, 0};
                if (there && g * GT + i * (GT / kLoads ? GT / kLoads : 1) + lane_tile < a.tile_cols)
                    w[i] = *reinterpret_cast<const u32x4*>(at + i * 1024);
            }
        }
    };
    u32x4 next[kLoads];
    const uint32_t c_begin = split * a.cells_per_split + wave;
    if (c_begin < c_end) load(c_begin * a.cell_groups, next);
    for (uint32_t c = c_begin; c < c_end; c += 4) {
        float cell = -inf;
        for (uint32_t k = 0; k < a.cell_groups; ++k) {
            const uint32_t g = c * a.cell_groups + k;
            if (g * GT >= a.tile_cols) break;
            u32x4 w[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) w[i] = next[i];
            const bool more = k + 1 < a.cell_groups && (g + 1) * GT < a.tile_cols;
            const uint32_t g_next = more ? g + 1 : (c + 4) * a.cell_groups;
            if (more || c + 4 < c_end) load(g_next, next);
            // columns from here on are none of the row's
            const uint32_t columns = a.V - g * (GT * kTile);
            const bool whole = columns >= (uint32_t)GT * kTile && there;
            auto logit = [&](int i, int j) {
                const float x = logit_of<DT>(w[i], j);
                if (whole) return x;
                const uint32_t column = (i * (GT / kLoads ? GT / kLoads : 1) + lane_tile) * kTile + part * kElems + j;
                return there && column < columns ? x : -inf;
            };
            auto group = [&](auto x_of) {
                float top = -inf;
#pragma unroll
                for (int i = 0; i < kLoads; ++i)
#pragma unroll
                    for (int j = 0; j < kElems; j += 2) top = fmaxf(fmaxf(top, x_of(i, j)), x_of(i, j + 1));
                cell = fmaxf(cell, top);
                const float m2 = fmaxf(most, top);
                const float now = m2 == -inf ? 0.0f : m2;
                // the sums move from the old maximum to the new one: sum d e^d over d + (old - new)
                const float by = most == -inf ? 0.0f : most - now, factor = exponential(by);
                if (ENTROPY) weighted = (weighted + at_least(by) * sum) * factor;
                sum *= factor;
                most = m2;
#pragma unroll
                for (int i = 0; i < kLoads; ++i)
#pragma unroll
                    for (int j = 0; j < kElems; ++j) {
                        const float d = x_of(i, j) - now;
                        const float e = exponential(d);
                        sum += e;
                        if (ENTROPY) weighted = __builtin_fmaf(at_least(d), e, weighted);
                    }
            };
            if (columns >= (uint32_t)GT * kTile) group([&](int i, int j) { return logit_of<DT>(w[i], j); });
            else group(logit);
        }
        if (a.cell_max) {
            // the lanes of a row: neighbours, and the other half of the wave where a load has two tiles
            cell = fmaxf(cell, lane_moved<0xB1>(cell));              // quad_perm 1, 0, 3, 2
            if constexpr (kPerRow == 4) cell = fmaxf(cell, lane_moved<0x4E>(cell));      // 2, 3, 0, 1
            else cell = fmaxf(cell, other_half(cell));
            if (there && part == 0 && lane_tile == 0) a.cell_max[((uint64_t)band * a.cells + c) * kTile + row] = cell;
        }
    }
    auto join = [&](float m2, float s2, float w2) {
        const float m3 = fmaxf(most, m2), now = m3 == -inf ? 0.0f : m3;
        const float by1 = most == -inf ? 0.0f : most - now, by2 = m2 == -inf ? 0.0f : m2 - now;
        const float f1 = exponential(by1), f2 = exponential(by2);
        if (ENTROPY) weighted = (weighted + at_least(by1) * sum) * f1 + (w2 + at_least(by2) * s2) * f2;
        sum = sum * f1 + s2 * f2;
        most = m3;
    };
    auto join_lanes = [&](int off) {
        const float m2 = __shfl_xor(most, off), s2 = __shfl_xor(sum, off), w2 = __shfl_xor(weighted, off);
        join(m2, s2, w2);
    };
    join_lanes(1);
    join_lanes(kPerRow == 4 ? 2 : 32);
    if (part == 0 && lane_tile == 0) {
        joined[0][wave][row] = most;
        joined[1][wave][row] = sum;
        joined[2][wave][row] = weighted;
    }
    __syncthreads();
    if (threadIdx.x >= kTile) return;
    most = -inf; sum = 0.0f; weighted = 0.0f;
    for (int w = 0; w < 4; ++w) join(joined[0][w][lane], joined[1][w][lane], joined[2][w][lane]);
    float* to = a.stats + (((uint64_t)band * a.splits + split) * kTile + lane) * 4;
    to[0] = most;
    to[1] = sum;
    to[2] = weighted;
}

// Order of the top: the larger value, of equal ones the lower id, as one number (+0 and -0 are equal).
__device__ __forceinline__ uint64_t top_key(float x, uint32_t id) {
    const uint32_t b = as_u32(x == 0.0f ? 0.0f : x);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - id);
}
__device__ __forceinline__ uint32_t key_id(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }
__device__ __forceinline__ float key_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return as_f32(b & 0x80000000u ? b & 0x7FFFFFFFu : ~b);
}

// Reductions over a wave by moves within the register file (a shuffle goes through LDS): rows of 16
// lanes by four rotations, then the rows' results out of scalar registers.
template <class Op>
__device__ __forceinline__ float wave_reduce(float x, Op op) {
    x = op(x, lane_moved<0x121>(x));   // row_ror:1, 2, 4, 8
    x = op(x, lane_moved<0x122>(x));
    x = op(x, lane_moved<0x124>(x));
    x = op(x, lane_moved<0x128>(x));
    const float a = as_f32(__builtin_amdgcn_readlane(as_u32(x), 0)), b = as_f32(__builtin_amdgcn_readlane(as_u32(x), 16));
    const float c = as_f32(__builtin_amdgcn_readlane(as_u32(x), 32)), d = as_f32(__builtin_amdgcn_readlane(as_u32(x), 48));
    return op(op(a, b), op(c, d));
}
__device__ __forceinline__ float wave_max(float x) {
    return wave_reduce(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
    return wave_reduce(x, [](float a, float b) { return a + b; });
}

// OWN: slots of a lane for logits that are their own cells; 0: cells of the scan.  TEAM: waves of a row (1 or
// 4), which all look for the bound and share out the cells that are read again.
template <int DT, uint32_t OWN, uint32_t TEAM>
__global__ __launch_bounds__(256) void token_logprobs_finish_kernel(const LogprobsArgs a) {
    constexpr int kSize = DT == IOMX_DT_F32 ? 4 : 2;
    constexpr float inf = __builtin_inff();
    constexpr uint32_t kSlots = OWN ? OWN : kMostCells / 64, kMostListed = OWN ? kMostCandidates : kMostChosen;
    const uint32_t all_cells = OWN ? a.V : a.cells;
    __shared__ uint32_t found[4][kMostCandidates];       // columns
    __shared__ uint16_t chosen[4][kMostChosen];
    __shared__ uint32_t counts[4];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t index = __builtin_amdgcn_readfirstlane(TEAM > 1 ? blockIdx.x : blockIdx.x * 4 + wave);   // of the row
    if (index >= a.rows) return;
    const uint32_t plane_index = divided(index, a.R, a.div_rows), r = index - plane_index * a.R;
    const uint32_t band = plane_index * a.bands + (r >> 4);
    uint64_t plane[6];
    walk_planes(a.walk, plane_index, plane);
    const uint8_t* row = a.logits + (plane[0] * a.logits_plane + (uint64_t)(r >> 4) * a.tile_cols * kTileSlots
                                     + (r & 15u) * kTile) * kSize;
    // everything that the workspace holds of the row, in one go: the cells' maxima ...
    float cells[kSlots];
    if (a.top_ids) {
        const float* maxima = a.cell_max + (uint64_t)band * a.cells * kTile + (r & 15u);
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i) {
            const uint32_t c = i * 64 + lane;
            if constexpr (OWN != 0) cells[i] = c < a.V ? logit_at<DT>(row, c) : -inf;
            else cells[i] = c < a.cells ? maxima[(uint64_t)c * kTile] : -inf;
        }
    }
    // ... and the splits' sums, one per lane (there are 64 at the most)
    float most = -inf, sum = 0.0f, weighted = 0.0f;
    if (lane < a.splits) {
        const f32x4_t from = *reinterpret_cast<const f32x4_t*>(a.stats + (((uint64_t)band * a.splits + lane) * kTile + (r & 15u)) * 4);
        most = from[0]; sum = from[1]; weighted = from[2];
    }
    // ... and the first 64 given tokens
    const uint64_t row_at = (uint64_t)(r >> 4), in_row = (r & 15u) * kTile;
    auto given_at = [&](uint32_t g) { return (row_at * a.given_tile_cols + (g >> 4)) * kTileSlots + in_row + (g & 15u); };
    uint32_t given = a.V;
    float given_logit = 0.0f;
    if (lane < a.G) {
        given = (uint32_t)a.tokens[plane[1] * a.given_plane + given_at(lane)];
        if (given < a.V) given_logit = logit_at<DT>(row, given);
    }
    const float m = wave_max(most);
    const float now = m == -inf ? 0.0f : m, by = most == -inf ? 0.0f : most - now, factor = exponential(by);
    weighted = (weighted + at_least(by) * sum) * factor;
    sum = wave_sum(sum * factor);
    weighted = wave_sum(weighted);
    // a NaN or +inf left the sum a NaN
    const bool bad = !(sum > 0.0f);
    const float nan = as_f32(kQuietNanF32);
    double log_sum;
    // (a hundred and more 64-bit instructions: where the loads of candidates are on their way)
    auto form_log = [&]() __attribute__((always_inline)) { log_sum = log((double)sum); };
    // Of two logits of 1e38 the difference comes first: next to either of them the logarithm is lost in 64 bits too.
    auto log_probability = [&](float logit) __attribute__((always_inline)) -> float {
        return (float)((double)logit - (double)now - log_sum);
    };
    auto put = [&](uint32_t place, uint32_t id, float logit) __attribute__((always_inline)) {
        const uint64_t at = (row_at * a.top_tile_cols + (place >> 4)) * kTileSlots + in_row + (place & 15u);
        a.top_ids[plane[4] * a.top_plane + at] = bad ? -1 : (int32_t)id;
        a.top_logprobs[plane[5] * a.top_plane + at] = bad ? nan : log_probability(logit);
    };
    // the K most likely tokens
    auto pick = [&]() __attribute__((always_inline)) {
        // A bound that at least K cells' maxima reach, so that at least K logits do, and not many more: from
        // the row's maximum downwards in steps that double, then halving the last step.
        auto reaching = [&](float bound) __attribute__((always_inline)) -> uint32_t {
            uint32_t n = 0;
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i)
                if (i * 64 < all_cells) n += __popcll(__ballot(cells[i] >= bound));
            return n;
        };
        auto largest_below = [&](float limit) __attribute__((always_inline)) -> float {
            float top = -inf;
#pragma unroll
            for (uint32_t i = 0; i < kSlots; ++i) top = fmaxf(top, cells[i] < limit ? cells[i] : -inf);
            return wave_max(top);
        };
        uint32_t ties = ~0u;                           // cells of exactly the bound that are looked at
        const float top = largest_below(inf);
        float over = top, step = fmaxf(1.0f, fabsf(top) * 0.0078125f);   // `over`: fewer than K reach it, or it is the top
        float bound;
        uint32_t reached;
        for (;;) {
            bound = fmaxf(top - step, -3.4028234663852886e38f);          // that one: every finite logit
            reached = reaching(bound);
            if (reached >= a.K || bound == -3.4028234663852886e38f) break;
            over = bound;
            step *= 2.0f;
        }
        // (of few cells nearly all would be taken, and far more logits with them)
        const uint32_t spare = (all_cells - a.K) / 4, enough = a.K + (spare < a.K / 2 ? spare : a.K / 2);
        for (int halvings = 0; halvings < 12 && reached > enough; ++halvings) {
            const float middle = bound * 0.5f + over * 0.5f;
            const uint32_t n = reaching(middle);
            if (n >= a.K) { bound = middle; reached = n; }
            else over = middle;
        }
        if (reached > kMostListed) {
            // (rows of equal logits) the K-th largest maximum itself: of the cells that have it, those
            // with the lowest columns make up the K cells that hold the K most likely tokens
            uint32_t larger = 0;
            bound = top;
            for (;;) {
                uint32_t equal = 0;
#pragma unroll
                for (uint32_t i = 0; i < kSlots; ++i) equal += __popcll(__ballot(cells[i] == bound));
                if (larger + equal >= a.K) break;
                larger += equal;
                bound = largest_below(bound);
            }
            ties = a.K - larger;
        }
        // the logits that reach it
        uint32_t count = 0, listed = 0;
#pragma unroll
        for (uint32_t i = 0; i < kSlots; ++i) {
            if (i * 64 >= all_cells) break;
            const uint64_t below = (1ull << lane) - 1, equal = __ballot(cells[i] == bound);
            const bool take = cells[i] > bound || (cells[i] == bound && (uint32_t)__popcll(equal & below) < ties);
            const uint64_t there = __ballot(take);
            const uint32_t place = listed + __popcll(there & below);
            if constexpr (OWN != 0) { if (take) found[wave][place] = i * 64 + lane; }
            else if (take) chosen[wave][place] = (uint16_t)(i * 64 + lane);
            listed += __popcll(there);
            if (ties != ~0u) ties -= __popcll(equal) < ties ? __popcll(equal) : ties;
        }
        const uint32_t per_cell = a.cell_groups * a.group_tiles;                 // tiles: 4, or a multiple of 8 or 16
        if constexpr (OWN != 0) {
            count = listed;
            form_log();
        } else {
            __builtin_amdgcn_wave_barrier();       // a wave's LDS operations are in order
            // A lane takes four columns of a tile; a wave, sixteen tiles: a part of one cell, or two or four
            // cells.  The loads of four such pieces are on their way together (with eight a step of 16 rows takes
            // 0.7 us longer, 2047 rows 0.7 us less).  Few logits reach the bound,
            // so a lane only notes which of its own do, a bit each, and the columns are listed from the bits.
            constexpr uint32_t kAhead = 4;
            const uint32_t parts = (per_cell + 15) / 16, shift = per_cell < 16 ? per_cell == 4 ? 2 : 1 : 0;   // 2^shift cells
            const uint32_t pieces = ((listed + (1u << shift) - 1) >> shift) * parts;
            const uint32_t lane_cell = (lane >> 2) >> (4 - shift), lane_tile = (lane >> 2) - (lane_cell << (4 - shift));
            // first of a lane's four columns of piece p, from a.V on if it has none
            auto columns_of = [&](uint32_t p) __attribute__((always_inline)) -> uint32_t {
                const uint32_t q = divided(p, parts, a.div_parts), entry = (q << shift) + lane_cell;
                const uint32_t tile_in_cell = (p - q * parts) * 16 + lane_tile;
                const uint32_t tile = (entry < listed ? chosen[wave][entry] : 0u) * per_cell + tile_in_cell;
                return p < pieces && entry < listed && tile_in_cell < per_cell ? tile * kTile + (lane & 3u) * 4 : ~0u;
            };
            const uint32_t p_first = TEAM > 1 ? wave * kAhead : 0;
            uint32_t p0 = p_first;
            do {
                u32x4 x[kAhead];
                uint32_t first[kAhead];
#pragma unroll
                for (uint32_t n = 0; n < kAhead; ++n) {
                    first[n] = columns_of(p0 + n);
                    // a tile's padding columns are read with it, and not looked at
                    const uint8_t* at = row + ((uint64_t)(first[n] < a.V ? first[n] >> 4 : 0u) * kTileSlots + (lane & 3u) * 4) * kSize;
                    if constexpr (DT == IOMX_DT_F32) x[n] = *reinterpret_cast<const u32x4*>(at);
                    else {
                        const u32x2 w = *reinterpret_cast<const u32x2*>(at);
                        x[n] = u32x4{w.x, w.y, 0, 0};
                    }
                }
                if (p0 == p_first) form_log();
                uint32_t hits = 0;
#pragma unroll
                for (uint32_t n = 0; n < kAhead; ++n)
#pragma unroll
                    for (uint32_t j = 0; j < 4; ++j)
                        hits |= (logit_of<DT>(x[n], j) >= bound && first[n] < a.V && first[n] + j < a.V ? 1u : 0u) << (4 * n + j);
                for (uint64_t there; (there = __ballot(hits != 0)) != 0;) {
                    const uint32_t bit = (uint32_t)__ffs(hits) - 1u, place = count + __popcll(there & ((1ull << lane) - 1));
                    if (hits && place < kMostCandidates) found[wave][place] = columns_of(p0 + (bit >> 2)) + (bit & 3u);
                    hits &= hits - 1;
                    count += __popcll(there);
                }
                p0 += TEAM * kAhead;
            } while (p0 < pieces && count <= kMostCandidates);
            if constexpr (TEAM > 1) {
                if (lane == 0) counts[wave] = count;
                __syncthreads();
                if (wave) return;
                count = counts[0] + counts[1] + counts[2] + counts[3];
            }
        }
        if (OWN || count <= kMostCandidates) {
            __builtin_amdgcn_wave_barrier();
            auto key_of = [&](uint32_t i) __attribute__((always_inline)) -> uint64_t {
                if (i >= count) return 0;
                uint32_t from = wave;
                if constexpr (TEAM > 1)
                    for (from = 0; i >= counts[from]; ++from) i -= counts[from];
                const uint32_t id = found[from][i];
                return top_key(logit_at<DT>(row, id), id);
            };
            const uint64_t one = key_of(lane), two = key_of(lane + 64);
            uint32_t before_one = 0, before_two = 0;
            for (uint32_t i = 0; i < count; ++i) {
                const uint64_t from = i < 64 ? one : two;
                const uint64_t key = (uint64_t)__builtin_amdgcn_readlane((uint32_t)(from >> 32), i & 63u) << 32
                                   | (uint32_t)__builtin_amdgcn_readlane((uint32_t)from, i & 63u);
                before_one += key > one;
                before_two += key > two;
            }
            if (lane < count && before_one < a.K) put(before_one, key_id(one), key_value(one));
            if (lane + 64 < count && before_two < a.K) put(before_two, key_id(two), key_value(two));
            // too few finite logits: the first of the others follow
            uint32_t place = count;
            for (uint32_t c0 = 0; place < a.K && c0 < a.V; c0 += 64) {
                const bool masked = c0 + lane < a.V && logit_at<DT>(row, c0 + lane) == -inf;
                const uint64_t there = __ballot(masked);
                const uint32_t mine = place + __popcll(there & ((1ull << lane) - 1));
                if (masked && mine < a.K) put(mine, c0 + lane, -inf);
                place += __popcll(there);
            }
            return;
        }
        // many equal logits at the bound: a pass over the chosen cells for each place
        uint64_t last = ~0ull;
        for (uint32_t place = 0; place < a.K; ++place) {
            uint64_t best = 0;
            for (uint32_t n = 0; n < listed; ++n) {
                const uint32_t from = chosen[wave][n] * per_cell * kTile;
                const uint32_t to = from + per_cell * kTile < a.V ? from + per_cell * kTile : a.V;
                for (uint32_t c = from + lane; c < to; c += 64) {
                    const uint64_t key = top_key(logit_at<DT>(row, c), c);
                    best = key < last && key > best ? key : best;
                }
            }
#pragma unroll
            for (int off = 1; off < 64; off *= 2) {
                const uint64_t other = __shfl_xor((unsigned long long)best, off);
                best = other > best ? other : best;
            }
            last = best;
            if (lane == 0) put(place, key_id(best), key_value(best));
        }
    };
    if (a.top_ids && !bad) pick();
    else form_log();
    if (TEAM > 1 && wave) return;
    if (a.top_ids && bad && lane < a.K) put(lane, 0, 0.0f);
    for (uint32_t g = lane; g < a.G; g += 64) {
        if (g >= 64) {
            given = (uint32_t)a.tokens[plane[1] * a.given_plane + given_at(g)];
            if (given < a.V) given_logit = logit_at<DT>(row, given);
        }
        a.logprobs[plane[2] * a.given_plane + given_at(g)] =
                given >= a.V ? -inf : bad ? nan : log_probability(given_logit);
    }
    if (a.entropy && lane == 0)
        a.entropy[plane[3] * a.entropy_plane + row_at * kTileSlots + in_row] = bad ? nan : (float)(log_sum - (double)weighted / sum);
}

namespace {

// Checks the operands and fills in everything of the arguments but the workspace.
int logprobs_request(int dtype, const iomx_view* logits, const iomx_view* tokens, const iomx_view* logprobs,
                     const iomx_view* entropy, const iomx_view* top_ids, const iomx_view* top_logprobs,
                     LogprobsArgs* a) {
    if (!leaf_bits(dtype)) return IOMX_ERR_UNSUPPORTED;
    IOMX_TRY(check_view(logits, leaf_bits(dtype)));
    if (!tokens != !logprobs || !top_ids != !top_logprobs) return IOMX_ERR_INVALID;
    if (!tokens && !entropy && !top_ids) return IOMX_ERR_INVALID;
    const iomx_view* v[6] = {logits, tokens, logprobs, entropy, top_ids, top_logprobs};
    for (int i = 1; i < 6; ++i) {
        if (!v[i]) continue;
        IOMX_TRY(check_view(v[i], 32));
        if (v[i]->rank != logits->rank) return IOMX_ERR_INVALID;
        for (uint32_t d = 0; d + 1 < logits->rank; ++d)
            if (v[i]->dims[d] != logits->dims[d]) return IOMX_ERR_INVALID;
        // an output stands alone
        for (int j = 0; i > 1 && j < 6; ++j)
            if (j != i && v[j] && v[j]->base == v[i]->base) return IOMX_ERR_INVALID;
    }
    const Matrix m = matrix_of(*logits);
    if (tokens && !same_extents(*tokens, *logprobs)) return IOMX_ERR_INVALID;
    if (top_ids && !same_extents(*top_ids, *top_logprobs)) return IOMX_ERR_INVALID;
    if (entropy && matrix_of(*entropy).cols != 1) return IOMX_ERR_INVALID;
    if (top_ids && matrix_of(*top_ids).cols > m.cols) return IOMX_ERR_INVALID;
    if (dtype != IOMX_DT_BF16 && dtype != IOMX_DT_F16 && dtype != IOMX_DT_F32) return IOMX_ERR_UNSUPPORTED;
    if (m.cols >= (1ull << 24)) return IOMX_ERR_UNSUPPORTED;
    if (top_ids && matrix_of(*top_ids).cols > kMaxTop) return IOMX_ERR_UNSUPPORTED;
    if (tokens && matrix_of(*tokens).cols > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    const uint32_t nlead = logits->rank - 2;
    uint64_t strides[6][kMaxLead] = {}, offsets[6] = {};
    for (int i = 0; i < 6; ++i) {
        const iomx_view* s = v[i] ? v[i] : logits;      // a missing operand walks along and is not touched
        offsets[i] = s->plane_offset;
        for (uint32_t d = 0; d < nlead; ++d) strides[i][d] = s->plane_strides[d];
    }
    IOMX_TRY(build_walk<6>(nlead, logits->dims, strides, offsets, &a->walk));
    uint64_t rows;
    if (mul_overflows(a->walk.planes, m.rows, &rows) || rows > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    a->logits = static_cast<const uint8_t*>(logits->base);
    a->logits_plane = m.plane_elems;
    a->R = (uint32_t)m.rows;
    a->V = (uint32_t)m.cols;
    a->tile_cols = (uint32_t)m.tile_cols;
    a->div_rows = make_fast_div(a->R);
    a->rows = (uint32_t)rows;
    a->bands = (uint32_t)m.tile_rows;
    a->div_bands = make_fast_div(a->bands);
    if (tokens) {
        const Matrix g = matrix_of(*tokens);
        a->tokens = static_cast<const int32_t*>(tokens->base);
        a->logprobs = static_cast<float*>(logprobs->base);
        a->given_plane = g.plane_elems;
        a->G = (uint32_t)g.cols;
        a->given_tile_cols = (uint32_t)g.tile_cols;
    }
    if (entropy) {
        a->entropy = static_cast<float*>(entropy->base);
        a->entropy_plane = matrix_of(*entropy).plane_elems;
    }
    if (top_ids) {
        const Matrix t = matrix_of(*top_ids);
        a->top_ids = static_cast<int32_t*>(top_ids->base);
        a->top_logprobs = static_cast<float*>(top_logprobs->base);
        a->top_plane = t.plane_elems;
        a->K = (uint32_t)t.cols;
        a->top_tile_cols = (uint32_t)t.tile_cols;
    }
    return IOMX_OK;
}

template <int DT> constexpr int kWideGroup = DT == IOMX_DT_F32 ? 16 : 8;

// Fewer than a fifth more cells than places (the cells are of 64 columns then; with a tenth more, a row in
// forty of 2241 logits has more than kMostCandidates above the bound of its 32 most likely).
bool picks_from_logits(const LogprobsArgs& a) { return 5 * a.cells < 6 * a.K; }
static_assert((6 * kMaxTop - 1) / 5 <= kMoreSlots, "a lane holds a slot of every such cell");

// The scan's layout, and the floats of workspace it takes.
int logprobs_layout(int dtype, LogprobsArgs* a, uint64_t* stats_floats, uint64_t* cell_floats) {
    // Groups of 64 columns for small vocabularies, so that even a row of few thousand logits has a
    // cell for each of the K most likely and a few more; cells of several groups where there would be too many.
    // Larger groups are 4 KiB of the 16-bit leaves and 16 KiB of F32 for a wave: 2047 rows of 128256
    // BF16 scan in 103 us with 8 tiles and in 116 us with 16 (half the waves for the registers), 333
    // rows of 50257 F32 in 18.7 us with 8 and 16.2 us with 16 (a wave has one or two groups).
    a->group_tiles = a->V < 16384 ? 4 : dtype == IOMX_DT_F32 ? kWideGroup<IOMX_DT_F32> : kWideGroup<IOMX_DT_BF16>;
    const uint32_t groups = (a->tile_cols + a->group_tiles - 1) / a->group_tiles;
    a->cell_groups = (groups + kMostCells - 1) / kMostCells;
    a->cells = (groups + a->cell_groups - 1) / a->cell_groups;
    a->div_parts = make_fast_div((a->cell_groups * a->group_tiles + 15) / 16);
    // six workgroups for each CU in all, a cell for each wave at the least
    const uint64_t bands = a->walk.planes * a->bands;
    uint64_t splits = bands >= 1536 ? 1 : (1536 + bands - 1) / bands;
    if (splits > (a->cells + 3) / 4) splits = (a->cells + 3) / 4;
    if (splits > 64) splits = 64;
    a->cells_per_split = (uint32_t)((a->cells + splits - 1) / splits);
    a->splits = (a->cells + a->cells_per_split - 1) / a->cells_per_split;
    a->div_splits = make_fast_div(a->splits);
    if (bands * a->splits > 0x7FFFFFF0ull) return IOMX_ERR_OVERFLOW;
    *stats_floats = bands * a->splits * kTile * 4;
    *cell_floats = a->top_ids && !picks_from_logits(*a) ? bands * a->cells * kTile : 0;
    return IOMX_OK;
}

template <int DT>
void launch_logprobs(const LogprobsArgs& a, hipStream_t st) {
    const dim3 grid((uint32_t)(a.walk.planes * a.bands * a.splits));
    if (a.group_tiles == 4 && a.entropy) hipLaunchKernelGGL((token_logprobs_scan_kernel<DT, 4, true>), grid, dim3(256), 0, st, a);
    else if (a.group_tiles == 4) hipLaunchKernelGGL((token_logprobs_scan_kernel<DT, 4, false>), grid, dim3(256), 0, st, a);
    else if (a.entropy) hipLaunchKernelGGL((token_logprobs_scan_kernel<DT, kWideGroup<DT>, true>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((token_logprobs_scan_kernel<DT, kWideGroup<DT>, false>), grid, dim3(256), 0, st, a);
    // Four waves of a row where there are few rows, and more pieces of cells than a wave has on their way
    // together: 16 rows of 128256, 20 most likely, 17.5 us and 22.6 with one wave; 333 rows of 50257 F32, 8
    // most likely, 24.7 and 26.0; 1024 rows of 32000, 10 most likely, 28.0 and 26.1; 16 rows of 32000, 5 most
    // likely (three pieces), 12.5 and 12.2.
    const bool team = a.rows <= kTeamRows && a.K * a.cell_groups * a.group_tiles > 64;
    const dim3 rows((a.rows + 3) / 4);
    if (picks_from_logits(a) && a.V <= 64 * kFewSlots) hipLaunchKernelGGL((token_logprobs_finish_kernel<DT, kFewSlots, 1>), rows, dim3(256), 0, st, a);
    else if (picks_from_logits(a)) hipLaunchKernelGGL((token_logprobs_finish_kernel<DT, kMoreSlots, 1>), rows, dim3(256), 0, st, a);
    else if (team) hipLaunchKernelGGL((token_logprobs_finish_kernel<DT, 0, 4>), dim3(a.rows), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((token_logprobs_finish_kernel<DT, 0, 1>), rows, dim3(256), 0, st, a);
    record_launch("token_logprobs", grid.x, 256, (uint64_t)a.rows * a.V);
}

}  // namespace

}  // namespace iomx

using namespace iomx;

extern "C" int iomx_token_logprobs_workspace(int dtype, const iomx_view* logits, const iomx_view* tokens,
                                             const iomx_view* logprobs, const iomx_view* entropy,
                                             const iomx_view* top_ids, const iomx_view* top_logprobs,
                                             uint64_t* bytes, uint64_t* alignment) {
    if (!bytes || !alignment) return IOMX_ERR_INVALID;
    LogprobsArgs a = {};
    IOMX_TRY(logprobs_request(dtype, logits, tokens, logprobs, entropy, top_ids, top_logprobs, &a));
    uint64_t stats, cells;
    IOMX_TRY(logprobs_layout(dtype, &a, &stats, &cells));
    *bytes = (stats + cells) * 4;
    *alignment = 256;
    return IOMX_OK;
}

extern "C" int iomx_launch_token_logprobs(int dtype, const iomx_view* logits, const iomx_view* tokens,
                                          const iomx_view* logprobs, const iomx_view* entropy,
                                          const iomx_view* top_ids, const iomx_view* top_logprobs,
                                          void* workspace, uint64_t workspace_bytes, iomx_stream_t stream) {
    LogprobsArgs a = {};
    IOMX_TRY(logprobs_request(dtype, logits, tokens, logprobs, entropy, top_ids, top_logprobs, &a));
    uint64_t stats, cells;
    IOMX_TRY(logprobs_layout(dtype, &a, &stats, &cells));
    if (!workspace || workspace_bytes < (stats + cells) * 4 || (reinterpret_cast<uintptr_t>(workspace) & 255u))
        return IOMX_ERR_INVALID;
    a.stats = static_cast<float*>(workspace);
    a.cell_max = cells ? a.stats + stats : nullptr;
    const hipStream_t st = native(stream);
    if (dtype == IOMX_DT_BF16) launch_logprobs<IOMX_DT_BF16>(a, st);
    else if (dtype == IOMX_DT_F16) launch_logprobs<IOMX_DT_F16>(a, st);
    else launch_logprobs<IOMX_DT_F32>(a, st);
    IOMX_HIP(hipGetLastError());
    return IOMX_OK;
}
