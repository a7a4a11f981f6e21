// Log probabilities of given tokens, entropy and the most likely tokens of vocabulary rows.
#include "iomx_packed.hpp"

namespace iomx {

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
};

template <int DT>
__device__ __forceinline__ float logit_at(const uint8_t* row, uint32_t c) {
    const uint64_t slot = (uint64_t)(c >> 4) * kTileSlots + (c & 15u);
    if constexpr (DT == IOMX_DT_F32) return reinterpret_cast<const float*>(row)[slot];
    else if constexpr (DT == IOMX_DT_BF16) return as_f32((uint32_t)reinterpret_cast<const uint16_t*>(row)[slot] << 16);
    else return (float)reinterpret_cast<const _Float16*>(row)[slot];
}

// One workgroup per row: a pass for the maximum, one for the sums, one for each top token.
template <int DT>
__global__ __launch_bounds__(256) void token_logprobs_kernel(const LogprobsArgs a) {
    constexpr float inf = __builtin_inff();
    __shared__ float shared_a[4], shared_b[4];
    __shared__ uint32_t shared_i[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t plane_index = divided(blockIdx.x, a.R, a.div_rows);
    const uint32_t r = blockIdx.x - plane_index * a.R;
    uint64_t plane[6];
    walk_planes(a.walk, plane_index, plane);
    const uint8_t* row = a.logits + (plane[0] * a.logits_plane + (uint64_t)(r >> 4) * a.tile_cols * kTileSlots
                                     + (r & 15u) * kTile) * (DT == IOMX_DT_F32 ? 4 : 2);
    // the maximum; a NaN or +inf shows as bad
    float m = -inf;
    bool bad = false;
    for (uint32_t c = tid; c < a.V; c += 256) {
        const float x = logit_at<DT>(row, c);
        bad = bad || !(x < inf);
        m = x > m ? x : m;
    }
    for (int off = 1; off < 64; off *= 2) m = fmaxf(m, __shfl_xor(m, off));
    if (lane == 0) shared_a[wave] = m;
    bad = __syncthreads_or(bad) != 0;
    m = fmaxf(fmaxf(shared_a[0], shared_a[1]), fmaxf(shared_a[2], shared_a[3]));
    bad = bad || m == -inf;
    __syncthreads();
    float sum = 0.0f, weighted = 0.0f;     // sum e^(x - m), sum (x - m) e^(x - m)
    for (uint32_t c = tid; c < a.V; c += 256) {
        const float x = logit_at<DT>(row, c);
        if (x == -inf) continue;
        const float e = expf(x - m);
        sum += e;
        weighted += (x - m) * e;
    }
    for (int off = 1; off < 64; off *= 2) {
        sum += __shfl_xor(sum, off);
        weighted += __shfl_xor(weighted, off);
    }
    if (lane == 0) { shared_a[wave] = sum; shared_b[wave] = weighted; }
    __syncthreads();
    sum = shared_a[0] + shared_a[1] + shared_a[2] + shared_a[3];
    weighted = shared_b[0] + shared_b[1] + shared_b[2] + shared_b[3];
    __syncthreads();
    const float log_sum = logf(sum), nan = as_f32(kQuietNanF32);
    const uint64_t row_at = (uint64_t)(r >> 4), in_row = (r & 15u) * kTile;
    for (uint32_t g = tid; a.tokens && g < a.G; g += 256) {
        const uint64_t at = (row_at * a.given_tile_cols + (g >> 4)) * kTileSlots + in_row + (g & 15u);
        const uint32_t id = (uint32_t)a.tokens[plane[1] * a.given_plane + at];
        a.logprobs[plane[2] * a.given_plane + at] = id >= a.V ? -inf : bad ? nan : logit_at<DT>(row, id) - m - log_sum;
    }
    if (a.entropy && tid == 0)
        a.entropy[plane[3] * a.entropy_plane + row_at * kTileSlots + in_row] = bad ? nan : log_sum - weighted / sum;
    if (!a.top_ids) return;
    float last = inf;
    uint32_t last_id = 0;
    for (uint32_t k = 0; k < a.K; ++k) {
        float best = -inf;
        uint32_t best_id = 0xFFFFFFFFu;
        for (uint32_t c = tid; c < a.V; c += 256) {
            const float x = logit_at<DT>(row, c);
            const bool after = k == 0 || x < last || (x == last && c > last_id);
            if (after && (x > best || best_id == 0xFFFFFFFFu)) { best = x; best_id = c; }
        }
        auto better = [&](float x, uint32_t id) {
            if (x > best || (x == best && id < best_id)) { best = x; best_id = id; }
        };
        for (int off = 1; off < 64; off *= 2) {
            const float x = __shfl_xor(best, off);
            better(x, __shfl_xor(best_id, off));
        }
        if (lane == 0) { shared_a[wave] = best; shared_i[wave] = best_id; }
        __syncthreads();
        for (uint32_t w = 0; w < 4; ++w) better(shared_a[w], shared_i[w]);
        __syncthreads();
        last = best;
        last_id = best_id;
        if (tid == 0) {
            const uint64_t at = (row_at * a.top_tile_cols + (k >> 4)) * kTileSlots + in_row + (k & 15u);
            a.top_ids[plane[4] * a.top_plane + at] = bad ? -1 : (int32_t)best_id;
            a.top_logprobs[plane[5] * a.top_plane + at] = bad ? nan : best - m - log_sum;
        }
    }
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
    *bytes = 0;
    *alignment = 1;
    return IOMX_OK;
}

extern "C" int iomx_launch_token_logprobs(int dtype, const iomx_view* logits, const iomx_view* tokens,
                                          const iomx_view* logprobs, const iomx_view* entropy,
                                          const iomx_view* top_ids, const iomx_view* top_logprobs,
                                          void* workspace, uint64_t workspace_bytes, iomx_stream_t stream) {
    (void)workspace;
    (void)workspace_bytes;
    LogprobsArgs a = {};
    IOMX_TRY(logprobs_request(dtype, logits, tokens, logprobs, entropy, top_ids, top_logprobs, &a));
    const dim3 grid((uint32_t)(a.walk.planes * a.R));
    const hipStream_t st = native(stream);
    if (dtype == IOMX_DT_BF16) hipLaunchKernelGGL(token_logprobs_kernel<IOMX_DT_BF16>, grid, dim3(256), 0, st, a);
    else if (dtype == IOMX_DT_F16) hipLaunchKernelGGL(token_logprobs_kernel<IOMX_DT_F16>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(token_logprobs_kernel<IOMX_DT_F32>, grid, dim3(256), 0, st, a);
    record_launch("token_logprobs", grid.x, 256, (uint64_t)grid.x * a.V);
    IOMX_HIP(hipGetLastError());
    return IOMX_OK;
}
