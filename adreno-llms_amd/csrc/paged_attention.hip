// Attention of many sequences' new tokens over a cache in pages (mi_attention): out = sum_j w_j v_j / sum_j w_j over the
// positions j that a row sees, w_j = exp(scale q k_j - their maximum), per query head.
#include "device_math.h"
#include "paged.h"

namespace mi {
namespace {

// A stored element as the number it stands for: the fp16 number nearest to code * scale.
template <int KIND, int D>
__device__ __forceinline__ float element(const uint8_t* pool, const uint16_t* scales, int64_t row, int e) {
    if constexpr (KIND == MI_KV_F16) return h_f(reinterpret_cast<const uint16_t*>(pool)[row * D + e]);
    if constexpr (KIND == MI_KV_INT8)
        return static_cast<float>(static_cast<_Float16>(static_cast<float>(static_cast<int8_t>(pool[row * D + e])) * h_f(scales[row])));
    const int b = pool[(row * D + e) / 2], code = (e & 1 ? b >> 4 : b & 15) - 8;
    return static_cast<float>(static_cast<_Float16>(static_cast<float>(code) * h_f(scales[row * (D / 32) + e / 32])));
}

// One wavefront per row and query head: a lane takes one of 64 positions for the scores, D / 64 elements for the sums.
template <int KIND, int D>
__global__ __launch_bounds__(64) void paged_rows_kernel(const AttentionArgs a) {
    __shared__ float q[D], w[64];
    __shared__ int64_t at[64];
    const int lane = threadIdx.x, r = blockIdx.x / a.n_heads, head = blockIdx.x % a.n_heads;
    const int b = sequence_of(a.p.q_start, a.p.n_seqs, r);
    if (b < 0) return;
    const Span s = span_of(a.p.q_start[b], a.p.q_start[b + 1], a.p.kv_len[b], a.p.n_tokens);
    if (r - s.first >= s.n) return;
    const int pos = s.pos + (r - s.first), kvh = head / (a.n_heads / a.p.n_kv_heads);
    for (int e = lane; e < D; e += 64) q[e] = h_f(a.q[r * a.ld_q + head * D + e]);
    const Tiles tiles = tiles_of(pos, pos, a.p.cap, a.window, a.sinks, 64);
    float base = -1.0e30f, sum = 0.0f, acc[D / 64];
    for (int d = 0; d < D / 64; ++d) acc[d] = 0.0f;
    for (int t = 0; t < tiles.count; ++t) {
        const int j = tile_at(tiles, t) * 64 + lane;
        int64_t row = -1;
        if (j < a.p.cap && sees(pos, j, a.window, a.sinks)) {
            const int page = divide(j, a.p.page), number = a.p.pages[static_cast<int64_t>(b) * a.p.max_pages + page];
            if (number >= 0 && number < a.p.n_pages) row = row_number(a.p, number, kvh, j - page * a.p.page.d);
        }
        __syncthreads();
        float score = -__builtin_huge_valf();
        if (row >= 0) {
            float dot = 0.0f;
            for (int e = 0; e < D; ++e) dot = fmaf(q[e], element<KIND, D>(a.p.k, a.p.k_scale, row, e), dot);
            score = dot * a.scale;
        }
        const float top = fmaxf(base, wave_max(score)), alpha = __expf(base - top), mine = __expf(score - top);
        w[lane] = mine;
        at[lane] = row;
        __syncthreads();
        base = top;
        sum *= alpha;
        for (int d = 0; d < D / 64; ++d) acc[d] *= alpha;
        for (int i = 0; i < 64; ++i) {
            if (at[i] < 0) continue;
            sum += w[i];
            for (int d = 0; d < D / 64; ++d) acc[d] = fmaf(w[i], element<KIND, D>(a.p.v, a.p.v_scale, at[i], lane + 64 * d), acc[d]);
        }
    }
    for (int d = 0; d < D / 64; ++d)
        a.out[r * a.ld_out + head * D + lane + 64 * d] = f_h(sum == 0.0f ? 0.0f : acc[d] / sum);
}

}  // namespace

bool launch_paged_attention(hipStream_t s, const AttentionArgs& a, void* /*workspace*/) {
    const dim3 grid(a.p.n_tokens * a.n_heads), block(64);
    auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, block, 0, s, a); };
    const bool wide = a.head_dim == 128;
    if (a.kind == MI_KV_F16) wide ? go(paged_rows_kernel<MI_KV_F16, 128>) : go(paged_rows_kernel<MI_KV_F16, 64>);
    else if (a.kind == MI_KV_INT8) wide ? go(paged_rows_kernel<MI_KV_INT8, 128>) : go(paged_rows_kernel<MI_KV_INT8, 64>);
    else wide ? go(paged_rows_kernel<MI_KV_Q4, 128>) : go(paged_rows_kernel<MI_KV_Q4, 64>);
    return MI_HIP_OK(hipGetLastError());
}

}  // namespace mi
