// What the kernels over a paged cache are handed: the structs of mi_attention.h as their kernels' arguments.
#pragma once
#include "../../include/mi_attention.h"
#include "common.h"
#include "paged_rule.h"

namespace mi {

struct PagedArgs {
    const uint8_t *k, *v;                     // pools
    const uint16_t *k_scale, *v_scale;
    const int *q_start, *kv_len, *pages;
    int n_seqs, n_tokens, max_pages, n_pages, n_kv_heads;
    int cap;                                  // positions of a page table
    Divider page;                             // by page_size
};
// Checks a call's cache and batch (what the host can see of them) and makes the kernels' form; false: refused, and said.
bool paged_args(const char* who, const mi_kv_cache* cache, const mi_kv_batch* batch, PagedArgs* out);

// Bytes of a row of head_dim values, and of its scales.
constexpr int row_bytes(int kind, int D) { return kind == MI_KV_F16 ? 2 * D : kind == MI_KV_INT8 ? D : D / 2; }
constexpr int row_scales(int kind, int D) { return kind == MI_KV_F16 ? 0 : kind == MI_KV_INT8 ? 1 : D / 32; }

// The number of row (page, head, slot), counted over all of a pool.  (A page has fewer than 2^31 rows: paged_args.)
__device__ __forceinline__ int64_t row_number(const PagedArgs& a, int page, int head, int slot) {
    return static_cast<int64_t>(static_cast<uint64_t>(static_cast<uint32_t>(page)) * static_cast<uint32_t>(a.n_kv_heads * a.page.d)) +
           static_cast<uint32_t>(head * a.page.d + slot);
}

// paged_attention.hip
struct AttentionArgs {
    PagedArgs p;
    const uint16_t* q;
    uint16_t* out;
    int64_t ld_q, ld_out;
    int n_heads, kind, head_dim, max_tokens;
    int window, sinks;
    float scale;
};
bool launch_paged_attention(hipStream_t s, const AttentionArgs& a, const StreamRoom& room);

}  // namespace mi
