/* mi_attention.h - attention of many sequences over a cache of keys and values in pages.
 *
 * mi_linear and mi_linear_batch take the projections of a whole batch of conversations; this header adds what lies
 * between them: the keys and values of one layer in a pool of pages that all sequences share, in fp16, int8 or Q4 (the
 * kinds that weights come in), rows written and quantised on the way, read back, and attention over them for any number of
 * new tokens per sequence: one (a decode step), a chunk of a prompt, or both in one batch.  A model with a sliding window
 * says how many positions a query sees, and how many first ones stay visible.
 *
 * The reference has one sequence, one contiguous fp16 cache and no window (KV cache QW/src/layers/attention.cpp:111-131,
 * kernels QW/kernels/attention.cl); what a query computes here is what those kernels compute for it, softmax(q k scale) v
 * per query head, key/value heads shared by n_heads / n_kv_heads query heads, with scores and sums in fp32.
 *
 * Conventions are those of mi_linear.h: 1 = enqueued, 0 and an "ERROR: ..." line on stderr = refused; nothing is allocated,
 * copied or waited for; device pointers are the caller's.  The structs are read during the call and may go away after it.
 * Lengths and page tables are device memory, read by the kernels: a captured call follows them from replay to replay.
 * Work split over the keys of a sequence meets in the stream's workspace, so it needs a stream of mi_stream_create (or the
 * null stream); on other streams a sequence's keys are not split, which is slower for few long sequences.  As with
 * every launch that uses the workspace, a graph replays on the stream it was captured on.
 */
#ifndef MI_ATTENTION_H
#define MI_ATTENTION_H

#ifdef __cplusplus
extern "C" {
#endif

#define MI_KV_F16 0
#define MI_KV_INT8 8
#define MI_KV_Q4 4

/* The keys and values of one layer: two pools [n_pages][n_kv_heads][page_size][row], a row being the head_dim values of one
 * position and head:
 *   MI_KV_F16   fp16; k_scale and v_scale are not used;
 *   MI_KV_INT8  int8 codes and an fp16 scale per row, scales [n_pages][n_kv_heads][page_size]: scale = fp16(greatest
 *               |x| / 127), code = x / scale rounded to the nearest integer (ties to even);
 *   MI_KV_Q4    4-bit codes plus 8, the even element in the low half of a byte, and an fp16 scale for each 32 elements,
 *               scales [n_pages][n_kv_heads][page_size][head_dim / 32]: scale = fp16(greatest |x| / 7).
 * The value of an element is the fp16 number nearest to code * scale.  Where the scale is 0 (all below about 2^-18 for int8,
 * 2^-22 for Q4) the codes are 0; a scale whose greatest value would pass 65504 is the one below that does not (515.5, 9352);
 * a row (Q4: 32 elements) that holds an infinity or a NaN gets the scale NaN and reads back as NaN.
 * head_dim 64 or 128; page_size any number of positions (with multiples of 16 the attention looks pages up 16 positions at
 * a time).  A contiguous cache is one of pages as long as the longest sequence.  Pools are 16-byte aligned (scales 8), and a
 * page of one pool, n_kv_heads * page_size * row bytes, is less than 2 GiB. */
typedef struct mi_kv_cache {
    void *k, *v;
    void *k_scale, *v_scale;
    int kind;
    int n_pages, page_size, n_kv_heads, head_dim;
} mi_kv_cache;

/* The sequences of a call.  Rows q_start[b] .. q_start[b + 1] - 1 of the call's row arrays are the new tokens of sequence b,
 * which has kv_len[b] positions, these included: row q_start[b] + i is at position kv_len[b] - n_b + i, n_b = q_start[b + 1] -
 * q_start[b] (0: nothing of the sequence is computed).  Position p lies in page pages[b * max_pages + p / page_size], row
 * p % page_size.  Device memory: q_start [n_seqs + 1] (ascending, within 0 .. n_tokens), kv_len [n_seqs], pages
 * [n_seqs][max_pages].  n_tokens: rows that the row arrays have; rows behind q_start[n_seqs] are padding and left as they
 * are.  max_tokens: what n_b is at most, a hint; a wrong one costs time, nothing else.  The kernels are chosen
 * by it and by max_pages * page_size, the bound of the lengths: a table much wider than that costs time for chunks of prompts.
 * Where q_start goes down somewhere it is not said which rows are computed, but no other memory and no later call is touched.
 * Several sequences may share pages that they only read.  A position before 0, past max_pages * page_size or in a page that
 * is not in 0 .. n_pages - 1 has no place in the cache: it is not written, reads back as zeros and is not seen. */
typedef struct mi_kv_batch {
    const int *q_start, *kv_len, *pages;
    int n_seqs, n_tokens, max_tokens, max_pages;
} mi_kv_batch;

/* Keys and values of the new tokens into their pages: row r's are k + r * ld_k and v + r * ld_v (fp16 elements, 2-byte aligned,
 * n_kv_heads * head_dim of them each), so they may be parts of stacked q | k | v rows.  Two rows at one position of one page:
 * either one's values stay, or for quantised kinds a mixture; a host that shares pages writes them once. */
int mi_kv_write(void* stream, const mi_kv_cache* cache, const mi_kv_batch* batch, const void* k, int ld_k, const void* v, int ld_v);

/* The same rows back out of their pages, as fp16: row r to k_out + r * ld_k and v_out + r * ld_v.  With q_start = 0, kv_len[0],
 * kv_len[0] + kv_len[1], ... that is every position of every sequence. */
int mi_kv_read(void* stream, const mi_kv_cache* cache, const mi_kv_batch* batch, void* k_out, int ld_k, void* v_out, int ld_v);

/* One call of mi_attention.  q: fp16 rows of n_heads * head_dim elements, ld_q from row to row (2-byte aligned); out: the same with
 * ld_out, written.  n_heads is a multiple of the cache's n_kv_heads.  Row at position p sees position j if 0 <= j <= p
 * and, with window > 0, also j > p - window or j < sinks (window <= 0: sinks mean nothing).  scale: what products are multiplied
 * with before the softmax, usually 1 / sqrt(head_dim); greater than 0, at most 65504.  A row that sees nothing (and one whose
 * scores are all -infinity) is written as zeros.  What a masked position holds, NaN and infinities included, does
 * not touch the row (next to such values a row may be summed in another order, with other roundings, and a chunk of many rows takes a
 * hundred times as long).  Scores may be of any size that fp32 holds.  out may not overlap q or the cache. */
typedef struct mi_attention_call {
    const mi_kv_cache* cache;
    const mi_kv_batch* batch;
    const void* q;
    void* out;
    int ld_q, ld_out, n_heads;
    float scale;
    int window, sinks;
} mi_attention_call;

/* Attention of the new tokens, whose own keys and values are in the cache already (mi_kv_write before it on the stream).
 * Products are fp16 x fp16, scores and sums fp32; a probability, relative to the row's running maximum, is rounded to fp16 once
 * before it meets the values.  The same call on the same data gives the same bits. */
int mi_attention(void* stream, const mi_attention_call* call);

#ifdef __cplusplus
}
#endif
#endif
