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

/* Rotary positions of new rows, between the projections and the cache.  Of each head of head_dim elements the first rot_dim are
 * pairs (x, y): elements i and i + rot_dim / 2, or with `interleaved` not 0 2 i and 2 i + 1, i = 0 .. rot_dim / 2 - 1, and become
 *   (x cos a - y sin a, y cos a + x sin a),  a = position[axis of i][row] * inv_freq[i];
 * the elements behind them are copied.  One position per row and axis: a text has one axis, pictures and films have their rows' time, line
 * and column.  A negative position turns the other way, by which keys can be turned back.
 *   q, q_out    rows of n_heads heads, ld_q and ld_q_out elements apart; k, k_out: of n_kv_heads, the same (either may have 0 heads and be
 *               null).  fp16, 2-byte aligned.  An output may be its own input, with the same ld; else outputs overlap nothing.
 *   position    int32 [n_axes][n_tokens], inv_freq fp32 [rot_dim / 2]: device memory.
 *   axis        host memory, read during the call: of each i the number of its axis; null: all 0.
 * head_dim even, up to 256; rot_dim even, 0 to head_dim; n_axes 1 to 4.  The angle is taken in 64 bits and what their roundings
 * leave, so that cosine and sine are right to fp32's last bits at any position; an output is rounded to fp16 once.  The reference has one axis, the halves' pairs and fp16 tables
 * (QW/kernels/rope.cl, QW/src/layers/attention.cpp:133-172), as mi_decoder_step keeps them. */
typedef struct mi_rope_call {
    const void *q, *k;
    void *q_out, *k_out;
    const float* inv_freq;
    const int* position;
    const unsigned char* axis;
    int ld_q, ld_k, ld_q_out, ld_k_out;
    int n_tokens, n_heads, n_kv_heads, head_dim, rot_dim, n_axes, interleaved;
} mi_rope_call;
int mi_rope(void* stream, const mi_rope_call* call);

/* ---- several continuations of a sequence ----------------------------------------------------------------------
 *
 * A host that has tokens drafted ahead, or keeps several beams, has more than one continuation of a sequence in the cache. */

/* Attention of drafted tokens.  The new rows of a sequence (mi_kv_write has put their keys and values behind the others, in the
 * order of the rows) are no text one after the other but, say, a tree: row i sees all positions before the sequence's new ones,
 * and its new row j if bit j % 32 of seen[row * words + j / 32] is set, `row` the number of i in the batch; its own bit is set by
 * the caller too.  Bits of rows that the sequence does not have count for nothing, rows past 32 * words are seen by none.
 * With a window the earlier positions j are those with j > p - window or j < sinks, p = position[row] being the row's place in its
 * text (as for mi_rope; taken as no less than the number of earlier positions and less than kv_len); the bits alone
 * decide among new rows.  seen [n_tokens][words] and position [n_tokens]: device memory, 4-byte aligned; position may be null where
 * there is no window.  words 1 to 65536.  All else as mi_attention. */
typedef struct mi_tree_mask {
    const unsigned* seen;
    const int* position;
    int words;
} mi_tree_mask;
int mi_attention_tree(void* stream, const mi_attention_call* call, const mi_tree_mask* tree);

/* Of the new rows of every sequence, accepted drafts stay and move together.  Of sequence b, with n_b new rows behind `before` = kv_len[b] -
 * n_b earlier positions, the rows numbered keep[q_start[b] + i], i = 0 .. kept[b] - 1, ascending, each of 0 .. n_b - 1, become
 * positions before + i, in every cache of `caches`; what the other positions hold is left as it is.  new_len[b] = before + kept[b] (kept
 * taken as within 0 .. n_b; less than 0 counts as 0) unless new_len is null; it overlaps none of the arrays that are read.
 * caches: n_caches of them, the layers of a model say, which differ in their pools alone; no pool is there twice, nor, of int8 and Q4 caches, one of
 * scales.  keep [n_tokens] (what lies behind a
 * sequence's kept ones is not read), kept [n_seqs], new_len [n_seqs]: device memory, 4-byte aligned.  Rows move as they are stored.  A row
 * or a place that is not in the cache, or a number out of range, moves nothing.  Where numbers do not ascend it is not said
 * which rows end up where, but no other positions are touched.  No two sequences of a call share a page that holds a new row. */
int mi_kv_keep(void* stream, const mi_kv_cache* caches, int n_caches, const mi_kv_batch* batch, const int* keep, const int* kept,
               int* new_len);

/* Sequences go on as copies of others: beam search's reordering.  Sequence b becomes what sequence f = source[b] is: new_len[b] = kv_len[f];
 * new_pages[b] is pages[f], up to the pages that kv_len[f] positions need, -1 behind them, but for a last page that is not full: its
 * kv_len[f] % page_size rows are copied, in every cache of `caches`, to page fresh[b], which takes its place (f = b keeps its own and fresh[b] is
 * not used).  Full pages are shared from then on, which the host counts.  source[b] outside 0 .. n_seqs - 1: new_len[b] = 0, all
 * pages -1.  kv_len[f] beyond the table, or a page (old or fresh) that is not in the pool: the number is passed on, nothing is copied.
 * `caches` as for mi_kv_keep.  A fresh page is nobody's: neither in `pages` nor twice in `fresh` among those that are used.  kv_len, source, fresh, new_len
 * [n_seqs], pages, new_pages [n_seqs][max_pages]: device memory, 4-byte aligned; new_len and new_pages overlap none of the others. */
typedef struct mi_kv_reorder_call {
    const int *kv_len, *pages, *source, *fresh;
    int *new_len, *new_pages;
    int n_seqs, max_pages;
} mi_kv_reorder_call;
int mi_kv_reorder(void* stream, const mi_kv_cache* caches, int n_caches, const mi_kv_reorder_call* call);

#ifdef __cplusplus
}
#endif
#endif
