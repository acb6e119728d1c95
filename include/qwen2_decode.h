/*
 * qwen2_decode.h -- C ABI of the fused decode-step kernels that sit between
 * the W4G64 linears of a Qwen2 decoder layer (one token per sequence, bf16
 * hidden states).  Same conventions as w4g64.h: plain device pointers, sizes,
 * a HIP stream as `void*`, int status codes W4G64_STATUS_*, the message of a
 * failed call in w4g64_last_error().  Nothing here allocates or synchronizes.
 *
 * With these, one decoder layer's decode step is at most seven launches:
 *   add_rmsnorm -> W4G64 q|k|v (one N = (H + 2 KVH) * D launch, bias)
 *   -> decode_attention -> W4G64 o_proj -> add_rmsnorm
 *   -> W4G64 gate|up (one N = 2 I launch) -> W4G64 down_proj,
 * and the step ends with add_rmsnorm -> lm_head (logits and greedy token).
 * At batch 1 it is five: each add_rmsnorm after the first is formed in the
 * staging of the linear that follows it (w4g64_linear_rmsnorm), and the down
 * projection's K-split partial sums are added there too
 * (w4g64_linear_partials, W4G64_DTYPE_F32_PARTIALS).
 */
#ifndef QWEN_INT4_HIP_QWEN2_DECODE_H
#define QWEN_INT4_HIP_QWEN2_DECODE_H

#include <stdint.h>

#include "w4g64.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Start of a decode step for `batch` sequences at the common position
 * p = *position (a device int64):
 *   x[b]   = embed[token_ids[b]]               (bf16 [batch, hidden]; a row of NaN
 *                                                for an id outside [0, vocab))
 *   cos[b][d], sin[b][d] = bf16(cos / sin(float(p) * inv_freq[d % (head_dim / 2)]))
 *                                              (bf16 [batch, head_dim], fp32 math)
 *   normed[b] = bf16(bf16(x[b] * rsqrt(mean(x[b]^2) + eps)) * norm_weight)
 *                                              (only when norm_weight and normed are
 *                                                given: the first layer's input norm)
 * token_ids int64 [batch], embed bf16 [vocab, hidden] (16-byte aligned, as x,
 * norm_weight and normed), inv_freq fp32 [head_dim / 2] (the rotary module's
 * buffer).  head_dim == 128.
 * Replaces: the embedding lookup of QwenModel.forward, RotaryEmbedding.forward
 *           for one position and the first layer's input RMSNorm
 *           (src/qwen_int4/model.py:22-31, :40-44, :182, :190). */
int qwen2_decode_prologue(const int64_t* token_ids, const void* embed, const int64_t* position, const float* inv_freq,
                          void* x, void* cos, void* sin, const void* norm_weight, float eps, void* normed,
                          int64_t batch, int64_t hidden, int64_t vocab, int64_t head_dim, void* stream);

/* Residual add + RMSNorm over `rows` rows of `hidden` bf16 values:
 *   s        = x                                   (delta == NULL)
 *            = bf16(x + bf16(delta))               (delta bf16, fp32, or fp32 partial
 *                                                   sums: W4G64_DTYPE_F32_PARTIALS)
 *   out_sum  = s                                   (may be NULL; may alias x)
 *   out_norm = bf16(bf16(s * rsqrt(mean(s^2) + eps)) * weight)
 * in fp32 arithmetic with the reference's two roundings.  hidden is a
 * multiple of 8, at most 8192; all pointers 16-byte aligned.
 * Replaces: RMSNorm.forward (src/qwen_int4/model.py:40-44) and the residual
 *           adds of DecoderLayer.forward (model.py:149-154; the MLP output is
 *           cast to bf16 first, model.py:136). */
int qwen2_add_rmsnorm(const void* x, const void* delta, int delta_dtype, const void* weight, float eps,
                      void* out_sum, void* out_norm, int64_t rows, int64_t hidden, void* stream);

/* Bytes of workspace qwen2_decode_attention needs (arrival counters, then
 * fp32 per-chunk partial results).  The counter area must be zero before the
 * first call; every call leaves it zero.  Calls sharing a workspace must be
 * ordered on one stream. */
int64_t qwen2_decode_attention_workspace_bytes(int64_t batch, int64_t num_kv_heads, int64_t max_length);

/* One decode step of grouped-query attention for `batch` sequences that all
 * sit at the same position p = *position (a device int64; clamped to
 * [0, max_length)):
 *   qkv      bf16 [batch, (num_heads + 2 num_kv_heads) * head_dim]: the fused
 *            q|k|v projection of the new token (bias included);
 *   cos, sin bf16 [batch, head_dim]: the rotary factors of position p;
 *   k_cache, v_cache bf16 [batch, num_kv_heads, max_length, head_dim].
 * Rotates q and k as q * cos + rotate_half(q) * sin with bf16 rounding after
 * each product and after the sum, writes the rotated key and the value at
 * position p, and writes
 *   out[b, h * head_dim + d] = bf16( softmax_t(q_h . k_t * scale) . v_t[d] ),
 *   t = 0..p, query head h reading key/value head h / (num_heads / num_kv_heads),
 * with fp32 scores, softmax and sums.  head_dim == 128,
 * num_heads / num_kv_heads <= 8, max_length <= 17408.  qkv, the caches and
 * the workspace must be 16-byte aligned, out 8-byte aligned.
 * Replaces: the rotary step and attention of QwenAttention.forward for one
 *           cached token (src/qwen_int4/model.py:17-31, :61-122). */
int qwen2_decode_attention(const void* qkv, const void* cos, const void* sin, void* k_cache, void* v_cache,
                           const int64_t* position, void* out, int64_t batch, int64_t num_heads,
                           int64_t num_kv_heads, int64_t head_dim, int64_t max_length, float scale,
                           void* workspace, int64_t workspace_bytes, void* stream);

/* qwen2_decode_attention without its merge: the same rotary step and cache
 * write, and every 64-position chunk's workgroup leaves its partial result
 * (per query head: score maximum m_c, sum l_c of exp(score - m_c), and the
 * exp-weighted value sums acc_c[128], fp32) in the workspace; chunks past the
 * position leave m_c = -inf, l_c = 0 and zero sums.  No output row is
 * written: w4g64_linear_attention_merge merges the chunks in the staging of
 * the o_proj linear, with the result qwen2_decode_attention would have
 * written.  Same arguments and workspace as qwen2_decode_attention, minus
 * `out`; the counter area is left untouched.
 * Replaces: with w4g64_linear_attention_merge, the rotary step, attention and
 *           o_proj of QwenAttention.forward for one cached token
 *           (src/qwen_int4/model.py:17-31, :61-122). */
int qwen2_decode_attention_partials(const void* qkv, const void* cos, const void* sin, void* k_cache,
                                    void* v_cache, const int64_t* position, int64_t batch, int64_t num_heads,
                                    int64_t num_kv_heads, int64_t head_dim, int64_t max_length, float scale,
                                    void* workspace, int64_t workspace_bytes, void* stream);

/* Bytes of workspace qwen2_prefill_attention must be given: bf16 [batch,
 * num_heads, length, head_dim] (checked; written only where out overlaps qkv,
 * any allocation of that size serves elsewhere, qkv itself among them). */
int64_t qwen2_prefill_attention_workspace_bytes(int64_t batch, int64_t num_heads, int64_t length);

/* Attention over a prompt of `length` positions per sequence.
 *   qkv bf16 [batch * length, (num_heads + 2 num_kv_heads) * head_dim] (q | k | v
 *     projections of every position, row b * length + i);
 *   cos, sin bf16 [batch * length, head_dim]: the rotary factors of position i;
 *   k_cache, v_cache bf16 [batch, num_kv_heads, max_length, head_dim].
 * Rotates q and k as qwen2_decode_attention does, writes the rotated keys and
 * the values at positions 0..length-1 of the caches (later positions are left
 * alone), and writes
 *   out[b * length + i, h * head_dim + d] =
 *       bf16( softmax_{t <= i}(q_{h,i} . k_t * scale) . v_t[d] )
 * with fp32 scores, softmax and sums (causal mask).  head_dim == 128,
 * num_heads / num_kv_heads <= 8, length <= max_length; qkv, the caches and
 * the workspace 16-byte aligned.  out may overlap qkv (the queries then go
 * through the workspace, which then must overlap neither).
 * Replaces: the rotary step, cache update and attention of
 *           QwenAttention.forward over a prompt (src/qwen_int4/model.py:17-31,
 *           :61-122, the causal mask of :94-120). */
int qwen2_prefill_attention(const void* qkv, const void* cos, const void* sin, void* k_cache, void* v_cache,
                            void* out, int64_t batch, int64_t length, int64_t num_heads, int64_t num_kv_heads,
                            int64_t head_dim, int64_t max_length, float scale, void* workspace,
                            int64_t workspace_bytes, void* stream);

/* Attention of `length` new positions per sequence after `past` cached ones,
 * with a growing cache and a key mask (the cached-generation path of a
 * left-padded batch).  total = past + length.
 *   q bf16 [batch * length, num_heads * head_dim], k, v bf16 [batch * length,
 *     num_kv_heads * head_dim]: the projections, row b * length + i;
 *   cos, sin bf16 [batch * length, head_dim]: the rows' rotary factors;
 *   past_k, past_v bf16 [batch, num_kv_heads, past, head_dim] (unused for past 0);
 *   mask uint8 [batch, total] or NULL: a zero excludes the key for its sequence.
 * Rotates q and k as qwen2_decode_attention does, writes new_k, new_v bf16
 * [batch, num_kv_heads, total, head_dim] = the past followed by the rotated
 * keys / the values (must not overlap the past), and writes
 *   out[b * length + i, h * head_dim + d] =
 *       bf16( softmax_t(q_{h,i} . k_t * scale) . v_t[d] ),
 *       t <= past + i and mask[b, t] != 0,
 * with fp32 scores, softmax and sums; a row without such a t gives zeros.
 * head_dim == 128; q, k, v and the caches 16-byte aligned.
 * Replaces: the rotary step, cache concatenation, masking and attention of
 *           QwenAttention.forward (src/qwen_int4/model.py:61-122). */
int qwen2_cached_attention(const void* q, const void* k, const void* v, const void* cos, const void* sin,
                           const void* past_k, const void* past_v, const uint8_t* mask, void* new_k, void* new_v,
                           void* out, int64_t batch, int64_t length, int64_t past, int64_t num_heads,
                           int64_t num_kv_heads, int64_t head_dim, float scale, void* stream);

/* ---------------------------------------------------------------------------
 * Paged serving: batches of sequences whose cached keys and values lie in pages
 * of one pool, several new positions per sequence and call.
 *
 * Rows (tokens) are packed: sequence b's new positions are rows cu_rows[b] ..
 * cu_rows[b + 1] - 1, and they are the last ones of its lengths[b] cached
 * positions: row i of n sits at position lengths[b] - n + i.  Position t of
 * sequence b lies in page page_table[b][t / page_size], place t % page_size.
 * cu_rows, lengths and page_table are read on the device; what they hold is
 * bounded there: no access leaves the buffers whatever it is, and no row from
 * cu_rows[batch] on is written but to be zeroed.
 * ------------------------------------------------------------------------- */

typedef struct qwen2_paged_cache {
    void* k;                       /* key of position t, head h: k + page * k_page + h * k_head */
    void* v;                       /*   + (t % page_size) * k_position; head_dim elements; v alike */
    int64_t k_page, k_head, k_position; /* strides in elements, multiples of 8 (16 bytes) */
    int64_t v_page, v_head, v_position;
    int64_t num_pages;             /* in [1, 2^31) */
    int64_t page_size;             /* a power of two in [16, 2^20] */
    const int32_t* page_table;     /* [batch, table_width], rows table_stride apart */
    int64_t table_width, table_stride;
    const int32_t* cu_rows;        /* [batch + 1], not falling, from 0 */
    const int32_t* lengths;        /* [batch], the new positions counted */
    int64_t batch, kv_heads, head_dim;
    int dtype;                     /* W4G64_DTYPE_BF16 or W4G64_DTYPE_F16: cache, q, k, v and outputs */
} qwen2_paged_cache;

/* Rows of a packed [rows, heads, head_dim] tensor: strides in elements. */
typedef struct qwen2_rows {
    void* data;                    /* 16-byte aligned */
    int64_t row, head;             /* multiples of 8 */
} qwen2_rows;

/* Rotates the new positions' queries and keys and writes keys and values into
 * their pages:
 *   out[r, h]                      = R(p) q[r, h]
 *   k of position p, head h        = R(p) k[r, h]
 *   v of position p, head h        = v[r, h]
 * where row r of sequence b has position p.  R(p) turns the first rotary_dim of
 * the head_dim dimensions, in pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1)
 * with `interleaved`, by the angle p * inv_freq[i]:
 *   (x, y) -> rotary_scale * (x cos - y sin, y cos + x sin);
 * the angle in 64 bits, the rest in fp32, rounded once.  (Stretched contexts are
 * a matter of inv_freq and rotary_scale.)  rotary_dim 0 turns nothing (inv_freq
 * may then be NULL).  out may be q itself (same data and strides).
 * A row whose page is not in the pool, or whose position is not in its table,
 * is not written to the cache.  Rows behind the last sequence are left as they
 * are, or zeroed in `out` with zero_rest.  Two rows of one call must not share
 * a place in the cache (sequences may share pages, but not the ones written).
 * head_dim and rotary_dim are multiples of 16, head_dim <= 256.
 * Replaces: the rotary step and cache concatenation of QwenAttention.forward
 *           (src/qwen_int4/model.py:17-31, :76-90) for packed sequences. */
int qwen2_paged_append(const qwen2_paged_cache* cache, const qwen2_rows* q, const qwen2_rows* k, const qwen2_rows* v,
                       const qwen2_rows* out, const float* inv_freq, int64_t rotary_dim, int interleaved,
                       float rotary_scale, int64_t rows, int64_t heads, int zero_rest, void* stream);

/* Attention of the new positions over the paged cache (theirs included: append
 * first):
 *   out[r, h] = softmax_t(scale * q[r, h] . k_t) v_t,   t = 0 .. p,
 * p the row's position, query head h reading key/value head
 * h / (heads / kv_heads); scores, softmax and sums in fp32, probabilities kept to
 * 16 bits (two terms), rounded once.  The first shared_pages entries of every
 * row of page_table must name the same pages (a prefix common to the batch): the
 * first row's are read, once for all sequences.  A row without a position
 * (lengths[b] too small) gives zeros; a row that reaches past its table, or to
 * a page that is not in the pool, gives NaN.  (Values are summed before the sum is
 * divided: the keys' number times the values' size has to stay in fp32.)  Rows behind the
 * last sequence are left as they are, or zeroed with zero_rest.  Keys and values at positions that
 * a row does not see take no part, whatever they hold.
 * An infinity or NaN among the values of a key that a row sees reaches the row
 * however small the key's weight.
 * head_dim is 64 or 128; heads a multiple of kv_heads; out must not overlap q.
 * A call is cut into workgroups by table_width and shared_pages, not by the lengths
 * (they are on the device): columns far behind the longest sequence do not change
 * the result but cost time.
 * The workspace (16-byte aligned) holds fp32 partial results; nothing in it
 * survives a call.  Calls sharing one must be ordered on one stream.
 * Replaces: masking and attention of QwenAttention.forward
 *           (src/qwen_int4/model.py:90-122) for packed sequences. */
int64_t qwen2_paged_attention_workspace_bytes(const qwen2_paged_cache* cache, int64_t rows, int64_t heads,
                                              int64_t shared_pages);
int qwen2_paged_attention(const qwen2_paged_cache* cache, const qwen2_rows* q, const qwen2_rows* out, int64_t rows,
                          int64_t heads, int64_t shared_pages, float scale, int zero_rest, void* workspace,
                          int64_t workspace_bytes, void* stream);

/* Which drafted tokens of a speculative step stand, and the token after them:
 *   token i of sequence b stands iff all before it do and
 *       uniforms[b, i] * q_i(x_i) < p_i(x_i),   x_i = draft_tokens[b, i],
 *   n = accepted[b] tokens stand, of the k = draft_lengths[b] (NULL: drafts);
 *   weights w = max(p_n - q_n, 0) for n < k, or p_k: the least v with
 *       sum_{u <= v} w_u > uniforms[b, drafts] * sum w        is token n.
 * p = target [batch, drafts + 1, vocab], q = draft [batch, drafts, vocab] of the
 * same dtype (fp32, bf16 or fp16), or NULL: q_i is 1 at x_i and 0 elsewhere
 * (tokens that no model drew).  Where max(p_n - q_n, 0) is zero everywhere the
 * weights are p_n.  uniforms fp32 [batch, drafts + 1], in [0, 1) (in the sum's
 * place a value outside counts as the nearest one inside, NaN as no choice).  A drafted id outside the
 * vocabulary does not stand, and its q is 0 there.  All in 64 bits, so that a
 * uniform next to a border falls where the definition says, but for roundings of
 * 2^-53 of the sums; what is drawn has weight.
 *   tokens[b, 0 .. n - 1] = the drafts that stand, tokens[b, n] the new token,
 *   -1 behind it; tokens[b, n] = -1 where the weights' sum is zero, infinite or
 *   NaN, or the uniform is NaN.  tokens int64 [batch, drafts + 1], accepted int32 [batch].
 * target's and draft's rows are target_row (draft_row) elements apart, sequences
 * target_batch (draft_batch).  The workspace (8-byte aligned) survives no call.
 * Replaces: the greedy choice of a step (src/qwen_int4/generation.py:51) where
 *           a step proposes several tokens. */
int64_t qwen2_verify_drafts_workspace_bytes(int64_t batch, int64_t drafts, int64_t vocab);
int qwen2_verify_drafts(const void* target, int64_t target_batch, int64_t target_row, const void* draft,
                        int64_t draft_batch, int64_t draft_row, int dtype, const int64_t* draft_tokens,
                        const int32_t* draft_lengths, const float* uniforms, int64_t* tokens, int32_t* accepted,
                        int64_t batch, int64_t drafts, int64_t vocab, void* workspace, int64_t workspace_bytes,
                        void* stream);

/* Causal attention over whole prompts of different lengths, packed:
 *   out[r, h] = softmax_t(scale * q[r, h] . k[t, g]) v[t, g],   t = first row of r's sequence .. r,
 * query head h reading key/value head g = h / (heads / kv_heads); sequence b's rows
 * are cu_rows[b] .. cu_rows[b + 1] - 1 (a device array of batch + 1, not falling, from
 * 0; what it holds is bounded there as the paged operators' is).  q, out [rows, heads,
 * head_dim], k, v [rows, kv_heads, head_dim]: parts of a fused projection are read in
 * place.  Scores, softmax and sums in fp32; a probability is rounded once to dtype
 * before it meets its value, and it is the rounded ones that the sum adds up; the result
 * is rounded once.  Rows of no sequence (behind the last one, or before cu_rows[0]) are
 * left as they are, or zeroed with zero_rest.  Keys and values that a row does not see take no part, whatever they hold;
 * an infinity or NaN among the values that it sees reaches it, however small the key's
 * weight.  (Values are summed before the sum is divided: the keys' number times the
 * values' size has to stay in fp32.)
 * head_dim is 64 or 128; heads a multiple of kv_heads; dtype W4G64_DTYPE_BF16 or
 * W4G64_DTYPE_F16; out must not overlap q, k and v.  No workspace.
 * Replaces: masking and attention of QwenAttention.forward over a prompt
 *           (src/qwen_int4/model.py:90-122) for packed sequences. */
int qwen2_packed_attention(const qwen2_rows* q, const qwen2_rows* k, const qwen2_rows* v, const qwen2_rows* out,
                           const int32_t* cu_rows, int64_t batch, int64_t rows, int64_t heads, int64_t kv_heads,
                           int64_t head_dim, int dtype, float scale, int zero_rest, void* stream);

/* ---------------------------------------------------------------------------
 * The pages of a paged cache: giving them out, forking sequences, compacting.
 *
 * page_users[p] (int32, num_pages) counts what names page p: entries of page
 * tables, and whatever else keeps it (a prefix cached without a sequence).  A page is
 * free where it is 0.  A table's entry names a page where it lies in [0, num_pages);
 * -1 is written where it names none.  Index arrays are device arrays; answers go to
 * arrays of their own, which must share no memory with what is read, so that a step
 * that has to be given up leaves its state whole.  All is bounded on the device: no
 * access leaves the buffers whatever lengths, entries and parents hold.  Whole
 * numbers alone decide, in a fixed order.  batch (and children) at most 2^20, num_pages
 * at most 2^24, batch * table_width below 2^31.  Workspaces (none where few pages and
 * entries are, then NULL may be given) are 4-byte aligned; nothing
 * in one survives a call, and calls that share one must be ordered on one stream.
 * ------------------------------------------------------------------------- */

/* Every row of the table gets the pages that its length needs: entry c of row b,
 * c < ceil(max(lengths[b], 0) / page_size), keeps the page that it names, or is given
 * the lowest free page, row after row and column after column; all others are -1 and
 * their pages given up (a length of 0 frees a sequence).  Pages given up in a call are
 * free from the next one on.
 *   new_table [batch, table_width], new_users[p] = page_users[p] - entries given up
 *   + entries given, missing[b] = pages that row b still lacks (its table's width or
 *   the pool too small; the last columns of the last rows go without first).
 * _cached: cached[b] (NULL: none) positions of row b hold keys and values already.  Of
 * the entries that hold them, c < ceil(cached[b] / page_size), one that names no page is
 * lost: no page is given there, for it would hold what another sequence left in it, but
 * the entry is -1 and counts as missing at every call until the row's length (or cached[b])
 * is brought below it.
 * page_table's rows lie table_stride apart.  page_size: a power of two in [16, 2^20].
 * Replaces: the growth of the cache in QwenAttention.forward (model.py:83-90),
 *           where keys and values lie in pages. */
int64_t qwen2_paged_resize_workspace_bytes(int64_t batch, int64_t table_width, int64_t num_pages);
int qwen2_paged_resize(const int32_t* page_table, int64_t table_stride, const int32_t* lengths, const int32_t* page_users,
                       int32_t* new_table, int32_t* new_users, int32_t* missing, int64_t batch, int64_t table_width,
                       int64_t num_pages, int64_t page_size, void* workspace, int64_t workspace_bytes, void* stream);
int qwen2_paged_resize_cached(const int32_t* page_table, int64_t table_stride, const int32_t* lengths, const int32_t* cached,
                              const int32_t* page_users, int32_t* new_table, int32_t* new_users, int32_t* missing,
                              int64_t batch, int64_t table_width, int64_t num_pages, int64_t page_size, void* workspace,
                              int64_t workspace_bytes, void* stream);

/* Pools of `layers` layers whose pages one table names: the key of page p, position
 * t, head h of layer l is k + l * k_layer + p * k_page + h * k_head + t * k_position, v
 * alike.  Strides in elements of 16 bits, multiples of 8; 16-byte aligned. */
typedef struct qwen2_page_pool {
    void* k;
    void* v;
    int64_t k_layer, k_page, k_head, k_position;
    int64_t v_layer, v_page, v_head, v_position;
    int64_t layers, num_pages, kv_heads;
    int64_t page_size;             /* a power of two in [16, 2^20] */
    int64_t head_dim;              /* a multiple of 8 up to 1024 */
} qwen2_page_pool;

/* The next batch of sequences, made of copies of this one's (samples of one prompt,
 * beams, a batch in another order): row i of the answer is sequence parents[i], or
 * none (length 0) where that is outside [0, batch).  A row holds the pages of its
 * length; full pages are shared, and of a last page that is not full the sequence's first
 * row (the lowest i) keeps the page itself, if page_users is 1 there, and every other one
 * is given the lowest free page, row after row, with the filled positions' keys and
 * values copied to it.  So no row's next position lies in a page that something else
 * names.  Sequences that no row descends from give up their pages, all give up what lies
 * behind their length; those are free from the next call on.
 *   new_table [children, table_width], new_lengths [children],
 *   new_users[p] = page_users[p] - entries of page_table + entries of new_table,
 *   missing[i] = 1 where a copy found no free page (its entry is -1), else 0.  Such a
 * row keeps its length, and what its last page held is lost to it: a resize that is to
 * grow it has to know (qwen2_paged_resize_cached), or would give it a page unwritten.
 * Replaces: nothing of the reference's: its batches decode greedily
 *           (src/qwen_int4/generation.py:10-115). */
int64_t qwen2_paged_fork_workspace_bytes(int64_t batch, int64_t children, int64_t table_width, int64_t num_pages);
int qwen2_paged_fork(const qwen2_page_pool* pool, const int32_t* page_table, int64_t table_stride, const int32_t* lengths,
                     const int32_t* page_users, const int32_t* parents, int32_t* new_table, int32_t* new_lengths,
                     int32_t* new_users, int32_t* missing, int64_t batch, int64_t children, int64_t table_width,
                     void* workspace, int64_t workspace_bytes, void* stream);

/* The n pages in use move to the pool's first n: those behind them, from the lowest
 * on, to the free ones among the first n, from the lowest on.
 *   moved_to[p] = where page p lies now, -1 for a free one; new_table [batch,
 *   table_width]: page_table's entries renamed by it; new_users[moved_to[p]] =
 *   page_users[p], 0 for all others.
 * Pages behind the first n keep what they hold, and may be given back.
 * Replaces: nothing of the reference's (one cache per batch). */
int64_t qwen2_paged_compact_workspace_bytes(int64_t batch, int64_t table_width, int64_t num_pages);
int qwen2_paged_compact(const qwen2_page_pool* pool, const int32_t* page_table, int64_t table_stride,
                        const int32_t* page_users, int32_t* new_table, int32_t* new_users, int32_t* moved_to, int64_t batch,
                        int64_t table_width, void* workspace, int64_t workspace_bytes, void* stream);

/* out[r, i] = silu(gate) * up in fp32, gate = gate_up[r, i], up = gate_up[r, I + i]
 * (bf16 inputs, the fused gate|up projection), silu(x) = x / (1 + exp(-x)).
 * Replaces: the SwiGLU product of QwenMLP.forward (src/qwen_int4/model.py:133-136). */
int qwen2_silu_mul(const void* gate_up, float* out, int64_t rows, int64_t intermediate, void* stream);

/* Bytes of workspace qwen2_lm_head needs for its argmax (one key per row
 * per workgroup; nothing in it survives a call); 0 for unsupported sizes.
 * Calls sharing a workspace must be ordered on one stream. */
int64_t qwen2_lm_head_workspace_bytes(int64_t rows, int64_t vocab, int64_t hidden);

/* Dense bf16 LM head of a decode step, with the greedy choice (a second,
 * one-workgroup-per-row launch on the same stream):
 *   logits[r, v] = bf16( sum_k x[r, k] * weight[v, k] )   (fp32 sums)
 *   argmax[r]    = the smallest v with the largest logits[r, v]
 *                  (NaN counts as the largest; -0 equals +0)
 * for x bf16 [rows, hidden], weight bf16 [vocab, hidden] (Qwen2's tied
 * embedding), logits bf16 [rows, vocab], argmax int64 [rows] or NULL (then
 * no workspace is needed).  rows <= 16, hidden a multiple of 128 and at most
 * 4096; x and weight 16-byte aligned, workspace 8-byte aligned.
 * Replaces: the tied lm_head projection of QwenInt4ForCausalLM
 *           (src/qwen_int4/model.py:217-218, :243-245) and the greedy choice
 *           logits[:, -1].argmax(dim=-1) (src/qwen_int4/generation.py:51). */
int qwen2_lm_head(const void* x, const void* weight, void* logits, int64_t* argmax, int64_t rows, int64_t vocab,
                  int64_t hidden, void* workspace, int64_t workspace_bytes, void* stream);

/* The greedy choice alone, over logits bf16 [rows, vocab] of any head:
 * argmax[r] as qwen2_lm_head's.  rows <= 65535; argmax and workspace 8-byte
 * aligned.  Bytes of workspace: one key per row and 4096 logits, 0 for
 * unsupported sizes; calls sharing it must be ordered on one stream.
 * Replaces: logits[:, -1].argmax(dim=-1) (src/qwen_int4/generation.py:51)
 *           past qwen2_lm_head's 16 rows. */
int64_t qwen2_argmax_workspace_bytes(int64_t rows, int64_t vocab);
int qwen2_argmax(const void* logits, int64_t* argmax, int64_t rows, int64_t vocab, void* workspace,
                 int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* QWEN_INT4_HIP_QWEN2_DECODE_H */
