/*
 * Serving several sequences from one paged KV cache, in f16 or 8 bits: new rows
 * appended with their heads' norm and rotation, attention over the pages, pages
 * read back, and drafted tokens verified against the model's probabilities.
 * Implemented by libq8gemv.so (kernels in the code object pages_gfx950.hsaco,
 * loaded by q8gemv_init).  No counterpart in the reference, which runs one
 * sequence over a flat f16 cache (model/qwen3_full.mlir:213-230, 1431-1526).
 *
 * A step runs some new rows of every sequence: one token, a chain of drafted
 * ones, or a chunk of a prompt.  In every layer kv_pages_append writes their k
 * and v into the pages and kv_pages_attn attends to them; behind f16_gemm_argmax
 * (f16_cache.h) kv_verify says which drafted tokens stand and samples the next.
 * qwen3_pages_step (qwen3_decode.h) runs a whole model this way.
 *
 * Conventions as in q8gemv.h: device pointers owned by the caller, status
 * codes, nothing allocates, arguments validated before anything is enqueued,
 * work only enqueued on `stream`, safe under graph capture.  Values that are
 * read from device memory (page tables, lengths, row starts, tokens) cannot be
 * refused on the host; each call says what an entry outside its range does, and
 * none makes a kernel read or write outside the buffers.
 */
#ifndef QWEN3_KV_PAGES_H
#define QWEN3_KV_PAGES_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define KV_PAGES_F16 0
#define KV_PAGES_Q8 1
#define KV_PAGES_MAX_SEQS 1024

/* A pool of pages.  Page p of layer l holds, for every kv head, page_size rows of
 * head_dim values of k (and of v): k and v are [layers, pages, kv_heads,
 * page_size, head_dim], of f16 (KV_PAGES_F16) or int8 codes (KV_PAGES_Q8).  A code
 * stands for itself times its row's scale: k_scale and v_scale f32 [layers,
 * pages, kv_heads, page_size] (NULL with f16 pages).  pages in [1, 2^24],
 * layers in [1, 1024], kv_heads in [1, 256], head_dim 64 or 128; page_size a
 * multiple of 16 up to 4096; all pointers 16-byte aligned.  The struct is read
 * by the host during the call only. */
typedef struct kv_pages {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t pages;
  int32_t layers, page_size, kv_heads, head_dim, type;
} kv_pages;

/* The sequences of a call and their new rows.  Slot p of sequence s is entry
 * p % page_size of page table[s * table_stride + p / page_size]; length[s] of its
 * slots are in use, its new rows among them.  Its new rows are rows start[s] ..
 * start[s + 1] - 1 of the call's row arrays, m of them, and row start[s] + i sits
 * in slot length[s] - m + i.  start NULL: one row each, row s (rows = seqs).
 * table: device int32 [seqs, max_pages] with table_stride >= max_pages, length:
 * device int32 [seqs], start: device int32 [seqs + 1], all 4-byte aligned.
 * seqs in [1, 1024], rows in [1, 2^23] (what the row arrays hold), max_rows in
 * [1, 2^23] the most rows of a sequence, max_pages >= 1 with max_pages *
 * page_size <= 2^24.
 * The starts do not descend (where they do it is open which rows are run).
 * A sequence whose rows are not 0 <= start[s] <= start[s + 1] <= rows or more
 * than max_rows is left out; so are rows that belong to no sequence (behind
 * start[seqs]).  What is left out has no effect and its outputs are not written.  A table entry outside
 * [0, pages) and a slot outside [0, max_pages * page_size) stand for nothing: such a
 * slot is not written, reads as zeros and is not attended to. */
typedef struct kv_batch {
  const int32_t* table;
  const int32_t* length;
  const int32_t* start;
  int64_t table_stride;
  int32_t seqs, max_pages, rows, max_rows;
} kv_batch;

/* The projections of new rows.  q, k, v: f16, row r of q at q + r q_stride
 * elements, its heads contiguous (so all three may lie in one product), strides
 * multiples of 8 and at least the heads' width, pointers 16-byte aligned.
 * q NULL: no queries (q_heads 0).  q_norm, k_norm: f16 [head_dim] weights of the
 * heads' norm, 2-byte aligned, NULL: no norm.  eps >= 0 finite; theta 0: no
 * rotation, else finite and > 0.  positions: device int32 [rows], NULL: a row's
 * slot.  q_out: as q, may be q itself with its stride; must not overlap k or v. */
typedef struct kv_rows {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  const void* q_norm;
  const void* k_norm;
  const int32_t* positions;
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  double eps, theta;
  int32_t q_heads;
} kv_rows;

/* Writes the batch's rows of one layer into the pages, and their queries to q_out:
 *   y = x / sqrt(mean x^2 + eps) w            over each head of q and k
 *   (y[i], y[i + D/2]) turned by position theta^(-2i/D), i < D/2
 * q rounded to f16; k and v to the pages' type, v as it stands.  8-bit rows, one
 * of each head: scale = f32(max |y| / 127), codes round(y / scale) to the
 * nearest, ties to even, at most 127 in magnitude; all zeros: scale and codes 0; a
 * row with an infinity or NaN: scale NaN, so that it reads as NaN.
 * k is computed in 64 bits up to its rounding (a sum in another order must
 * not move a value over a code's border), f16 values rounded to f32 first; q in 32 but
 * for its angles, off by at most 2^-20 of |y[i]| + |y[i + D/2]| before it is rounded.
 * The table may name a page twice only where no slot is written through both. */
int kv_pages_append(const kv_pages* pages, int32_t layer, const kv_batch* batch,
                    const kv_rows* rows, void* stream);

/* Attention of the batch's rows in one layer, each over its sequence's slots up to
 * its own (the k and v of which are in the pages already):
 *   s[r,h,j] = scale q[r,h] . k[j, h / (q_heads / kv_heads)]
 *   out[r,h] = sum_j softmax_j(s[r,h]) v[j, ...],  lse[r,h] = log sum_j exp s[r,h,j]
 * A row that sees no slot, or only scores of -inf, is empty: out 0, lse -inf.  What
 * slots hold that a row does not see is never used, NaN and infinities included;
 * a value of out whose v holds an infinity or NaN in a slot the row sees is not
 * finite.  q, out: f16 rows as in kv_rows; lse: f32 [rows, q_heads], may be NULL.
 * out must not overlap q (workgroups that share a row read q while others
 * write).  q_heads a multiple of kv_heads, at most 32 times it and at most 256; scale
 * positive and below 2^118; max_rows at most 256.  Scores, statistics and sums are
 * f32; a weight (with v's scale) enters its product with v to 2^-22 of itself or 2^-31 of the
 * row's largest, whichever is more, so that N slots add at most N 2^-31 of the largest
 * weight times the largest |v| to the error of a value of out.
 * workspace: device memory of kv_pages_attn_workspace_bytes (256-byte aligned);
 * fill it with zeros once before its first use.  Its first 64 KiB are counters, zeros again
 * behind every call, that nothing else may write; the rest is needed only during the call.
 * The size depends on the heads and on max_rows alone, and that of the largest
 * max_rows of a session serves all its calls.  Calls that may overlap (streams,
 * graphs) need one each. */
size_t kv_pages_attn_workspace_bytes(const kv_pages* pages, const kv_batch* batch,
                                     int32_t q_heads);
int kv_pages_attn(const kv_pages* pages, int32_t layer, const kv_batch* batch, const void* q,
                  int64_t q_stride, int32_t q_heads, float scale, void* out, int64_t out_stride,
                  float* lse, void* workspace, size_t workspace_bytes, void* stream);

/* The batch's rows read back, out of layers layer .. layer + layers - 1: row r of
 * layer layer + l to k_out (and v_out) + l layer_stride + r row_stride elements,
 * f16 [kv_heads, head_dim] each; 8-bit values as f16(f32(code * scale)).  With
 * start = the running sums of the lengths whole sequences are read, with
 * row_stride = kv_heads * head_dim and layer_stride = max_seq * row_stride into the flat
 * cache of f16_cache.h.  Strides multiples of 8, row_stride at least kv_heads *
 * head_dim, and so layer_stride, which is ignored with one layer; rows do not overlap.  k_out or v_out may be NULL. */
int kv_pages_read(const kv_pages* pages, int32_t layer, int32_t layers, const kv_batch* batch,
                  void* k_out, void* v_out, int64_t row_stride, int64_t layer_stride,
                  void* stream);

/* Drafted tokens against the model's probabilities, from given random numbers.
 * Rows as in kv_batch: sequence s ran rows start[s] .. start[s + 1] - 1 (start
 * NULL: row s), tokens[r] (device int32 [rows]) being row r's own token: of its m
 * rows the first carries the last token known, the other m - 1 drafted ones.
 * logits: f16, row r at logits + r logits_stride, [vocab]: what follows row r.
 *   p[r,j] = exp(logits[r,j] / T) / sum        T = temperature[s] (f32 [seqs],
 *            NULL: 1); T <= 0 or NaN: 1 at the lowest index of the maximum, 0 else
 *   q[r,j] the drafter's probabilities of what follows row r, f32 [vocab] at draft + r
 *            draft_stride (those of a sequence's last row are not read); entries
 *            that are not > 0 count as 0.  draft NULL: 1 at the drafted token, 0 else
 * The token x = tokens[r + 1] drafted behind row r is accepted if uniform[r] q[r,x] <
 * p[r,x], as long as all before it were.  Behind the n accepted ones one more is
 * taken: j is the lowest index with c[j] > uniform[last row] c[vocab - 1], c the running
 * sums of w[j] = max(p[r,j] - q[r,j], 0) in the row r that refused, of p[r,j]
 * where that is zero throughout or no token was refused (the last index with w > 0
 * where no sum is larger).
 * out (device int32 [seqs, out_stride]): the accepted tokens, then that one, -1
 * up to max_rows entries; accepted (int32 [seqs]): n; logprob (f32 [seqs,
 * out_stride], may be NULL): log p of each token under its row, 0 behind them.
 * A NaN logit counts as -inf; where the maximum is +inf all such share the
 * probability; a row of -inf alone has p = 0, accepts nothing and gives token -1
 * (logprob 0).  A drafted token outside [0, vocab) is refused (draft NULL: w = p).
 * A sequence without rows, or left out as in kv_batch, gives accepted 0 and -1s.
 * uniform: f32 [rows], values in [0, 1).  Everything but the logprobs' last
 * rounding is computed in 64 bits and fixed order; a p[r,j] below 2^-990 of the row's
 * largest may count as 0.
 * rows in [1, 65535], seqs in [1, 1024], max_rows in [1, 256], out_stride >=
 * max_rows, vocab in [1, 2^24]; strides >= vocab; logits 2-byte, the others
 * 4-byte aligned.  workspace: kv_verify_workspace_bytes (256-byte aligned); fill it
 * with zeros once before its first use.  Its first 256 KiB are counters, zeros again behind every
 * call, that nothing else may write; the rest is needed only during the call.  That of the
 * largest rows, seqs and vocab of a session serves all its calls; calls that may
 * overlap need one each. */
typedef struct kv_drafts {
  const void* logits;
  const int32_t* tokens;
  const int32_t* start;
  const float* temperature;
  const float* draft;
  const float* uniform;
  int32_t* out;
  int32_t* accepted;
  float* logprob;
  int64_t logits_stride, draft_stride, out_stride;
  int32_t vocab, rows, seqs, max_rows;
} kv_drafts;

size_t kv_verify_workspace_bytes(int32_t rows, int32_t seqs, int32_t vocab);
int kv_verify(const kv_drafts* drafts, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
