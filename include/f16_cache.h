/*
 * Operators over an f16 KV cache for drafted tokens and for caches that run
 * full, and the vocabulary product over several token rows.  Implemented by
 * libq8gemv.so (kernels in the code object cache_gfx950.hsaco, loaded by
 * q8gemv_init).  No counterpart in the reference, which runs one token at a
 * time over a cache that only grows (model/qwen3_full.mlir:1431-1526).
 *
 * A program drafts a tree of tokens, runs all its nodes through the model at
 * once (f16_attn_tree in every layer, f16_gemm_argmax behind the last), moves
 * the k and v of the path the model agrees with to the front (f16_cache_compact)
 * and adds up the attention every cached position got (f16_attn_weights_add).
 * When the cache is full, f16_cache_select picks the positions worth keeping by
 * those sums and f16_cache_compact moves them together.  qwen3_tree_step and
 * its companions (qwen3_decode.h) run a whole model this way.
 *
 * Conventions as in q8gemv.h: device pointers owned by the caller, status
 * codes, nothing allocates, arguments validated before anything is enqueued,
 * work only enqueued on `stream`, safe under graph capture.  Values that are
 * read from device memory (parents, masks, paths, kept positions) cannot be
 * refused on the host; each call says what an entry outside its range does,
 * and none makes a kernel read or write outside the buffers.
 */
#ifndef QWEN3_F16_CACHE_H
#define QWEN3_F16_CACHE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define F16_TREE_MAX_NODES 256  /* nodes of a tree, rows of one call */
#define F16_MAX_GROUP 32        /* query heads that share a kv head */

/* A KV cache of one sequence in the flat layout of qwen3_decode.h: k and v are
 * f16 [layers * max_seq, kv_heads, head_dim], the entry of layer l, slot p in
 * row l * max_seq + p.  `weights` (may be NULL where a call does not need it)
 * is f32 [layers, kv_heads, max_seq]: the attention each slot got.
 * max_seq in [1, 2^24], layers in [1, 1024], kv_heads in [1, 256], head_dim 64
 * or 128; k and v 16-byte, weights 4-byte aligned.  A single layer is a cache
 * with layers = 1 at that layer's address.  The struct is read by the host
 * during the call only. */
typedef struct f16_cache {
  void* k;
  void* v;
  float* weights;
  int64_t max_seq;
  int32_t layers, kv_heads, head_dim;
} f16_cache;

/* The masks of a tree of n nodes in [1, 256] given by its parents (device
 * int32 [n]; every parent before its children): parents[i] in [0, i) is the
 * node before i, -1 puts i right behind the cache.  Any other value marks i as
 * padding, and so does an ancestor that is padding.
 * mask: device u32 [n, ceil(n / 32)], bit j % 32 of word j / 32 of row i set
 * where j is i or an ancestor of i; a padding row has no bit.  depth (may be
 * NULL): device int32 [n], the ancestors of i, so that i sits depth[i]
 * positions behind the first; -1 for padding. */
int f16_tree_mask(const int32_t* parents, int32_t n, uint32_t* mask, int32_t* depth, void* stream);

/* Attention of n rows (nodes of a drafted tree, or a chunk of tokens) in one
 * layer of a cache whose slots 0 .. len - 1 hold the sequence so far and whose
 * slots len .. len + n - 1 hold the k and v of the n rows:
 *   s[i,h,j] = scale q[i,h] . k[j, h / (q_heads / kv_heads)]
 *   out[i,h] = sum_j softmax_j(s[i,h]) v[j, ...],  lse[i,h] = log sum_j exp s[i,h,j]
 * over j < len and the slots len + a with bit a of row i of `mask` set (as
 * f16_tree_mask writes it; any bits are allowed, those from n on are ignored).
 * mask NULL: row i sees rows 0 .. i (a chunk of consecutive tokens).  A row
 * without a bit below n is empty: out 0, lse -inf, whatever its q holds.  What
 * masked slots and slots from len + n on hold is never used, NaN and infinities
 * included.
 * q: f16, row i at q + i q_stride elements, q_heads x head_dim contiguous;
 * out: the same with out_stride; lse: f32 [n, q_heads], may be NULL.
 * q_heads a multiple of kv_heads, at most 32 times it and at most 256; strides
 * multiples of 8 elements and at least q_heads * head_dim; q and out 16-byte,
 * mask and lse 4-byte aligned; n in [1, 256], len >= 0, len + n <= max_seq;
 * scale finite and positive.  Scores, statistics and sums are f32; a weight enters
 * its product with v to 2^-22 of itself.
 * workspace: device memory of f16_attn_tree_workspace_bytes (256-byte aligned;
 * may be NULL where that is 0), needed only during the call, nothing to
 * initialise.  The size does not shrink as len or n grows and covers every call of
 * fewer rows over as many slots (len + n), so that of max_seq - n and n serves all
 * calls of up to n rows of a session.  Calls that may overlap need one each. */
size_t f16_attn_tree_workspace_bytes(const f16_cache* cache, int32_t len, int32_t n,
                                     int32_t q_heads);
int f16_attn_tree(const f16_cache* cache, int32_t layer, int32_t len, const void* q,
                  int64_t q_stride, int32_t q_heads, const uint32_t* mask, int32_t n, float scale,
                  void* out, int64_t out_stride, float* lse, void* workspace,
                  size_t workspace_bytes, void* stream);

/* The attention that n tokens at slots len .. len + n - 1 paid to every slot,
 * added to cache->weights in all layers at once.  Token i is row r = path[i]
 * (device int32 [n]; NULL: r = i) of q and lse, which are kept from
 * f16_attn_tree: q f16 [layers, rows, q_heads x head_dim] with strides
 * q_layer_stride and q_stride (elements), lse f32 [layers, rows, q_heads] with
 * stride lse_layer_stride.  For slots j < len
 *   weights[l,h',j] += sum_i sum_{h of h'} exp(scale q[l,r,h] . k[l,j,h'] - lse[l,r,h])
 * and for the new slots j = len .. len + n - 1, which token i sees from
 * i >= j - len on, the sum replaces what was there.  A path entry outside
 * [0, rows) and a row with lse -inf add nothing.  Other slots stay as they are.
 * Every sum is f32 in a fixed order.  n in [1, 256], rows in [1, 2^20],
 * q_layer_stride a multiple of 8 (ignored with one layer); the rest as in
 * f16_attn_tree. */
int f16_attn_weights_add(const f16_cache* cache, int32_t len, const void* q,
                         int64_t q_layer_stride, int64_t q_stride, int32_t q_heads,
                         const float* lse, int64_t lse_layer_stride, int32_t rows,
                         const int32_t* path, int32_t n, float scale, void* stream);

/* The slots to keep of len >= budget, in every layer and kv head: the first
 * `sinks`, the last `recent`, and of those between the budget - sinks - recent
 * with the largest weights (equal weights: the lower slot first; -0 equals 0,
 * NaN counts below every number).  keep: device int32 [layers, kv_heads,
 * budget], ascending.  1 <= budget <= len <= max_seq, sinks, recent >= 0,
 * sinks + recent <= budget. */
int f16_cache_select(const f16_cache* cache, int32_t len, int32_t budget, int32_t sinks,
                     int32_t recent, int32_t* keep, void* stream);

/* Slot base + j of dst becomes slot base + keep[j] of src, j = 0 .. count - 1,
 * in every layer and kv head: k, v and, where both caches have them, weights.
 * keep: device int32, with per_head != 0 [layers, kv_heads, count] (as
 * f16_cache_select writes it, base 0), else [count] for all (an accepted path
 * of a tree, base = len).  An entry outside [0, src max_seq - base) leaves its
 * destination slot as it was, and so stays every slot outside base .. base +
 * count - 1.  dst may be src (or share all of its buffers with the same
 * max_seq): then keep must be strictly ascending, or the values moved are
 * unspecified.  Otherwise the buffers must not overlap, keep may have any
 * order, and max_seq may differ (a move into a smaller cache).  The two caches
 * agree in layers, kv_heads and head_dim; base >= 0, count >= 0, base + count
 * <= both max_seq.  count = 0 does nothing. */
int f16_cache_compact(const f16_cache* src, const f16_cache* dst, const int32_t* keep,
                      int per_head, int32_t base, int32_t count, void* stream);

/* f16_gemv_argmax_rows (q8gemv.h) for n token rows: logits[i] = f16(W x[i]) and
 * tokens[i] = the lowest index of the maximal f16 logit of row i (-1 if none is
 * > -inf; NaN never wins).  W f16 [w_rows, 1024], w_rows in [1, 2^31); x f16
 * [n, 1024], n in [1, 256]; logits f16 [n, w_rows], NULL to skip writing them;
 * tokens device int32 [n].  W, x and workspace 16-byte, logits 2-byte, tokens
 * 4-byte aligned.  workspace: f16_gemm_argmax_workspace_bytes(n) bytes, needed
 * only during the call, nothing to initialise; calls that may overlap need one
 * each. */
size_t f16_gemm_argmax_workspace_bytes(int32_t n);
int f16_gemm_argmax(const void* w_f16, int64_t w_rows, const void* x_f16, int32_t n,
                    void* logits_f16, int32_t* tokens, void* workspace, void* stream);

#ifdef __cplusplus
}
#endif
#endif
