// Argument blocks of the kernels in cache_kernels.hip, shared with the host
// code that fills them (cache_shim.cpp).
#ifndef QWEN3_CACHE_ARGS_H
#define QWEN3_CACHE_ARGS_H

#include <stdint.h>

constexpr int kTreeMax = 256;  // nodes of a tree, rows of a call

struct AttnTreeArgs {
  const uint16_t *k, *v;  // the layer's base, [max_seq, kv_heads, head_dim]
  const uint16_t* q;
  const uint32_t* mask;  // [n, mask_words] or null: rows see the rows before them
  uint16_t* out;
  float* lse;  // or null
  int64_t q_stride, out_stride;
  float* part;     // [splits, kv_heads, rows, head_dim] outputs of the splits
  float* part_ml;  // [kv_heads, rows, 2, splits] their references and sums
  int32_t len, n, q_heads, kv_heads, group;
  uint32_t group_inv;      // ceil(2^32 / group): r / group for group > 1, r < 2^13
  int32_t splits, blocks;  // blocks of 32 slots in a split
  float scale;                         // with log2 e: scores in base-2 units
};

struct WeightsArgs {
  const uint16_t* k;
  float* weights;
  const uint16_t* q;
  const float* lse;
  const int32_t* path;  // or null
  int64_t max_seq, q_layer_stride, q_stride, lse_layer_stride;
  int32_t kv_heads, q_heads, group, len, n, rows;
  uint32_t group_inv;  // as in AttnTreeArgs
  int32_t blocks;      // blocks of 32 slots a wave takes
  float scale;         // with log2 e
};

struct SelectArgs {
  const float* weights;
  int32_t* keep;
  int64_t max_seq;
  int32_t len, budget, sinks, recent;
};

struct CompactArgs {
  const uint16_t *k, *v;
  const float* w;  // or null
  uint16_t *k_to, *v_to;
  float* w_to;
  const int32_t* keep;
  int64_t src_seq, dst_seq;
  int32_t kv_heads, head_dim, per_head, base, count;
  int32_t range;  // kept slots of one workgroup
  int32_t in_place;  // source and destination are one
};

struct GemmArgmaxArgs {
  const uint16_t *w, *x;  // [rows, 1024], [n, 1024]
  uint16_t* logits;       // [n, rows] or null
  uint64_t* part;         // [n, workgroups] argmax keys
  int32_t rows, n;
  int32_t whole8;         // every row of logits starts on 8 bytes
};

#endif
