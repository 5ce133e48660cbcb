// Argument blocks of the kernels in pages_kernels.hip, shared with the host
// code that fills them (pages_shim.cpp), and the index arithmetic both sides and the
// CPU tests use.
#ifndef QWEN3_PAGES_ARGS_H
#define QWEN3_PAGES_ARGS_H

#include <stdint.h>

#if defined(__HIP_DEVICE_COMPILE__) || defined(__HIPCC__)
#define PAGES_FN __host__ __device__ __forceinline__
#else
#define PAGES_FN inline
#endif

// A call's sequences, and where the pages of one layer are.
struct PagesBatch {
  const int32_t *table, *length, *start;  // start may be null
  int64_t table_stride;
  int32_t seqs, rows, max_rows;
  int32_t pages, page_size, slots;  // slots: max_pages * page_size
  int32_t tiles;                    // page_size / 16
  uint32_t tiles_inv;               // ceil(2^32 / tiles), 0 for one
};

// floor(tile / tiles) for tile < 2^20 and tiles <= 2^8: the error of the rounded
// inverse, under tiles / 2^32 of tile, stays below one part in tiles.
PAGES_FN int32_t page_of_tile(const PagesBatch& b, int32_t tile) {
  return b.tiles_inv ? (int32_t)(((uint64_t)(uint32_t)tile * b.tiles_inv) >> 32) : tile;
}

// The rows [lo, lo + m) of sequence s given by its two starts; m = 0 where it is
// left out.
PAGES_FN int32_t rows_of(const PagesBatch& b, int32_t lo, int32_t hi) {
  return lo >= 0 && hi >= lo && hi <= b.rows && hi - lo <= b.max_rows ? hi - lo : 0;
}

// Whether slot p of a sequence is one, and its page's place in the pool is too.
PAGES_FN bool slot_ok(const PagesBatch& b, int64_t p) { return p >= 0 && p < b.slots; }
PAGES_FN bool page_ok(const PagesBatch& b, int32_t page) { return page >= 0 && page < b.pages; }

// The slots that row i of a sequence's m rows sees: those before its own and its own.
PAGES_FN int32_t slots_seen(const PagesBatch& b, int32_t length, int32_t m, int32_t i) {
  const int64_t n = (int64_t)length - m + 1 + i;
  return n <= 0 ? 0 : n < b.slots ? (int32_t)n : b.slots;
}

struct PagesAppendArgs {
  PagesBatch b;
  const uint16_t *q, *k, *v;  // q may be null
  uint16_t* q_out;
  const uint16_t *q_norm, *k_norm;  // or null
  const int32_t* positions;         // or null
  int64_t q_stride, k_stride, v_stride, q_out_stride;
  void *k_to, *v_to;  // the layer's pages
  float *k_scale, *v_scale;
  double eps;
  int32_t q_heads, kv_heads, rotate;
  double turns[64];  // theta^(-2i/D) / 2 pi
};

struct PagesAttnArgs {
  PagesBatch b;
  const void *k, *v;  // the layer's pages
  const float *k_scale, *v_scale;
  const uint16_t* q;
  uint16_t* out;
  float* lse;  // or null
  int64_t q_stride, out_stride;
  int32_t q_heads, kv_heads, group;
  uint32_t group_inv;  // ceil(2^32 / group): r / group for group > 1, r < 2^13
  uint32_t scale_bits; // f32: with log2 e, and with the unit of codes in the products
  int32_t workers;     // workgroups of a kv head and row block
  int32_t* count;      // [row blocks, kv heads, workers] parts that have arrived
  float* part;         // [row blocks, kv heads, workers, 2, rows, head_dim]
  float* part_ml;      // the same with 2: their references and sums
};

struct PagesReadArgs {
  PagesBatch b;
  const void *k, *v;
  const float *k_scale, *v_scale;
  uint16_t *k_out, *v_out;  // or null
  int64_t row_stride, layer_stride;
  int32_t kv_heads;
};

constexpr int kSeqsMax = 1024;
// Counters lie this many words apart: those of one cache line take their turns, 4 ns each.
constexpr int kCountStep = 32;
// A row's maximum, its lowest index, and the sum of exp((x - top) / T).
struct VerifyStat {
  double sum;
  float top;
  int32_t first;
};

// What decides a sequence's last token: its row, 256 log2(e) / T and T, the accepted
// tokens, the random number, and the token that was refused.
struct VerifyPick {
  VerifyStat row;
  double unit;
  float heat, u;
  int32_t n, told;
};

struct VerifyArgs {
  PagesBatch b;  // start, seqs, rows, max_rows
  const uint16_t* logits;
  const int32_t* tokens;
  const float *temperature, *draft, *uniform;
  int32_t *out, *accepted;
  float* logprob;
  int64_t logits_stride, draft_stride, out_stride;
  int32_t vocab, chunks, parts;  // chunks of a row in the first launch, parts in the second
  int32_t* count;     // [2, kSeqsMax, kCountStep] workgroups of a sequence that have come to a launch's end
  VerifyPick* picks;  // [seqs]
  double* sums;       // [rows, chunks] of exp((x - top) / T)
  double* tops;       // [rows, chunks] the maximum and its lowest index
  double* rest;       // [seqs, parts, 2] sums of max(p - q, 0) and of p in the deciding row
};

#endif
