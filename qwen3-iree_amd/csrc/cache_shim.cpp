// Host side of include/f16_cache.h: argument checks and launches of the
// kernels in cache_kernels.hip.
#include "f16_cache.h"
#include "cache_args.h"
#include "q8gemv.h"
#include "shim_internal.h"

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

namespace {

struct {
  hipModule_t module = nullptr;
  hipFunction_t mask = nullptr, rope = nullptr, attn[2][4] = {}, merge[2] = {};
  hipFunction_t weights[2][5] = {}, select[4] = {}, compact = nullptr;
  hipFunction_t argmax[3] = {}, argmax_final = nullptr;
} c;

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return q8_shim::error(code, buf);
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

int check_ready() {
  int rc = q8_shim::ready();
  if (rc) return rc;
  if (!c.module)
    return fail(Q8_ERR_CODE_OBJECT, "cache_gfx950.hsaco was not found or lacks a kernel");
  return Q8_OK;
}

int check_cache(const f16_cache* a, const char* name) {
  if (!a) return fail(Q8_ERR_NULL_POINTER, "null %s", name);
  if (a->max_seq < 1 || a->max_seq > (1LL << 24))
    return fail(Q8_ERR_BAD_SHAPE, "%s: max_seq %lld outside [1, 2^24]", name, (long long)a->max_seq);
  if (a->layers < 1 || a->layers > 1024)
    return fail(Q8_ERR_BAD_SHAPE, "%s: %d layers outside [1, 1024]", name, a->layers);
  if (a->kv_heads < 1 || a->kv_heads > 256)
    return fail(Q8_ERR_BAD_SHAPE, "%s: %d kv heads outside [1, 256]", name, a->kv_heads);
  if (a->head_dim != 64 && a->head_dim != 128)
    return fail(Q8_ERR_BAD_SHAPE, "%s: head_dim %d is not 64 or 128", name, a->head_dim);
  if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->weights, 4))
    return fail(Q8_ERR_MISALIGNED, "%s: k and v 16, weights 4-byte alignment", name);
  return Q8_OK;
}

// rows of query heads over a cache: what attention and its weights share
int check_rows(const f16_cache* a, int32_t len, int32_t n, int32_t q_heads, int64_t q_stride,
               float scale) {
  if (q_heads < 1 || q_heads > 256 || q_heads % a->kv_heads ||
      q_heads / a->kv_heads > F16_MAX_GROUP)
    return fail(Q8_ERR_BAD_SHAPE, "%d query heads over %d kv heads", q_heads, a->kv_heads);
  if (n < 1 || n > F16_TREE_MAX_NODES)
    return fail(Q8_ERR_BAD_SHAPE, "n %d outside [1, %d]", n, F16_TREE_MAX_NODES);
  if (len < 0 || (int64_t)len + n > a->max_seq)
    return fail(Q8_ERR_BAD_SHAPE, "slots [%d, %d + %d) outside the cache of %lld", len, len, n,
                (long long)a->max_seq);
  if (q_stride % 8 || q_stride < (int64_t)q_heads * a->head_dim)
    return fail(Q8_ERR_BAD_SHAPE, "row stride %lld is no multiple of 8 of at least %d",
                (long long)q_stride, q_heads * a->head_dim);
  if (!(scale > 0.0f) || !std::isfinite(scale))
    return fail(Q8_ERR_BAD_ARGUMENT, "scale %g is not finite and positive", scale);
  return Q8_OK;
}

constexpr float kLog2e = 1.44269504088896341f;

// ceil(2^32 / group), for the kernels' division of a row by it
uint32_t group_inverse(int group) { return (uint32_t)((0xffffffffull + group) / group); }

// How f16_attn_tree divides its work.
struct AttnPlan {
  int kernel;  // rows of a workgroup: 16, 32, 64, 128; position groups 4, 2, 1, 1
  int row_blocks, splits, blocks;
  int splits_max;  // before the blocks are dealt out evenly; does not shrink with len
};

constexpr int kMaxSplits = 64;  // one lane each in the merge

// Rows of a workgroup: a wave's one tile of 16 up to 64 rows, and above them too
// (several row blocks, whose K and V come out of L2) until every CU has 65 blocks of
// 64 rows and 32 slots to do; then two tiles a wave.  us a layer (16 query over 8 kv
// heads of 128), one and two tiles: 61 nodes, 1024 slots 12.4 / 15.0, 8191 22.8 / 23.8;
// 128, 2048 16.8 / 20.7, 16384 43.7 / 47.7, 30000 71.6 / 67.2; 256, 300 18.6 / 22.3,
// 6000 39.5 / 43.0, 8191 47.6 / 44.0, 16384 73.7 / 69.8.
//
// Splits of the nb blocks of 32 slots: each costs a partial written and merged,
// the first one a launch, and each block of a split costs a round of its
// workgroups, so about sqrt(nb) of them (somewhat more where waves share a block),
// and none up to 10 blocks.  With 1 / 4 / 8 / 16 / 32 splits:
//   1 node, 300 slots (10 blocks) 6.8 / 7.8 / 8.1, 1000 (32) 10.7 / 9.0 / 8.4 / 8.7
//   / 9.2, 4000 (126) 46.2 / 18.8 / 13.4 / 11.0 / 10.8, 16384 (513) 104 / 36.2 / 23.7
//   / 20.5 / 20.5 (64: 24.2); 30 nodes, 1024 (33) 20.4 / 11.9 / 10.5 / 11.0 / 11.3; 13
//   nodes, 8191 (257) 138 / 44.3 / 27.3 / 20.1 / 16.8.
// At most one workgroup a CU where it takes the CU's LDS (up to 16 rows), else two;
// above 64 rows as many as fill every CU once, or twice where that leaves each split
// 8 blocks: 256 nodes, 1024 slots (5 blocks at two) 22.0 at one and 24.9 at two; 128,
// 2048 16.9 and 19.2; 4000 slots and 256 nodes (17 blocks) 36.5 and 34.1; 8191 and 61
// (8) 22.7 and 22.9.
AttnPlan attn_plan(const f16_cache* a, int32_t len, int32_t n, int32_t q_heads) {
  const int rows = n * (q_heads / a->kv_heads), cus = q8_shim::compute_units();
  const int nb = (len + n + 31) / 32;
  const int64_t work = (int64_t)((rows + 63) / 64) * a->kv_heads * nb;
  AttnPlan p{};
  p.kernel = rows <= 16 ? 0 : rows <= 32 ? 1 : rows <= 64 || work < 65 * cus ? 2 : 3;
  const int per_wg = 16 << p.kernel;
  p.row_blocks = (rows + per_wg - 1) / per_wg;
  const int root = (int)((p.kernel > 0 && rows <= 64 ? 1.5 : 1.25) * std::sqrt((double)nb));
  const int one = std::max(1, cus / (a->kv_heads * p.row_blocks));
  const int two = std::max(1, 2 * cus / (a->kv_heads * p.row_blocks));
  const int most = p.kernel == 0 || rows > 64 ? one : two;
  if (nb <= 10) p.splits_max = 1;
  else if (rows > 64 && nb >= 8 * two) p.splits_max = std::min(two, kMaxSplits);
  else p.splits_max = std::min({root, most, kMaxSplits});
  p.blocks = (nb + p.splits_max - 1) / p.splits_max;
  p.splits = (nb + p.blocks - 1) / p.blocks;
  return p;
}

// partial outputs, then their references and sums
size_t attn_part_floats(const f16_cache* a, int32_t n, int32_t q_heads, int splits) {
  return (size_t)splits * n * q_heads * a->head_dim;
}

// What one call needs.  It may be less for more rows: a further row block means fewer
// splits.
size_t attn_workspace(const f16_cache* a, const AttnPlan& p, int32_t n, int32_t q_heads) {
  if (p.splits_max == 1) return 0;
  return 4 * (attn_part_floats(a, n, q_heads, p.splits_max) + 2 * (size_t)n * q_heads * p.splits_max);
}

constexpr int kArgmaxWgsMax = 512;  // keys a token has in the workspace

}  // namespace

namespace q8_shim {

void cache_load(const char* path) {
  hipModule_t m = nullptr;
  if (hipModuleLoad(&m, path) != hipSuccess) return;
  struct {
    hipFunction_t* fn;
    const char* name;
  } names[] = {{&c.mask, "tree_mask_k"},
               {&c.rope, "tree_rope_k"},
               {&c.attn[0][0], "attn_tree_64_11"},
               {&c.attn[0][1], "attn_tree_64_21"},
               {&c.attn[0][2], "attn_tree_64_41"},
               {&c.attn[0][3], "attn_tree_64_42"},
               {&c.attn[1][0], "attn_tree_128_11"},
               {&c.attn[1][1], "attn_tree_128_21"},
               {&c.attn[1][2], "attn_tree_128_41"},
               {&c.attn[1][3], "attn_tree_128_42"},
               {&c.merge[0], "attn_merge_64"},
               {&c.merge[1], "attn_merge_128"},
               {&c.weights[0][0], "weights_add_64_1"},
               {&c.weights[0][1], "weights_add_64_2"},
               {&c.weights[0][2], "weights_add_64_4"},
               {&c.weights[0][3], "weights_add_64_many"},
               {&c.weights[0][4], "weights_add_64_stream"},
               {&c.weights[1][0], "weights_add_128_1"},
               {&c.weights[1][1], "weights_add_128_2"},
               {&c.weights[1][2], "weights_add_128_4"},
               {&c.weights[1][3], "weights_add_128_many"},
               {&c.weights[1][4], "weights_add_128_stream"},
               {&c.select[0], "cache_select_4"},
               {&c.select[1], "cache_select_16"},
               {&c.select[2], "cache_select_48"},
               {&c.select[3], "cache_select_any"},
               {&c.compact, "cache_compact_k"},
               {&c.argmax[0], "gemm_argmax_64"},
               {&c.argmax[1], "gemm_argmax_128"},
               {&c.argmax[2], "gemm_argmax_256"},
               {&c.argmax_final, "gemm_argmax_final"}};
  for (auto& n : names) {
    if (hipModuleGetFunction(n.fn, m, n.name) != hipSuccess) {
      (void)hipModuleUnload(m);
      return;
    }
  }
  c.module = m;
}

void cache_unload() {
  if (c.module) (void)hipModuleUnload(c.module);
  c.module = nullptr;
}

int tree_rope(const int32_t* depth, int32_t position, int32_t n, void* table, hipStream_t stream) {
  int rc = check_ready();
  if (rc) return rc;
  void* args[] = {&depth, &position, &table};
  return launch(c.rope, (uint32_t)n, 64, args, stream);
}

size_t attn_tree_need(const f16_cache* a, int32_t len, int32_t n, int32_t q_heads) {
  return attn_workspace(a, attn_plan(a, len, n, q_heads), n, q_heads);
}

}  // namespace q8_shim

extern "C" {

int f16_tree_mask(const int32_t* parents, int32_t n, uint32_t* mask, int32_t* depth,
                  void* stream) {
  if (!parents || !mask) return fail(Q8_ERR_NULL_POINTER, "null parents or mask");
  if (!aligned(parents, 4) || !aligned(mask, 4) || !aligned(depth, 4))
    return fail(Q8_ERR_MISALIGNED, "parents, mask and depth 4-byte alignment");
  if (n < 1 || n > F16_TREE_MAX_NODES)
    return fail(Q8_ERR_BAD_SHAPE, "n %d outside [1, %d]", n, F16_TREE_MAX_NODES);
  int rc = check_ready();
  if (rc) return rc;
  void* args[] = {&parents, &n, &mask, &depth};
  return q8_shim::launch(c.mask, 1, kTreeMax, args, static_cast<hipStream_t>(stream));
}

size_t f16_attn_tree_workspace_bytes(const f16_cache* a, int32_t len, int32_t n,
                                     int32_t q_heads) {
  if (check_cache(a, "cache") || check_rows(a, len, n, q_heads, 1 << 20, 1.0f)) return 0;
  // the most that any call of up to n rows over as many slots in all needs
  size_t most = 0;
  for (int32_t i = 1; i <= n; ++i)
    most = std::max(most, q8_shim::attn_tree_need(a, len + n - i, i, q_heads));
  return most;
}

int f16_attn_tree(const f16_cache* a, int32_t layer, int32_t len, const void* q, int64_t q_stride,
                  int32_t q_heads, const uint32_t* mask, int32_t n, float scale, void* out,
                  int64_t out_stride, float* lse, void* workspace, size_t workspace_bytes,
                  void* stream) {
  int rc = check_cache(a, "cache");
  if (rc) return rc;
  if (!a->k || !a->v || !q || !out) return fail(Q8_ERR_NULL_POINTER, "null k, v, q or out");
  if (layer < 0 || layer >= a->layers)
    return fail(Q8_ERR_LAYER_RANGE, "layer %d outside [0, %d)", layer, a->layers);
  if ((rc = check_rows(a, len, n, q_heads, q_stride, scale))) return rc;
  if (out_stride % 8 || out_stride < (int64_t)q_heads * a->head_dim)
    return fail(Q8_ERR_BAD_SHAPE, "row stride %lld is no multiple of 8 of at least %d",
                (long long)out_stride, q_heads * a->head_dim);
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(mask, 4) || !aligned(lse, 4))
    return fail(Q8_ERR_MISALIGNED, "q and out 16, mask and lse 4-byte alignment");
  if ((rc = check_ready())) return rc;
  const AttnPlan plan = attn_plan(a, len, n, q_heads);
  const size_t need = attn_workspace(a, plan, n, q_heads);
  if (need && !workspace) return fail(Q8_ERR_NULL_POINTER, "null workspace");
  if (!aligned(workspace, 256)) return fail(Q8_ERR_MISALIGNED, "workspace 256-byte alignment");
  if (workspace_bytes < need)
    return fail(Q8_ERR_BAD_SHAPE, "workspace of %zu bytes < %zu needed", workspace_bytes, need);
  const int64_t base = (int64_t)layer * a->max_seq * a->kv_heads * a->head_dim;
  AttnTreeArgs args{static_cast<const uint16_t*>(a->k) + base,
                    static_cast<const uint16_t*>(a->v) + base,
                    static_cast<const uint16_t*>(q),
                    mask,
                    static_cast<uint16_t*>(out),
                    lse,
                    q_stride,
                    out_stride,
                    static_cast<float*>(workspace),
                    static_cast<float*>(workspace) +
                        attn_part_floats(a, n, q_heads, plan.splits),
                    len,
                    n,
                    q_heads,
                    a->kv_heads,
                    q_heads / a->kv_heads,
                    group_inverse(q_heads / a->kv_heads),
                    plan.splits,
                    plan.blocks,
                    scale * kLog2e};
  void* p[] = {&args};
  const int d = a->head_dim / 64 - 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint32_t heads = (uint32_t)a->kv_heads;
  if ((rc = q8_shim::launch3(c.attn[d][plan.kernel], heads, (uint32_t)plan.row_blocks,
                             (uint32_t)plan.splits, 256, p, st)))
    return rc;
  if (plan.splits == 1) return Q8_OK;
  return q8_shim::launch3(c.merge[d], (uint32_t)((n * args.group + 3) / 4), heads, 1, 256, p, st);
}

int f16_attn_weights_add(const f16_cache* a, int32_t len, const void* q, int64_t q_layer_stride,
                         int64_t q_stride, int32_t q_heads, const float* lse,
                         int64_t lse_layer_stride, int32_t rows, const int32_t* path, int32_t n,
                         float scale, void* stream) {
  int rc = check_cache(a, "cache");
  if (rc) return rc;
  if (!a->k || !a->weights || !q || !lse)
    return fail(Q8_ERR_NULL_POINTER, "null k, weights, q or lse");
  if ((rc = check_rows(a, len, n, q_heads, q_stride, scale))) return rc;
  if (rows < 1 || rows > (1 << 20))
    return fail(Q8_ERR_BAD_SHAPE, "rows %d outside [1, 2^20]", rows);
  if (!path && n > rows) return fail(Q8_ERR_BAD_SHAPE, "n %d exceeds the %d rows", n, rows);
  if (a->layers > 1 && (q_layer_stride % 8 || q_layer_stride < 0 || lse_layer_stride < 0))
    return fail(Q8_ERR_BAD_SHAPE, "layer strides %lld, %lld", (long long)q_layer_stride,
                (long long)lse_layer_stride);
  if (!aligned(q, 16) || !aligned(lse, 4) || !aligned(path, 4))
    return fail(Q8_ERR_MISALIGNED, "q 16, lse and path 4-byte alignment");
  if ((rc = check_ready())) return rc;
  const int group = q_heads / a->kv_heads, tiles = (n * group + 15) / 16;
  const int64_t nb = (len + n + 31) / 32, heads = (int64_t)a->layers * a->kv_heads;
  // above 64 rows: shared queries where there are workgroups enough.  256 tokens of one
  // layer, with and without: 8000 slots (520 workgroups) 32.0 and 28.2 us, 12000 (768)
  // 32.6 and 33.2, 16384 (1040) 42.1 and 47.1; 64 tokens: 8000 (504) 11.0 and 10.8,
  // 16384 (1032) 16.2 and 17.6
  const bool shared = (len + n + 127) / 128 * heads >= 3 * q8_shim::compute_units();
  const int kernel = tiles <= 1 ? 0 : tiles <= 2 ? 1 : tiles <= 4 ? 2 : shared ? 4 : 3;
  const int64_t blocks = std::clamp<int64_t>(nb * heads / (q8_shim::compute_units() * 16), 1, 16);
  WeightsArgs args{static_cast<const uint16_t*>(a->k),
                   a->weights,
                   static_cast<const uint16_t*>(q),
                   lse,
                   path,
                   a->max_seq,
                   q_layer_stride,
                   q_stride,
                   lse_layer_stride,
                   a->kv_heads,
                   q_heads,
                   group,
                   len,
                   n,
                   rows,
                   group_inverse(group),
                   (int32_t)blocks,
                   scale * kLog2e};
  void* p[] = {&args};
  const int64_t wgs = kernel == 4   ? (len + n + 127) / 128
                      : kernel == 3 ? (len + n + 63) / 64
                                    : (nb + 4 * blocks - 1) / (4 * blocks);
  return q8_shim::launch3(c.weights[a->head_dim / 64 - 1][kernel], (uint32_t)wgs,
                          (uint32_t)a->kv_heads, (uint32_t)a->layers, 256, p,
                          static_cast<hipStream_t>(stream));
}

int f16_cache_select(const f16_cache* a, int32_t len, int32_t budget, int32_t sinks,
                     int32_t recent, int32_t* keep, void* stream) {
  int rc = check_cache(a, "cache");
  if (rc) return rc;
  if (!a->weights || !keep) return fail(Q8_ERR_NULL_POINTER, "null weights or keep");
  if (!aligned(keep, 4)) return fail(Q8_ERR_MISALIGNED, "keep 4-byte alignment");
  if (len > a->max_seq || budget < 1 || budget > len)
    return fail(Q8_ERR_BAD_SHAPE, "budget %d of %d slots in a cache of %lld", budget, len,
                (long long)a->max_seq);
  if (sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return fail(Q8_ERR_BAD_SHAPE, "%d first and %d last slots in a budget of %d", sinks, recent,
                budget);
  if ((rc = check_ready())) return rc;
  SelectArgs args{a->weights, keep, a->max_seq, len, budget, sinks, recent};
  void* p[] = {&args};
  const int slots = len - sinks - recent;
  // a thread's 4, 16 or 48 weights in registers where they hold all slots
  const int kernel = slots <= 4096 ? 0 : slots <= 16384 ? 1 : slots <= 49152 ? 2 : 3;
  return q8_shim::launch(c.select[kernel],
                         (uint32_t)(a->layers * a->kv_heads), 1024, p,
                         static_cast<hipStream_t>(stream));
}

int f16_cache_compact(const f16_cache* src, const f16_cache* dst, const int32_t* keep,
                      int per_head, int32_t base, int32_t count, void* stream) {
  int rc = check_cache(src, "src");
  if (rc) return rc;
  if ((rc = check_cache(dst, "dst"))) return rc;
  if (!src->k || !src->v || !dst->k || !dst->v)
    return fail(Q8_ERR_NULL_POINTER, "null k or v");
  if (src->layers != dst->layers || src->kv_heads != dst->kv_heads ||
      src->head_dim != dst->head_dim)
    return fail(Q8_ERR_BAD_SHAPE, "the caches differ in layers, kv_heads or head_dim");
  if (base < 0 || count < 0 || (int64_t)base + count > src->max_seq ||
      (int64_t)base + count > dst->max_seq)
    return fail(Q8_ERR_BAD_SHAPE, "slots [%d, %d + %d) outside a cache of %lld and one of %lld",
                base, base, count, (long long)src->max_seq, (long long)dst->max_seq);
  const bool weights = src->weights && dst->weights;
  const bool same = src->k == dst->k || src->v == dst->v || (weights && src->weights == dst->weights);
  if (same && (src->k != dst->k || src->v != dst->v || src->max_seq != dst->max_seq ||
               (weights && src->weights != dst->weights)))
    return fail(Q8_ERR_BAD_ARGUMENT, "src and dst share some of their buffers but not all");
  if (count > 0 && !keep) return fail(Q8_ERR_NULL_POINTER, "null keep");
  if (!aligned(keep, 4)) return fail(Q8_ERR_MISALIGNED, "keep 4-byte alignment");
  if ((rc = check_ready())) return rc;
  if (count == 0) return Q8_OK;
  CompactArgs args{static_cast<const uint16_t*>(src->k),
                   static_cast<const uint16_t*>(src->v),
                   weights ? src->weights : nullptr,
                   static_cast<uint16_t*>(dst->k),
                   static_cast<uint16_t*>(dst->v),
                   weights ? dst->weights : nullptr,
                   keep,
                   src->max_seq,
                   dst->max_seq,
                   src->kv_heads,
                   src->head_dim,
                   per_head ? 1 : 0,
                   base,
                   count,
                   count,
                   same ? 1 : 0};
  const int parts = 2 * (src->head_dim / 64) + (weights ? 1 : 0);
  const int heads = src->layers * src->kv_heads;
  int ranges = 1;
  if (!same) {
    // a move between caches may be cut up: four workgroups a CU, 256 slots or more each
    ranges = std::clamp(4 * q8_shim::compute_units() / (heads * parts), 1, (count + 255) / 256);
    args.range = ((count + ranges - 1) / ranges + 255) / 256 * 256;
    ranges = (count + args.range - 1) / args.range;
  }
  void* p[] = {&args};
  return q8_shim::launch3(c.compact, (uint32_t)(parts * ranges), (uint32_t)src->kv_heads,
                          (uint32_t)src->layers, 256, p, static_cast<hipStream_t>(stream));
}

size_t f16_gemm_argmax_workspace_bytes(int32_t n) {
  if (n < 1 || n > F16_TREE_MAX_NODES) return 0;
  return (size_t)n * 8 * kArgmaxWgsMax;
}

int f16_gemm_argmax(const void* w_f16, int64_t w_rows, const void* x_f16, int32_t n,
                    void* logits_f16, int32_t* tokens, void* workspace, void* stream) {
  if (!w_f16 || !x_f16 || !tokens || !workspace)
    return fail(Q8_ERR_NULL_POINTER, "null w, x, tokens or workspace");
  if (w_rows < 1 || w_rows >= (1LL << 31))
    return fail(Q8_ERR_BAD_SHAPE, "w_rows=%lld outside [1, 2^31)", (long long)w_rows);
  if (n < 1 || n > F16_TREE_MAX_NODES)
    return fail(Q8_ERR_BAD_SHAPE, "n %d outside [1, %d]", n, F16_TREE_MAX_NODES);
  if (!aligned(w_f16, 16) || !aligned(x_f16, 16) || !aligned(workspace, 16) ||
      !aligned(logits_f16, 2) || !aligned(tokens, 4))
    return fail(Q8_ERR_MISALIGNED, "w, x and workspace 16, logits 2, tokens 4-byte alignment");
  int rc = check_ready();
  if (rc) return rc;
  const int64_t tiles = (w_rows + 127) / 128;
  int wgs = (int)std::min<int64_t>({kArgmaxWgsMax, q8_shim::compute_units(), tiles});
  GemmArgmaxArgs args{static_cast<const uint16_t*>(w_f16),
                      static_cast<const uint16_t*>(x_f16),
                      static_cast<uint16_t*>(logits_f16),
                      static_cast<uint64_t*>(workspace),
                      (int32_t)w_rows,
                      n,
                      w_rows % 4 == 0 && aligned(logits_f16, 8)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  void* p[] = {&args};
  if ((rc = q8_shim::launch(c.argmax[n <= 64 ? 0 : n <= 128 ? 1 : 2], (uint32_t)wgs, 512, p, st)))
    return rc;
  void* fargs[] = {&workspace, &wgs, &tokens};
  return q8_shim::launch(c.argmax_final, (uint32_t)n, 64, fargs, st);
}

}  // extern "C"
