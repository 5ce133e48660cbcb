// Host side of include/kv_pages.h: argument checks and launches of the
// kernels in pages_kernels.hip.
#include "kv_pages.h"
#include "pages_args.h"
#include "q8gemv.h"
#include "shim_internal.h"

#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>

namespace {

struct {
  hipModule_t module = nullptr;
  // [head_dim 64, 128][f16, q8]
  hipFunction_t append[2][2][2] = {}, attn[2][2][3] = {}, read[2][2] = {};
  hipFunction_t sums[2] = {}, rest[2] = {};  // chunks of 2048, 8192
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
    return fail(Q8_ERR_CODE_OBJECT, "pages_gfx950.hsaco was not found or lacks a kernel");
  return Q8_OK;
}

int check_pages(const kv_pages* a) {
  if (!a) return fail(Q8_ERR_NULL_POINTER, "null pages");
  if (a->type != KV_PAGES_F16 && a->type != KV_PAGES_Q8)
    return fail(Q8_ERR_INVALID_KIND, "page type %d", a->type);
  if (a->pages < 1 || a->pages > (1LL << 24))
    return fail(Q8_ERR_BAD_SHAPE, "%lld pages outside [1, 2^24]", (long long)a->pages);
  if (a->layers < 1 || a->layers > 1024)
    return fail(Q8_ERR_BAD_SHAPE, "%d layers outside [1, 1024]", a->layers);
  if (a->kv_heads < 1 || a->kv_heads > 256)
    return fail(Q8_ERR_BAD_SHAPE, "%d kv heads outside [1, 256]", a->kv_heads);
  if (a->head_dim != 64 && a->head_dim != 128)
    return fail(Q8_ERR_BAD_SHAPE, "head_dim %d is not 64 or 128", a->head_dim);
  if (a->page_size < 16 || a->page_size > 4096 || a->page_size % 16)
    return fail(Q8_ERR_BAD_SHAPE, "page_size %d is no multiple of 16 in [16, 4096]", a->page_size);
  if (!a->k || !a->v) return fail(Q8_ERR_NULL_POINTER, "null k or v");
  if (a->type == KV_PAGES_Q8 && (!a->k_scale || !a->v_scale))
    return fail(Q8_ERR_NULL_POINTER, "8-bit pages without scales");
  if (!aligned(a->k, 16) || !aligned(a->v, 16) || !aligned(a->k_scale, 16) ||
      !aligned(a->v_scale, 16))
    return fail(Q8_ERR_MISALIGNED, "k, v and their scales 16-byte alignment");
  return Q8_OK;
}

int check_layers(const kv_pages* a, int32_t layer, int32_t layers) {
  if (layer < 0 || layers < 1 || (int64_t)layer + layers > a->layers)
    return fail(Q8_ERR_LAYER_RANGE, "layers [%d, %d + %d) outside [0, %d)", layer, layer, layers,
                a->layers);
  return Q8_OK;
}

int check_rows(const int32_t* start, int32_t seqs, int32_t rows, int32_t max_rows, int32_t most,
               int32_t most_each) {
  if (seqs < 1 || seqs > KV_PAGES_MAX_SEQS)
    return fail(Q8_ERR_BAD_SHAPE, "%d sequences outside [1, %d]", seqs, KV_PAGES_MAX_SEQS);
  if (rows < 1 || rows > most)
    return fail(Q8_ERR_BAD_SHAPE, "%d rows outside [1, %d]", rows, most);
  if (max_rows < 1 || max_rows > most_each)
    return fail(Q8_ERR_BAD_SHAPE, "%d rows of a sequence outside [1, %d]", max_rows, most_each);
  if (!start && rows != seqs)
    return fail(Q8_ERR_BAD_SHAPE, "%d rows of %d sequences without starts", rows, seqs);
  if (!aligned(start, 4)) return fail(Q8_ERR_MISALIGNED, "start 4-byte alignment");
  return Q8_OK;
}

int check_batch(const kv_pages* a, const kv_batch* b) {
  if (!b) return fail(Q8_ERR_NULL_POINTER, "null batch");
  if (!b->table || !b->length) return fail(Q8_ERR_NULL_POINTER, "null table or length");
  int rc = check_rows(b->start, b->seqs, b->rows, b->max_rows, 1 << 23, 1 << 23);
  if (rc) return rc;
  if (b->max_pages < 1 || (int64_t)b->max_pages * a->page_size > (1LL << 24))
    return fail(Q8_ERR_BAD_SHAPE, "%d pages of %d slots outside [1, 2^24] slots", b->max_pages,
                a->page_size);
  if (b->table_stride < b->max_pages)
    return fail(Q8_ERR_BAD_SHAPE, "table stride %lld < %d pages", (long long)b->table_stride,
                b->max_pages);
  if (!aligned(b->table, 4) || !aligned(b->length, 4))
    return fail(Q8_ERR_MISALIGNED, "table and length 4-byte alignment");
  return Q8_OK;
}

PagesBatch batch_args(const kv_pages* a, const kv_batch* b) {
  PagesBatch r{};
  r.table = b->table;
  r.length = b->length;
  r.start = b->start;
  r.table_stride = b->table_stride;
  r.seqs = b->seqs;
  r.rows = b->rows;
  r.max_rows = b->max_rows;
  r.pages = (int32_t)a->pages;
  r.page_size = a->page_size;
  r.slots = b->max_pages * a->page_size;
  r.tiles = a->page_size / 16;
  r.tiles_inv = r.tiles == 1 ? 0 : (uint32_t)((0xffffffffull + r.tiles) / r.tiles);
  return r;
}

int check_stride(const char* name, const void* p, int64_t stride, int64_t width) {
  if (stride % 8 || stride < width)
    return fail(Q8_ERR_BAD_SHAPE, "%s stride %lld is no multiple of 8 of at least %lld", name,
                (long long)stride, (long long)width);
  if (!aligned(p, 16)) return fail(Q8_ERR_MISALIGNED, "%s 16-byte alignment", name);
  return Q8_OK;
}

int check_heads(const kv_pages* a, int32_t q_heads) {
  if (q_heads < 1 || q_heads > 256 || q_heads % a->kv_heads || q_heads / a->kv_heads > 32)
    return fail(Q8_ERR_BAD_SHAPE, "%d query heads over %d kv heads", q_heads, a->kv_heads);
  return Q8_OK;
}

int64_t layer_rows(const kv_pages* a) { return a->pages * a->kv_heads * a->page_size; }
int64_t row_bytes(const kv_pages* a) { return (int64_t)a->head_dim * (a->type ? 1 : 2); }
int dim_of(const kv_pages* a) { return a->head_dim / 64 - 1; }

template <class P>
P* layer_at(const kv_pages* a, P* p, int32_t layer, int64_t bytes) {
  auto at = reinterpret_cast<uintptr_t>(p);
  return p ? reinterpret_cast<P*>(at + (uintptr_t)(layer * layer_rows(a) * bytes)) : nullptr;
}

uint32_t float_bits(float f) {
  uint32_t u;
  std::memcpy(&u, &f, 4);
  return u;
}

constexpr float kLog2e = 1.44269504088896341f;
constexpr int32_t kAttnRowsMax = 256;
constexpr int kVerifyRowsMax = 65535;
// Up to this many rows a CU, kv_pages_append gives a row 512 threads, all its heads at once,
// where 256 take two turns: 1 row of 32 heads 4.5 -> 4.0 us, 256 rows 5.1 -> 4.5, 512 rows 6.0 ->
// 5.9, but 1024 rows 7.7 -> 8.1 and 8192 rows 32.5 -> 42.3 (8-bit pages, replayed in a graph).
constexpr int kAppendWide = 2;

// How kv_pages_attn divides its work: as many 16-row tiles a workgroup as its rows fill, since
// a page is read once for all of them, up to the four that registers hold; and as many workgroups
// as are resident together (two a CU, one with four tiles), which then share the slots
// evenly: 4 x 131072 slots 1631 -> 194 us against a workgroup a sequence and head.
struct AttnPlan {
  int tiles;       // 0, 1, 2: 1, 2, 4 tiles of 16 rows a workgroup
  int row_blocks;
  int workers;     // workgroups of a kv head and row block
  size_t parts() const { return (size_t)2 * 16 * (1 << tiles); }  // rows of a workgroup's two
};

AttnPlan attn_plan(const kv_pages* a, int32_t max_rows, int32_t q_heads) {
  const int rows = max_rows * (q_heads / a->kv_heads);
  AttnPlan p{};
  p.tiles = rows <= 16 ? 0 : rows <= 32 ? 1 : 2;
  const int per_wg = 16 << p.tiles;
  p.row_blocks = (rows + per_wg - 1) / per_wg;
  const int wgs = (p.tiles == 2 ? 1 : 2) * q8_shim::compute_units();
  p.workers = std::max(1, wgs / (a->kv_heads * p.row_blocks));
  return p;
}

// Counters in front, where no layout of the parts reaches, then the parts.
constexpr size_t kCountBytes = 1 << 16;

size_t attn_workspace(const kv_pages* a, const AttnPlan& p) {
  const size_t wgs = (size_t)a->kv_heads * p.row_blocks * p.workers;
  return kCountBytes + wgs * p.parts() * (a->head_dim + 2) * 4;
}

// The counters, in front where no layout of the rest reaches.
constexpr size_t kVerifyCounts = 2 * kSeqsMax * kCountStep * sizeof(int32_t);

// Logits of a workgroup: 8192, or 2048 where that leaves CUs without a workgroup.  Of
// 151936 logits, by 2048 and 8192: both launches of 1 row 12.1 and 15.8 us, the first of 185 rows
// 45.2 and 29.6, of 27 rows 16.4 and 11.0, the second of 7 sequences 9.2 and 10.7, of 64
// 25.3 and 23.0.
int verify_chunk(int32_t rows, int32_t vocab) {
  return (int64_t)rows * ((vocab + 8191) / 8192) >= q8_shim::compute_units() ? 8192 : 2048;
}

}  // namespace

namespace q8_shim {

void pages_load(const char* path) {
  hipModule_t m = nullptr;
  if (hipModuleLoad(&m, path) != hipSuccess) return;
  bool ok = true;
  auto get = [&](hipFunction_t* fn, const char* name) {
    ok = ok && hipModuleGetFunction(fn, m, name) == hipSuccess;
  };
  for (int d = 0; d < 2; ++d)
    for (int q = 0; q < 2; ++q) {
      char name[64];
      const char* type = q ? "q8" : "f16";
      for (int wide = 0; wide < 2; ++wide) {
        snprintf(name, sizeof(name), "pages_append_%s%d_%s", wide ? "wide_" : "", 64 << d, type);
        get(&c.append[d][q][wide], name);
      }
      snprintf(name, sizeof(name), "pages_read_%d_%s", 64 << d, type);
      get(&c.read[d][q], name);
      for (int t = 0; t < 3; ++t) {
        snprintf(name, sizeof(name), "pages_attn_%d_%s_%d", 64 << d, type, 1 << t);
        get(&c.attn[d][q][t], name);
      }
    }
  for (int i = 0; i < 2; ++i) {
    get(&c.sums[i], i ? "verify_sums_4" : "verify_sums_1");
    get(&c.rest[i], i ? "verify_rest_4" : "verify_rest_1");
  }
  if (!ok) {
    (void)hipModuleUnload(m);
    return;
  }
  c.module = m;
}

void pages_unload() {
  if (c.module) (void)hipModuleUnload(c.module);
  c.module = nullptr;
}

int pages_check(const kv_pages* a, const kv_batch* batch, int32_t q_heads) {
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_batch(a, batch))) return rc;
  if ((rc = check_heads(a, q_heads))) return rc;
  if (batch->max_rows > kAttnRowsMax)
    return fail(Q8_ERR_BAD_SHAPE, "%d rows of a sequence outside [1, %d]", batch->max_rows,
                kAttnRowsMax);
  return Q8_OK;
}

int pages_ready() { return check_ready(); }

size_t pages_attn_need(const kv_pages* a, int32_t max_rows, int32_t q_heads) {
  size_t most = 0;
  for (int32_t m = 1; m <= max_rows; ++m)
    most = std::max(most, attn_workspace(a, attn_plan(a, m, q_heads)));
  return most;
}

}  // namespace q8_shim

extern "C" {

int kv_pages_append(const kv_pages* a, int32_t layer, const kv_batch* batch, const kv_rows* x,
                    void* stream) {
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_layers(a, layer, 1))) return rc;
  if ((rc = check_batch(a, batch))) return rc;
  if (!x || !x->k || !x->v) return fail(Q8_ERR_NULL_POINTER, "null rows, k or v");
  const int64_t kv = (int64_t)a->kv_heads * a->head_dim;
  if ((rc = check_stride("k", x->k, x->k_stride, kv))) return rc;
  if ((rc = check_stride("v", x->v, x->v_stride, kv))) return rc;
  if (x->q) {
    if (!x->q_out) return fail(Q8_ERR_NULL_POINTER, "null q_out");
    if ((rc = check_heads(a, x->q_heads))) return rc;
    const int64_t width = (int64_t)x->q_heads * a->head_dim;
    if ((rc = check_stride("q", x->q, x->q_stride, width))) return rc;
    if ((rc = check_stride("q_out", x->q_out, x->q_out_stride, width))) return rc;
    if (x->q == x->q_out && x->q_stride != x->q_out_stride)
      return fail(Q8_ERR_BAD_ARGUMENT, "q and q_out are one with two strides");
  } else if (x->q_heads) {
    return fail(Q8_ERR_NULL_POINTER, "%d query heads without q", x->q_heads);
  }
  if (!aligned(x->q_norm, 2) || !aligned(x->k_norm, 2) || !aligned(x->positions, 4))
    return fail(Q8_ERR_MISALIGNED, "q_norm and k_norm 2, positions 4-byte alignment");
  if (!(x->eps >= 0.0) || !std::isfinite(x->eps))
    return fail(Q8_ERR_BAD_ARGUMENT, "eps %g is not finite and at least 0", x->eps);
  if (x->theta != 0.0 && (!(x->theta > 0.0) || !std::isfinite(x->theta)))
    return fail(Q8_ERR_BAD_ARGUMENT, "theta %g is not 0 or finite and positive", x->theta);
  if ((rc = check_ready())) return rc;
  PagesAppendArgs args{};
  args.b = batch_args(a, batch);
  args.q = static_cast<const uint16_t*>(x->q);
  args.k = static_cast<const uint16_t*>(x->k);
  args.v = static_cast<const uint16_t*>(x->v);
  args.q_out = static_cast<uint16_t*>(x->q_out);
  args.q_norm = static_cast<const uint16_t*>(x->q_norm);
  args.k_norm = static_cast<const uint16_t*>(x->k_norm);
  args.positions = x->positions;
  args.q_stride = x->q_stride;
  args.k_stride = x->k_stride;
  args.v_stride = x->v_stride;
  args.q_out_stride = x->q_out_stride;
  args.k_to = layer_at(a, static_cast<uint8_t*>(a->k), layer, row_bytes(a));
  args.v_to = layer_at(a, static_cast<uint8_t*>(a->v), layer, row_bytes(a));
  args.k_scale = layer_at(a, a->k_scale, layer, 4);
  args.v_scale = layer_at(a, a->v_scale, layer, 4);
  args.eps = x->eps;
  args.q_heads = x->q_heads;
  args.kv_heads = a->kv_heads;
  args.rotate = x->theta != 0.0;
  if (args.rotate) {
    // one power, then products in 64-bit mantissas (a power each took 2.5 us a call)
    const long double step = std::pow((long double)x->theta, -2.0L / a->head_dim);
    long double turn = 1.0L / 6.283185307179586476925286766559L;
    for (int i = 0; i < a->head_dim / 2; ++i, turn *= step) args.turns[i] = (double)turn;
  }
  void* p[] = {&args};
  const bool wide = batch->rows <= kAppendWide * q8_shim::compute_units();
  return q8_shim::launch(c.append[dim_of(a)][a->type][wide], (uint32_t)batch->rows,
                         wide ? 512 : 256, p, static_cast<hipStream_t>(stream));
}

size_t kv_pages_attn_workspace_bytes(const kv_pages* a, const kv_batch* batch, int32_t q_heads) {
  if (check_pages(a) || check_batch(a, batch) || check_heads(a, q_heads) ||
      batch->max_rows > kAttnRowsMax)
    return 0;
  return q8_shim::pages_attn_need(a, batch->max_rows, q_heads);
}

int kv_pages_attn(const kv_pages* a, int32_t layer, const kv_batch* batch, const void* q,
                  int64_t q_stride, int32_t q_heads, float scale, void* out, int64_t out_stride,
                  float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_layers(a, layer, 1))) return rc;
  if ((rc = check_batch(a, batch))) return rc;
  if (!q || !out) return fail(Q8_ERR_NULL_POINTER, "null q or out");
  if ((rc = check_heads(a, q_heads))) return rc;
  if (batch->max_rows > kAttnRowsMax)
    return fail(Q8_ERR_BAD_SHAPE, "%d rows of a sequence outside [1, %d]", batch->max_rows,
                kAttnRowsMax);
  const int64_t width = (int64_t)q_heads * a->head_dim;
  if ((rc = check_stride("q", q, q_stride, width))) return rc;
  if ((rc = check_stride("out", out, out_stride, width))) return rc;
  const float by = scale * kLog2e * (a->type == KV_PAGES_Q8 ? 512.0f : 1.0f);
  if (!(scale > 0.0f) || !std::isfinite(by))
    return fail(Q8_ERR_BAD_ARGUMENT, "scale %g is not positive and below 2^118", scale);
  if (q == out) return fail(Q8_ERR_BAD_ARGUMENT, "out is q");
  if (!aligned(lse, 4)) return fail(Q8_ERR_MISALIGNED, "lse 4-byte alignment");
  const AttnPlan plan = attn_plan(a, batch->max_rows, q_heads);
  const size_t need = attn_workspace(a, plan);
  if (!workspace) return fail(Q8_ERR_NULL_POINTER, "null workspace");
  if (!aligned(workspace, 256)) return fail(Q8_ERR_MISALIGNED, "workspace 256-byte alignment");
  if (workspace_bytes < need)
    return fail(Q8_ERR_BAD_SHAPE, "workspace of %zu bytes < %zu needed", workspace_bytes, need);
  if ((rc = check_ready())) return rc;
  const int group = q_heads / a->kv_heads;
  const size_t wgs = (size_t)a->kv_heads * plan.row_blocks * plan.workers;
  char* const ws = static_cast<char*>(workspace);
  PagesAttnArgs args{batch_args(a, batch),
                     layer_at(a, static_cast<const uint8_t*>(a->k), layer, row_bytes(a)),
                     layer_at(a, static_cast<const uint8_t*>(a->v), layer, row_bytes(a)),
                     layer_at(a, static_cast<const float*>(a->k_scale), layer, 4),
                     layer_at(a, static_cast<const float*>(a->v_scale), layer, 4),
                     static_cast<const uint16_t*>(q),
                     static_cast<uint16_t*>(out),
                     lse,
                     q_stride,
                     out_stride,
                     q_heads,
                     a->kv_heads,
                     group,
                     (uint32_t)((0xffffffffull + group) / group),
                     float_bits(by),
                     plan.workers,
                     reinterpret_cast<int32_t*>(ws),
                     reinterpret_cast<float*>(ws + kCountBytes),
                     reinterpret_cast<float*>(ws + kCountBytes) + wgs * plan.parts() * a->head_dim};
  void* p[] = {&args};
  return q8_shim::launch3(c.attn[dim_of(a)][a->type][plan.tiles], (uint32_t)a->kv_heads,
                          (uint32_t)plan.row_blocks, (uint32_t)plan.workers, 256, p,
                          static_cast<hipStream_t>(stream));
}

int kv_pages_read(const kv_pages* a, int32_t layer, int32_t layers, const kv_batch* batch,
                  void* k_out, void* v_out, int64_t row_stride, int64_t layer_stride,
                  void* stream) {
  int rc = check_pages(a);
  if (rc) return rc;
  if ((rc = check_layers(a, layer, layers))) return rc;
  if ((rc = check_batch(a, batch))) return rc;
  const int64_t width = (int64_t)a->kv_heads * a->head_dim;
  if ((rc = check_stride("k_out", k_out, row_stride, width))) return rc;
  if ((rc = check_stride("v_out", v_out, row_stride, width))) return rc;
  if (layers > 1 && (layer_stride % 8 || layer_stride < width))
    return fail(Q8_ERR_BAD_SHAPE, "layer stride %lld is no multiple of 8 of at least %lld",
                (long long)layer_stride, (long long)width);
  if ((rc = check_ready())) return rc;
  if (!k_out && !v_out) return Q8_OK;
  PagesReadArgs args{batch_args(a, batch),
                     layer_at(a, static_cast<const uint8_t*>(a->k), layer, row_bytes(a)),
                     layer_at(a, static_cast<const uint8_t*>(a->v), layer, row_bytes(a)),
                     layer_at(a, static_cast<const float*>(a->k_scale), layer, 4),
                     layer_at(a, static_cast<const float*>(a->v_scale), layer, 4),
                     static_cast<uint16_t*>(k_out),
                     static_cast<uint16_t*>(v_out),
                     row_stride,
                     layers > 1 ? layer_stride : 0,
                     a->kv_heads};
  void* p[] = {&args};
  return q8_shim::launch3(c.read[dim_of(a)][a->type], (uint32_t)((batch->rows + 3) / 4),
                          (uint32_t)layers, 1, 256, p, static_cast<hipStream_t>(stream));
}

size_t kv_verify_workspace_bytes(int32_t rows, int32_t seqs, int32_t vocab) {
  if (check_rows(&rows, seqs, rows, 1, kVerifyRowsMax, kAttnRowsMax) || vocab < 1 ||
      vocab > (1 << 24))
    return 0;
  const size_t chunks = (size_t)(vocab + 2047) / 2048;
  return kVerifyCounts + 16 * chunks * ((size_t)rows + seqs) + sizeof(VerifyPick) * (size_t)seqs;
}

int kv_verify(const kv_drafts* d, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d || !d->logits || !d->tokens || !d->uniform || !d->out || !d->accepted || !workspace)
    return fail(Q8_ERR_NULL_POINTER,
                "null drafts, logits, tokens, uniform, out, accepted or workspace");
  int rc = check_rows(d->start, d->seqs, d->rows, d->max_rows, kVerifyRowsMax, kAttnRowsMax);
  if (rc) return rc;
  if (d->vocab < 1 || d->vocab > (1 << 24))
    return fail(Q8_ERR_BAD_SHAPE, "vocab %d outside [1, 2^24]", d->vocab);
  if (d->logits_stride < d->vocab || (d->draft && d->draft_stride < d->vocab))
    return fail(Q8_ERR_BAD_SHAPE, "row strides %lld, %lld < vocab %d",
                (long long)d->logits_stride, (long long)d->draft_stride, d->vocab);
  if (d->out_stride < d->max_rows)
    return fail(Q8_ERR_BAD_SHAPE, "out stride %lld < %d rows of a sequence",
                (long long)d->out_stride, d->max_rows);
  if (!aligned(d->logits, 2) || !aligned(d->tokens, 4) || !aligned(d->temperature, 4) ||
      !aligned(d->draft, 4) || !aligned(d->uniform, 4) || !aligned(d->out, 4) ||
      !aligned(d->accepted, 4) || !aligned(d->logprob, 4) || !aligned(workspace, 256))
    return fail(Q8_ERR_MISALIGNED, "logits 2, workspace 256, the others 4-byte alignment");
  const size_t need = kv_verify_workspace_bytes(d->rows, d->seqs, d->vocab);
  if (workspace_bytes < need)
    return fail(Q8_ERR_BAD_SHAPE, "workspace of %zu bytes < %zu needed", workspace_bytes, need);
  if ((rc = check_ready())) return rc;
  VerifyArgs args{};
  args.b.start = d->start;
  args.b.seqs = d->seqs;
  args.b.rows = d->rows;
  args.b.max_rows = d->max_rows;
  args.logits = static_cast<const uint16_t*>(d->logits);
  args.tokens = d->tokens;
  args.temperature = d->temperature;
  args.draft = d->draft;
  args.uniform = d->uniform;
  args.out = d->out;
  args.accepted = d->accepted;
  args.logprob = d->logprob;
  args.logits_stride = d->logits_stride;
  args.draft_stride = d->draft_stride;
  args.out_stride = d->out_stride;
  args.vocab = d->vocab;
  const int chunk = verify_chunk(d->rows, d->vocab), part = verify_chunk(d->seqs, d->vocab);
  args.chunks = (d->vocab + chunk - 1) / chunk;
  args.parts = (d->vocab + 2047) / 2048;
  args.count = static_cast<int32_t*>(workspace);
  args.picks = reinterpret_cast<VerifyPick*>(static_cast<char*>(workspace) + kVerifyCounts);
  args.sums = reinterpret_cast<double*>(args.picks + d->seqs);
  args.tops = args.sums + (size_t)d->rows * args.chunks;
  args.rest = args.tops + (size_t)d->rows * args.chunks;
  void* p[] = {&args};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if ((rc = q8_shim::launch3(c.sums[chunk == 8192], (uint32_t)args.chunks, (uint32_t)d->rows, 1, 256,
                             p, st)))
    return rc;
  return q8_shim::launch3(c.rest[part == 8192], (uint32_t)((d->vocab + part - 1) / part),
                          (uint32_t)d->seqs, 1, 256, p, st);
}

}  // extern "C"
