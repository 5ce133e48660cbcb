// Kernels of include/kv_pages.h: rows appended to a paged KV cache, attention over
// it, rows read back, and the verification of drafted tokens.
#include "decode_device.h"
#include "pages_args.h"
#include "verify_exp.h"

#include <type_traits>

namespace {

constexpr float kLn2 = 0.693147180559945309f;

// The sequence of row `row` (the wave's): the last whose start is not behind it, found
// by counting, 64 sequences at a time.  lo: its first row, m: how many; -1: none's.  of: the
// sequence's entry of `values` (null: left alone), requested with the starts.
template <class V>
__device__ __forceinline__ int seq_of_row(const PagesBatch& b, int row, int& lo, int& m,
                                          const V* values, V& of) {
  if (!b.start) {
    lo = row;
    m = 1;
    if (values) of = values[row];
    return row;
  }
  const int lane = threadIdx.x & 63;
  int n = 0, begin = 0, end = 0;
  V value = V();
  for (int s0 = 0; s0 < b.seqs; s0 += 64) {
    const int s = s0 + lane < b.seqs ? s0 + lane : b.seqs - 1;
    const int first = b.start[s], next = b.start[s + 1];
    const V mine = values ? values[s] : V();
    const int here =
        __popcll(__builtin_amdgcn_ballot_w64(s0 + lane < b.seqs && first <= row));
    if (here == 0) break;
    n = s0 + here;
    begin = first;
    end = next;
    value = mine;
    if (here < 64) break;
  }
  const int s = __builtin_amdgcn_readfirstlane(n) - 1;
  if (s < 0) return -1;
  auto pick = [&](int v) { return __builtin_amdgcn_readlane(v, s & 63); };
  lo = pick(begin);
  m = rows_of(b, lo, pick(end));
  of = __builtin_bit_cast(V, pick(__builtin_bit_cast(int, value)));
  return row >= lo && row < lo + m ? s : -1;
}

// The row of kv head h that holds slot p of sequence s, -1 for none.
__device__ __forceinline__ int64_t pool_row(const PagesBatch& b, int s, int64_t p, int kv_heads,
                                            int h) {
  if (!slot_ok(b, p)) return -1;
  const int at = page_of_tile(b, (int)p >> 4);
  const int page = b.table[(int64_t)s * b.table_stride + at];
  if (!page_ok(b, page)) return -1;
  return ((int64_t)page * kv_heads + h) * b.page_size + ((int)p - at * b.page_size);
}

// 8 halves that start on any 2 bytes
__device__ __forceinline__ u32x4 load_words4(const uint16_t* p) {
  typedef u32x4 __attribute__((aligned(2))) Any;
  return *(const GLOBAL_AS Any*)p;
}

__device__ __forceinline__ float half_at(u32x4 v, int j) {
  return (float)as_half((uint16_t)(v[j >> 1] >> (16 * (j & 1))));
}

}  // namespace

// --------------------------------------------------------------- append ----
//
// One workgroup a row; D / 8 lanes a head, 8 values each, the row's q, k and v heads
// side by side (and in turn where there are more than the threads hold).  The rotation's
// partners, dims i and i + D/2, are lanes half a head apart.  The angles' cosines and sines are
// worked out once a row, by one wave while the others norm their heads.  k and v in f64: the
// rounding to codes must not depend on an order of sums; q, which only rounds to f16, in
// f32 (8997 rows 45.5 -> 40.9 us).
// Few rows are bound by latency (the starts, the page's entry, the angles, the store: 1 row
// 2.9 us, 171 rows 4.9 us of 32 heads), many by the f64 operations: 8997 rows with 8-bit
// pages 40.9 us, where their 129 MB would take 25 and the operations take 26.  A wave a row was
// slower, and so were 64 registers for an eighth wave a SIMD, which spill (44.6 us).
namespace {

template <int kCtrl>
__device__ __forceinline__ double lane_of(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)b, kCtrl, 0xf, 0xf, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(b >> 32), kCtrl, 0xf, 0xf, true);
  return __builtin_bit_cast(double, lo | (uint64_t)hi << 32);
}

// f over a head's D / 8 lanes, in every one: lanes xor 1, xor 2, then the halves of 8 and of
// 16 mirrored (whose quads and eights hold one value by then).
template <int D, class F>
__device__ __forceinline__ double over_head(double v, F f) {
  v = f(v, lane_of<0xb1>(v));
  v = f(v, lane_of<0x4e>(v));
  v = f(v, lane_of<0x141>(v));
  if constexpr (D == 128) v = f(v, lane_of<0x140>(v));
  return v;
}

// The value half a head away: lane xor 8 of 16, xor 4 of 8.
template <int D>
__device__ __forceinline__ double other_half(double v) {
  if constexpr (D == 128) return lane_of<0x128>(v);
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_ds_swizzle((uint32_t)b, 0x101f);
  const uint32_t hi = __builtin_amdgcn_ds_swizzle((uint32_t)(b >> 32), 0x101f);
  return __builtin_bit_cast(double, lo | (uint64_t)hi << 32);
}

// Where the cosine and sine of frequency i lie: lanes that read theirs together do so from
// banks of their own.
template <int D>
__device__ __forceinline__ int turn_at(int i) {
  return (i & 7) * (D / 16) + (i >> 3);
}

// Norm of a head's lane, by weights wv.
template <int D>
__device__ __forceinline__ void norm_head(double (&y)[8], u32x4 wv, double eps) {
  double ss = 0.0;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss += y[j] * y[j];
  ss = over_head<D>(ss, [](double a, double b) { return a + b; });
  const double r = rsqrt(ss / D + eps);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = y[j] * r * (double)half_at(wv, j);
}

// Rotation of a head's lane c by turn[turn_at(i)] = (cos, sin).
template <int D>
__device__ __forceinline__ void turn_head(double (&y)[8], int c, const double2* turn) {
  const bool second = c >= D / 16;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const double2 a = turn[turn_at<D>((8 * c) % (D / 2) + j)];
    const double o = other_half<D>(y[j]);
    y[j] = y[j] * a.x + o * (second ? a.y : -a.y);
  }
}

// The queries' norm and rotation, which no code depends on, in f32: off by at most 2^-20 of
// |y[i]| + |y[i + D/2]| before the rounding to f16.
template <int D>
__device__ __forceinline__ void norm_head(float (&y)[8], u32x4 wv, float eps) {
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) ss = fmaf(y[j], y[j], ss);
  ss += dpp<0xb1>(ss);
  ss += dpp<0x4e>(ss);
  ss += dpp<0x141>(ss);
  if constexpr (D == 128) ss += dpp<0x140>(ss);
  const float r = __builtin_amdgcn_rsqf(ss * (1.0f / D) + eps);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = y[j] * r * half_at(wv, j);
}
template <int D>
__device__ __forceinline__ void turn_head(float (&y)[8], int c, const float2* turn) {
  const bool second = c >= D / 16;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float2 a = turn[turn_at<D>((8 * c) % (D / 2) + j)];
    float o;
    if constexpr (D == 128)
      o = dpp<0x128>(y[j]);
    else
      o = __uint_as_float(__builtin_amdgcn_ds_swizzle(__float_as_uint(y[j]), 0x101f));
    y[j] = fmaf(o, second ? a.y : -a.y, y[j] * a.x);
  }
}

__device__ __forceinline__ u32x4 packed8(const float (&y)[8]) {
  u32x4 o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = pack_f16x2(y[2 * j], y[2 * j + 1]);
  return o;
}
__device__ __forceinline__ u32x4 packed8(const double (&y)[8]) {
  u32x4 o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = pack_f16x2((float)y[2 * j], (float)y[2 * j + 1]);
  return o;
}

// The 8 codes of a lane and their head's scale.  y / scale is y times 1 / scale, rounded to
// a multiple of 2^-36: a quotient that lies on a border exactly (a v of 11 bits by a
// scale of 24 can; the next ones are 2^-25 away) is on it again, and the sum with
// 1.5 2^52 leaves the nearest integer, ties to even, in the low bits.
template <int D>
__device__ __forceinline__ uint2 codes8(const double (&y)[8], float& scale) {
  double top = 0.0;
  bool fine = true;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    top = fmax(top, fabs(y[j]));
    fine = fine && fabs(y[j]) < __builtin_inf();
  }
  if (!fine) top = __builtin_inf();
  top = over_head<D>(top, [](double a, double b) { return fmax(a, b); });
  const bool real = top < __builtin_inf();
  scale = real ? (float)(top / 127.0) : __builtin_nanf("");
  uint2 code = {0, 0};
  if (!real || scale == 0.0f) return code;
  const double inv = 1.0 / (double)scale;
  double q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = y[j] * inv;
  if (__builtin_amdgcn_ballot_w64(scale < 1.17549435e-38f) != 0) {  // a scale of few bits
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = fmin(fmax(q[j], -127.0), 127.0);
  }
  uint32_t low[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    low[j] = (uint32_t)__builtin_bit_cast(uint64_t, ((q[j] + 98304.0) - 98304.0) + 6755399441055744.0);
  const uint32_t pairs[4] = {__builtin_amdgcn_perm(low[1], low[0], 0x0c0c0400),
                             __builtin_amdgcn_perm(low[3], low[2], 0x0c0c0400),
                             __builtin_amdgcn_perm(low[5], low[4], 0x0c0c0400),
                             __builtin_amdgcn_perm(low[7], low[6], 0x0c0c0400)};
  code.x = pairs[0] | pairs[1] << 16;
  code.y = pairs[2] | pairs[3] << 16;
  return code;
}

template <int D, bool Q8, int kThreads>
__device__ __forceinline__ void pages_append(const PagesAppendArgs& A) {
  constexpr int G = D / 8, kHeads = kThreads / G;
  __shared__ double2 turn[D / 2];
  __shared__ float2 turn_f[D / 2];
  const int t = threadIdx.x, c = t % G, row = blockIdx.x;
  const int heads = A.q_heads + 2 * A.kv_heads;
  auto request = [&](int h) {
    const bool is_q = h < A.q_heads, is_v = h >= A.q_heads + A.kv_heads;
    const uint16_t* from = is_q   ? A.q + row * A.q_stride + h * D
                           : is_v ? A.v + row * A.v_stride + (h - A.q_heads - A.kv_heads) * D
                                  : A.k + row * A.k_stride + (h - A.q_heads) * D;
    return load_global(reinterpret_cast<const u32x4*>(from + 8 * c));
  };
  int h = t / G;
  u32x4 x = {};
  if (h < heads) x = request(h);
  u32x4 qw = {}, kw = {};
  if (A.q_norm) qw = load_words4(A.q_norm + 8 * c);
  if (A.k_norm) kw = load_words4(A.k_norm + 8 * c);
  const int position = A.positions ? A.positions[row] : 0;
  const double step = t < D / 2 ? A.turns[t] : 0.0;
  int lo, m, length = 0;
  const int s = seq_of_row(A.b, row, lo, m, A.b.length, length);
  if (s < 0) return;
  const int64_t slot = (int64_t)length - m + (row - lo);
  const int64_t to = pool_row(A.b, s, slot, A.kv_heads, 0);  // of head 0
  double y[8];
  auto normed = [&](u32x4 x) {  // a k or v into y
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = (double)half_at(x, j);
    if (h < A.q_heads + A.kv_heads && A.k_norm) norm_head<D>(y, kw, A.eps);
  };
  if (A.rotate && t < D / 2) {
    const double by = (double)(A.positions ? (int64_t)position : slot) * step;
    double2 a;
    sincospi(2.0 * (by - rint(by)), &a.y, &a.x);
    turn[turn_at<D>(t)] = a;
    turn_f[turn_at<D>(t)] = make_float2((float)a.x, (float)a.y);
  }
  if (h >= A.q_heads && h < heads) normed(x);  // while the angles' wave is busy
  if (A.rotate) __syncthreads();
  // (an eps that f32 does not hold: a head of zeros stays one)
  const float eps = A.eps > 0.0 ? fmaxf((float)A.eps, 1.2e-38f) : 0.0f;
  bool more = false;
  for (; h < A.q_heads; h += kHeads, more = true) {
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = half_at(x, j);
    if (h + kHeads < heads) x = request(h + kHeads);
    if (A.q_norm) norm_head<D>(q, qw, eps);
    if (A.rotate) turn_head<D>(q, c, turn_f);
    *reinterpret_cast<u32x4*>(A.q_out + row * A.q_out_stride + h * D + 8 * c) = packed8(q);
  }
  for (; h < heads; h += kHeads, more = true) {
    if (more) normed(x);
    const u32x4 here = x;
    if (h + kHeads < heads) x = request(h + kHeads);
    const bool is_v = h >= A.q_heads + A.kv_heads;
    const int64_t at = to + (int64_t)(h - A.q_heads - (is_v ? A.kv_heads : 0)) * A.b.page_size;
    void* pool = is_v ? A.v_to : A.k_to;
    if (!is_v && A.rotate) turn_head<D>(y, c, turn);
    if constexpr (Q8) {
      float scale;
      const uint2 code = codes8<D>(y, scale);
      if (to >= 0) {
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + at * D + 8 * c) = code;
        if (c == 0) (is_v ? A.v_scale : A.k_scale)[at] = scale;
      }
    } else if (to >= 0) {
      *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(pool) + at * D + 8 * c) =
          is_v ? here : packed8(y);
    }
  }
}

}  // namespace

#define PAGES_APPEND(D, N, Q8)                                                                    \
  extern "C" __global__ __launch_bounds__(256) void pages_append_##D##_##N(PagesAppendArgs A) {    \
    pages_append<D, Q8, 256>(A);                                                                  \
  }                                                                                               \
  extern "C" __global__ __launch_bounds__(512) void pages_append_wide_##D##_##N(PagesAppendArgs A) { \
    pages_append<D, Q8, 512>(A);                                                                  \
  }
PAGES_APPEND(64, f16, false)
PAGES_APPEND(64, q8, true)
PAGES_APPEND(128, f16, false)
PAGES_APPEND(128, q8, true)

// ------------------------------------------------------------ attention ----
//
// The rows of one kv head are its query heads' rows of a sequence's m new rows, r =
// group i + head, in tiles of 16.  A wave works on blocks of 32 slots without LDS, K and
// V straight from memory into registers:
//   S^T = K Q^T (v_mfma_f32_16x16x32_f16: exact products, f32 sums): lane (c16, grp)
//     holds the scores of row c16 at slots 4 grp + e and 16 + 4 grp + e, e < 4;
//   weights 2^(s - m) against a reference m per row, which is set kRefRoom
//     below the first block's maximum and moves only when the sum of a lane's 8
//     weights passes kSumMax;
//   O^T += V^T P^T with the weights as they stand in the lanes: the product's 32 k
//     slots mean slots 4 grp + e, 16 + 4 grp + e.  A lane reads those 8 slots' dims
//     (D/16) c16 .. + D/16 - 1 and pairs them up by byte permutes; MFMA n of the
//     D / 16 makes the dims (D/16) i + n.
// K and V come from memory once and are used by one wave alone: LDS would only add a stop.
// A block's registers are requested again for the wave's next block as soon as they have
// been used (a second set of them spilled), two waves a SIMD cover the rest.  Four tiles of
// head_dim 128 leave room for one wave; two tiles spill, 2 registers in f16 and 4 in 8 bits, and
// four tiles in 8 bits 5, which go to accumulators.  Bound by
// memory where sequences are long: 4 x 131072 slots of 8 kv heads in 8 bits, 1.1 GB, 193 us, 5.7 TB/s
// (a copy 5.1); 16 sequences, 45 rows over 34052 slots in all, f16, 140 MB, 35 us, 4.0 TB/s, of which
// cut sequences and ramps take 8; 1 x 300 slots 8 us, all latency.
// A weight goes into the product as the sum of two f16 values: 2^-22 of itself, 2^-25 where
// the second is subnormal, which is 2^-31 of a row's largest weight, 2^6 at least.
// 8-bit codes become f16 multiples of 2^-9, exact; a row's k scale multiplies its
// score and its v scale its weight, so that the reference is that of s + log2 v_scale.
namespace {

#define CONST_AS __attribute__((address_space(4)))

constexpr float kRefRoom = 6.0f, kRefMax = 10.0f, kSumMax = 16384.0f;
constexpr float kCodeUnit = 512.0f;    // codes stand in the products as code / 512
constexpr float kLeastLogScale = -64.0f;  // values below 2^-57 leave no trace in an f16
// A weight whose v scale is next to nothing adds to the sum of weights alone, which would
// pass what an f32 holds: the reference moves for these too, which then are 2^74 at most
// (kRefMax - kLeastLogScale), 2^98 the sum of 2^24.
constexpr float kPlainMax = 0x1p64f;

// 0x00b200b1 for two bytes, as f16 numbers u 2^-24, times 2^15 less 128 2^-9
__device__ __forceinline__ f16x2 code_pair(uint32_t bytes) {
  const f16x2 u = __builtin_bit_cast(f16x2, bytes);
  const f16x2 a = {(_Float16)32768.0f, (_Float16)32768.0f}, b = {(_Float16)-0.25f, (_Float16)-0.25f};
  return __builtin_elementwise_fma(u, a, b);
}
// 8 codes in order
__device__ __forceinline__ f16x8 code8(uint32_t lo, uint32_t hi) {
  lo ^= 0x80808080u;
  hi ^= 0x80808080u;
  const f16x2 a = code_pair(__builtin_amdgcn_perm(0, lo, 0x0c010c00)),
              b = code_pair(__builtin_amdgcn_perm(0, lo, 0x0c030c02)),
              c = code_pair(__builtin_amdgcn_perm(0, hi, 0x0c010c00)),
              d = code_pair(__builtin_amdgcn_perm(0, hi, 0x0c030c02));
  return (f16x8){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

__device__ __forceinline__ uint32_t special_bits(uint32_t b) {
  return ((b & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}

// Words of global memory, W at a time.
template <int W>
struct Words {
  uint32_t w[W];
};
template <int W>
__device__ __forceinline__ Words<W> load_words(const uint8_t* p) {
  typedef uint32_t V __attribute__((ext_vector_type(W)));
  Words<W> r;
  if constexpr (W == 1) {
    r.w[0] = *(const GLOBAL_AS uint32_t*)p;
  } else {
    const V v = *(const GLOBAL_AS V*)p;
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = v[i];
  }
  return r;
}

template <int D, bool Q8, int T>
struct AttnWave {
  static constexpr int kBytes = Q8 ? D : 2 * D;  // of a row
  static constexpr int kK = kBytes / 64;         // 16-byte pieces of a lane's K row share
  static constexpr int kV = kBytes / 64;         // words of a lane's V row share
  // Where the two tiles of 16 slots of block b are: rows of the pool; bit nt of ok: the
  // tile's page is one.
  struct Place {
    int64_t row0, row1;
    int ok, b;
    __device__ __forceinline__ int64_t row(int nt) const { return nt ? row1 : row0; }
  };
  struct Block {
    u32x4 k[2][kK];
    Words<kV> v[8];
    f32x4 ks[2], vs[2];
  };

  const PagesAttnArgs& A;
  const int kvh, lane, c16, grp;
  const float scale;
  const CONST_AS int32_t* table;  // the sequence's
  f16x8 qf[T][D / 32];
  int seen[T];
  float m[T], l[T];
  f32x4 o[T][D / 16];

  __device__ __forceinline__ AttnWave(const PagesAttnArgs& A, int kvh)
      : A(A), kvh(kvh), lane(threadIdx.x & 63), c16(lane & 15), grp(lane >> 4),
        scale(__uint_as_float(A.scale_bits)) {}

  // Q as the B operand: column c16 is row row0 + 16 j + c16, its dims as K's lanes
  // hold theirs
  __device__ __forceinline__ void start(int lo, int rows, int length, int row0) {
    const int R = rows * A.group;
#pragma unroll
    for (int j = 0; j < T; ++j) {
      int r = row0 + 16 * j + c16;
      r = r < R ? r : R - 1;
      const int i = A.group == 1 ? r : (int)__umulhi((uint32_t)r, A.group_inv);
      seen[j] = slots_seen(A.b, length, rows, i);
      const uint16_t* q = A.q + (int64_t)(lo + i) * A.q_stride +
                          (kvh * A.group + r - i * A.group) * D;
#pragma unroll
      for (int st = 0; st < D / 32; ++st) {
        const int dim = Q8 ? 64 * (st >> 1) + 16 * grp + 8 * (st & 1) : 32 * st + 8 * grp;
        qf[j][st] =
            __builtin_bit_cast(f16x8, load_global(reinterpret_cast<const u32x4*>(q + dim)));
      }
      m[j] = -__builtin_inff();
      l[j] = 0.0f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[j][d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    }
  }

  // The pool row of slot 16 tile; ok = false (and a row of page 0) for none.
  __device__ __forceinline__ int64_t tile_row(int tile, bool& ok) const {
    ok = tile < A.b.slots >> 4;
    const int at = page_of_tile(A.b, ok ? tile : 0);
    int page = table[at], entry = 16 * (tile - at * A.b.tiles);
    ok = ok && page_ok(A.b, page);
    if (!ok) page = entry = 0;
    return ((int64_t)page * A.kv_heads + kvh) * A.b.page_size + entry;
  }
  __device__ __forceinline__ Place place(int b, int nb) const {  // b = -1 from block nb on
    Place p;
    p.b = b < nb ? b : -1;
    b = b < nb ? b : 0;
    bool ok0, ok1;
    p.row0 = tile_row(2 * b, ok0);
    p.row1 = tile_row(2 * b + 1, ok1);
    p.ok = ok0 | ok1 << 1;
    return p;
  }

  __device__ __forceinline__ void request_k(Block& x, const Place& p) const {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const uint8_t* kt = static_cast<const uint8_t*>(A.k) + p.row(nt) * kBytes;
#pragma unroll
      for (int i = 0; i < kK; ++i)
        x.k[nt][i] = load_global(
            reinterpret_cast<const u32x4*>(kt + (uint32_t)(c16 * kBytes + 64 * i + 16 * grp)));
      if constexpr (Q8)
        x.ks[nt] = *(const GLOBAL_AS f32x4*)(A.k_scale + p.row(nt) + (uint32_t)(4 * grp));
    }
  }
  __device__ __forceinline__ void request_v(Block& x, const Place& p) const {
    const uint8_t* vb = static_cast<const uint8_t*>(A.v);
    if constexpr (Q8) {
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
        x.vs[nt] = *(const GLOBAL_AS f32x4*)(A.v_scale + p.row(nt) + (uint32_t)(4 * grp));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x.v[e] = load_words<kV>(vb + p.row(e >> 2) * kBytes +
                              (uint32_t)((4 * grp + (e & 3)) * kBytes + 4 * kV * c16));
  }

  // The lane's slots 4 grp + e, 16 + 4 grp + e that row j sees, bits 0 .. 7.
  __device__ __forceinline__ int sees(const Place& x, int j) const {
    int bits = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      bits |= (32 * x.b + 16 * (e >> 2) + 4 * grp + (e & 3) < seen[j] && (x.ok >> (e >> 2) & 1)) << e;
    return bits;
  }

  // V as the A operand of dims (D/16) i + d
  __device__ __forceinline__ f16x8 v_frag(const Block& x, int d) const {
    if constexpr (Q8) {
      f16x2 p[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        p[e] = code_pair(__builtin_amdgcn_perm(x.v[2 * e + 1].w[d >> 2], x.v[2 * e].w[d >> 2],
                                               0x0c000c00u | (4 + (d & 3)) << 16 | (d & 3)));
      return (f16x8){p[0].x, p[0].y, p[1].x, p[1].y, p[2].x, p[2].y, p[3].x, p[3].y};
    } else {
      u32x4 p;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        p[e] = __builtin_amdgcn_perm(x.v[2 * e + 1].w[d >> 1], x.v[2 * e].w[d >> 1],
                                     d & 1 ? 0x07060302u : 0x05040100u);
      return __builtin_bit_cast(f16x8, p);
    }
  }

  // Block x at `here`; the registers of its K and of its V are filled again with those at
  // `next` (if b >= 0) as soon as they have been used.  unmasked: the slots that every
  // row of the wave sees.
  __device__ __forceinline__ void block(Block& x, const Place& here, const Place& next,
                                        int unmasked) {
    const bool masked = 32 * here.b + 32 > unmasked || here.ok != 3;
    f16x8 ph[T], pl[T];
    f32x4 sc[T][2];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int st = 0; st < D / 32; ++st) {
        f16x8 kf;
        if constexpr (Q8)
          kf = code8(x.k[nt][st >> 1][2 * (st & 1)], x.k[nt][st >> 1][2 * (st & 1) + 1]);
        else
          kf = __builtin_bit_cast(f16x8, x.k[nt][st]);
#pragma unroll
        for (int j = 0; j < T; ++j)
          sc[j][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              kf, qf[j][st], st == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : sc[j][nt], 0, 0, 0);
      }
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      f32x4 f = {scale, scale, scale, scale};
      if constexpr (Q8) f *= x.ks[nt];
#pragma unroll
      for (int j = 0; j < T; ++j) sc[j][nt] *= f;
    }
    if (next.b >= 0) request_k(x, next);
#pragma unroll
    for (int j = 0; j < T; ++j) {
      float sv[8], vs[8];  // scores in base-2 units, v scales
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sv[e] = sc[j][e >> 2][e & 3];
        vs[e] = Q8 ? x.vs[e >> 2][e & 3] : 1.0f;
      }
      if (masked) {
        const int bits = sees(here, j);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!(bits >> e & 1)) {
            sv[e] = -__builtin_inff();
            vs[e] = 0.0f;
          }
      }
      // p: weights; pv: times the v scales, what goes into the product
      float p[8], pv[8], plain = 0.0f;
      auto weigh = [&](float ref) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          p[e] = __builtin_amdgcn_exp2f(sv[e] - ref);
          pv[e] = Q8 ? p[e] * vs[e] : p[e];
        }
        if constexpr (Q8)
          plain = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        return ((pv[0] + pv[1]) + (pv[2] + pv[3])) + ((pv[4] + pv[5]) + (pv[6] + pv[7]));
      };
      float sum = weigh(m[j]);
      if (__builtin_amdgcn_ballot_w64(!(sum <= kSumMax) || !(plain <= kPlainMax)) != 0) {
        float mx = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < 8; ++e)
          mx = fmaxf(mx, Q8 ? sv[e] + fmaxf(__builtin_amdgcn_logf(vs[e]), kLeastLogScale) : sv[e]);
        mx = max_col4(mx);
        const bool grow = mx > m[j] + kRefMax;
        const float mn = grow ? mx - kRefRoom : m[j];
        const float alpha = grow ? __builtin_amdgcn_exp2f(m[j] - mn) : 1.0f;
        // every score so far masked: reference 0, weights 2^-inf = 0
        sum = weigh(mn == -__builtin_inff() ? 0.0f : mn);
        l[j] *= alpha;
        m[j] = mn;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) o[j][d] *= alpha;
      }
      l[j] += Q8 ? plain : sum;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        const f16x2 hi = __builtin_convertvector((f32x2_t){pv[e], pv[e + 1]}, f16x2);
        ph[j][e] = hi.x;
        ph[j][e + 1] = hi.y;
        const f16x2 lo = f16_rest(hi, pv[e], pv[e + 1]);
        pl[j][e] = lo.x;
        pl[j][e + 1] = lo.y;
      }
    }
    bool any = false;
    if constexpr (Q8) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int i = 0; i < kV; ++i) x.v[e].w[i] ^= 0x80808080u;
    } else {
      // A masked weight of 0 times an infinity would reach every row: infinities and
      // NaN are left out of the product.
      if (masked) {
        uint32_t special = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int i = 0; i < kV; ++i) special |= special_bits(x.v[e].w[i]);
        any = __builtin_amdgcn_ballot_w64(special != 0) != 0;
        if (any) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int i = 0; i < kV; ++i) {
              const uint32_t one = special_bits(x.v[e].w[i]) >> 15;
              x.v[e].w[i] &= ~((one << 16) - one);
            }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < D / 16; d += 2) {
      const f16x8 v0 = v_frag(x, d), v1 = v_frag(x, d + 1);
#pragma unroll
      for (int j = 0; j < T; ++j) {
        o[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[j], o[j][d], 0, 0, 0);
        o[j][d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[j], o[j][d + 1], 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < T; ++j) {
        o[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[j], o[j][d], 0, 0, 0);
        o[j][d + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[j], o[j][d + 1], 0, 0, 0);
      }
    }
    if (next.b >= 0) request_v(x, next);
    // The infinities and NaN left out go to the rows that see them, value by value.
    if constexpr (!Q8) {
      if (any) {
#pragma unroll 1
        for (int e = 0; e < 32; ++e) {
          bool ok;
          const int64_t row = tile_row(2 * here.b + (e >> 4), ok) + (e & 15);
          if (!ok) continue;
          const uint16_t* v = static_cast<const uint16_t*>(A.v) + row * D + D / 4 * grp;
#pragma unroll
          for (int j = 0; j < T; ++j) {
            if (32 * here.b + e >= seen[j]) continue;
#pragma unroll
            for (int d = 0; d < D / 4; ++d) {
              const uint16_t w = v[d];
              if ((w & 0x7c00u) == 0x7c00u)
                o[j][d % (D / 16)][d / (D / 16)] += (float)as_half(w);
            }
          }
        }
      }
    }
  }
};

// Partial results go between workgroups, which may sit on different XCDs: past the L2s.
__device__ __forceinline__ void put_pair(float* p, float a, float b) {
  const uint64_t v = __float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32;
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_pair(const float* p) {
  const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// The maximum over 16 lanes, and over the wave.
__device__ __forceinline__ float row_max16(float v) {
  v = fmaxf(v, dpp<0xb1>(v));
  v = fmaxf(v, dpp<0x4e>(v));
  v = fmaxf(v, dpp<0x141>(v));
  return fmaxf(v, dpp<0x140>(v));
}
__device__ __forceinline__ float wave_max(float v) { return max_col4(row_max16(v)); }

__device__ __forceinline__ int wave_scan(int v) {  // inclusive: rows of 16, then the rows before
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

// The work of a kv head and row block is the sequences' slots, in rounds of 128 (a block for
// each of the four waves), one sequence behind the other.  The grid's `workers`
// workgroups take equal shares of the rounds.  A sequence that lies in one share is
// finished there; of one that is cut each part leaves its (m, l, O) in the workspace,
// and the workgroup that comes last puts them together, in order.
template <int D, bool Q8, int T>
__device__ __forceinline__ void pages_attn(const PagesAttnArgs& A) {
  constexpr int kRows = 16 * T, kDims = D / 16, kStride = D + 4;
  __shared__ float so[4][16][kStride];
  __shared__ float sm[4][kRows], sl[4][kRows];
  __shared__ int ends[kSeqsMax], totals[4], longest[4], arrived;
  __shared__ int3 seqs[kSeqsMax];  // first row, rows, length
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6), lane = t & 63;
  const int kvh = blockIdx.x, rb = blockIdx.y, me = blockIdx.z;
  const int row0 = kRows * rb;
  auto node = [&A](int r) { return A.group == 1 ? r : (int)__umulhi((uint32_t)r, A.group_inv); };
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  auto blocks = [&](int rows, int length) {  // of 32 slots that this row block sees
    const int R = rows * A.group;
    const int last = (row0 + kRows < R ? row0 + kRows : R) - 1;
    return (slots_seen(A.b, length, rows, node(last)) + 31) >> 5;
  };

  // the sequences' running sums of rounds; one round at least where there are rows
  int sum = 0, most = 0;
  for (int s0 = 0; s0 < A.b.seqs; s0 += 256) {
    const int s = s0 + t;
    int n = 0;
    if (s < A.b.seqs) {
      const int length = A.b.length[s], lo = A.b.start ? A.b.start[s] : s;
      const int rows = A.b.start ? rows_of(A.b, lo, A.b.start[s + 1]) : 1;
      if (row0 < rows * A.group) {
        n = (blocks(rows, length) + 3) >> 2;
        n = n > 0 ? n : 1;
      }
      seqs[s] = {lo, rows, length};
    }
    const float wave_most = wave_max((float)n);
    n = wave_scan(n);
    if (lane == 63) {
      totals[wave] = n;
      longest[wave] = (int)wave_most;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) n += totals[w];
      most = longest[w] > most ? longest[w] : most;
    }
    if (s < A.b.seqs) ends[s] = sum + n;
    sum += (totals[0] + totals[1]) + (totals[2] + totals[3]);
    __syncthreads();
  }
  sum = uniform(sum);
  // Equal shares; as long as the longest sequence where that is four rounds or little more
  // than a share (a cut costs about 6 us: 48 x 1700 slots 41.7 -> 38.6 us, 1 x 300 9.1 -> 8.4);
  // and not so short that joining the parts of a sequence, 17 ns a row and part, takes longer
  // than the rounds, about 1 us each (1 x 8000 slots, 24 rows of a kv head 39 -> 22 us).
  int share = uniform((int)((uint32_t)(sum + A.workers - 1) / (uint32_t)A.workers));
  if (most <= 4 || 2 * most <= 3 * share) share = share > most ? share : most;
  const int rows_here = A.b.max_rows * A.group < kRows ? A.b.max_rows * A.group : kRows;
  const int least =
      uniform((int)(__builtin_sqrtf((float)most * (float)rows_here * 0.012f) + 0.5f));
  share = share > least ? share : least;
  int begin = me * share, end = begin + share < sum ? begin + share : sum, s = 0;
  if (share >= most && A.b.seqs <= A.workers) {
    // a sequence each, none cut (64 sequences of 100 to 300 slots 15.6 -> 10.3 us; whole shares
    // for sequences that are cut anyway cost more than they gave)
    if (me >= A.b.seqs) return;
    s = me;
    begin = s ? uniform(ends[s - 1]) : 0;
    end = uniform(ends[s]);
    if (begin == end) return;
  } else {
    if (begin >= end) return;
    for (int i = lane; i - lane < A.b.seqs; i += 64)
      s += __popcll(__builtin_amdgcn_ballot_w64(i < A.b.seqs && ends[i < A.b.seqs ? i : 0] <= begin));
    s = uniform(s);
  }

  typedef AttnWave<D, Q8, T> Wave;
  Wave w(A, kvh);
  const int row = t >> 4, d0 = kDims * (t & 15);  // of a tile, in the sums below
  auto write = [=, &A](int r, int lo, float M, float L, const float (&o)[kDims]) {
    const int i = node(r), h = kvh * A.group + r - i * A.group;
    const bool none = L == 0.0f;  // no slot, or none with a weight
    const float inv = none ? 0.0f : (Q8 ? kCodeUnit : 1.0f) / L;
    uint32_t packed[kDims / 2];
#pragma unroll
    for (int d = 0; d < kDims / 2; ++d)
      packed[d] = none ? 0u : pack_f16x2(o[2 * d] * inv, o[2 * d + 1] * inv);
    uint16_t* to = A.out + (int64_t)(lo + i) * A.out_stride + h * D + d0;
    if constexpr (D == 128)
      *reinterpret_cast<u32x4*>(to) = (u32x4){packed[0], packed[1], packed[2], packed[3]};
    else
      *reinterpret_cast<uint2*>(to) = make_uint2(packed[0], packed[1]);
    if (A.lse && (t & 15) == 0)
      A.lse[(int64_t)(lo + i) * A.q_heads + h] =
          none ? -__builtin_inff() : kLn2 * (M + __builtin_amdgcn_logf(L));
  };
  // worker x's first or last cut sequence of this head and row block
  const int head0 = (rb * A.kv_heads + kvh) * A.workers;
  auto part_at = [=](int x, bool opens) { return (int64_t)(2 * (head0 + x) + (opens ? 1 : 0)) * kRows; };

  for (int at = begin; at < end; ++s) {
    const int from = s ? uniform(ends[s - 1]) : 0, to = uniform(ends[s]);
    if (from == to) continue;
    const int till = to < end ? to : end;
    const int3 seq = seqs[s];
    const int lo = uniform(seq.x), rows = uniform(seq.y), length = uniform(seq.z);
    const int R = rows * A.group;
    const int unmasked = uniform(slots_seen(A.b, length, rows, node(row0)));
    int nb = uniform(blocks(rows, length));
    nb = nb < 4 * (till - from) ? nb : 4 * (till - from);
    w.table = (const CONST_AS int32_t*)(A.b.table + s * A.b.table_stride);
    const int b0 = 4 * (at - from) + wave;
    {
      typename Wave::Block x;
      typename Wave::Place here = w.place(b0, nb), next = w.place(b0 + 4, nb);
      if (here.b >= 0) {
        w.request_k(x, here);
        w.request_v(x, here);
      }
      w.start(lo, rows, length, row0);
      while (here.b >= 0) {
        const typename Wave::Place after = w.place(next.b + 4, next.b >= 0 ? nb : 0);
        w.block(x, here, next, unmasked);
        here = next;
        next = after;
      }
    }
    const bool whole = from >= begin && to <= end;
    if (at != begin) __syncthreads();  // the sequence before is done with LDS
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const float l = sum_col4(w.l[j]);
      if (w.grp == 0) {
        sm[wave][16 * j + w.c16] = w.m[j];
        sl[wave][16 * j + w.c16] = l;
      }
    }
#pragma unroll
    for (int j = 0; j < T; ++j) {
      if (j > 0) __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int d = 0; d < D / 16; d += 4)
          *reinterpret_cast<f32x4*>(&so[wave][w.c16][D / 4 * w.grp + D / 16 * e + d]) =
              (f32x4){w.o[j][d][e], w.o[j][d + 1][e], w.o[j][d + 2][e], w.o[j][d + 3][e]};
      __syncthreads();
      const int r = row0 + 16 * j + row;
      if (r < R) {
        float M = -__builtin_inff(), L = 0.0f, o[kDims];
#pragma unroll
        for (int g = 0; g < 4; ++g) M = fmaxf(M, sm[g][16 * j + row]);
        const float ref = M == -__builtin_inff() ? 0.0f : M;
#pragma unroll
        for (int d = 0; d < kDims; ++d) o[d] = 0.0f;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float f = __builtin_amdgcn_exp2f(sm[g][16 * j + row] - ref);
          L += sl[g][16 * j + row] * f;
#pragma unroll
          for (int d = 0; d < kDims; ++d) o[d] += so[g][row][d0 + d] * f;
        }
        if (whole) {
          write(r, lo, M, L, o);
        } else {
          const int64_t slot = part_at(me, at == from) + 16 * j + row;
#pragma unroll
          for (int d = 0; d < kDims; d += 2) put_pair(A.part + slot * D + d0 + d, o[d], o[d + 1]);
          if ((t & 15) == 0) put_pair(A.part_ml + 2 * slot, M, L);
        }
      }
    }
    at = till;
    if (whole) continue;
    const int x0 = from / share, parts = (to - 1) / share - x0 + 1;
    wait_vm<0>();  // this thread's part has arrived
    __syncthreads();
    if (t == 0)
      arrived = __hip_atomic_fetch_add(A.count + head0 + x0, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (uniform(arrived) != parts - 1) continue;
    if (t == 0)
      __hip_atomic_store(A.count + head0 + x0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // The last: 16 threads a row and every `take`-th part of it, then those in order.
    for (int j = 0; j < T; ++j) {
      const int left = R - row0 - 16 * j;
      if (left <= 0) break;
      const int wide = left >= 9 ? 16 : left >= 5 ? 8 : left >= 3 ? 4 : left;  // rows, a power of two
      const int take = 16 / wide, mine = row & (wide - 1), g = row / wide;
      float M = -__builtin_inff(), L = 0.0f, o[kDims];
#pragma unroll
      for (int d = 0; d < kDims; ++d) o[d] = 0.0f;
      constexpr int kAhead = 4;
      if (mine < left)
        for (int p0 = g; p0 < parts; p0 += kAhead * take) {
          float2 ml[kAhead], v[kAhead][kDims / 2];
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const int p = p0 + k * take;
            const int64_t slot = part_at(x0 + (p < parts ? p : g), (p < parts ? p : g) == 0) + 16 * j + mine;
            ml[k] = get_pair(A.part_ml + 2 * slot);
#pragma unroll
            for (int d = 0; d < kDims / 2; ++d) v[k][d] = get_pair(A.part + slot * D + d0 + 2 * d);
            if (p >= parts) ml[k] = make_float2(-__builtin_inff(), 0.0f);
          }
          float top = M;
#pragma unroll
          for (int k = 0; k < kAhead; ++k) top = fmaxf(top, ml[k].x);
          const float ref = top == -__builtin_inff() ? 0.0f : top;
          const float f = __builtin_amdgcn_exp2f(M - ref);
          L *= f;
#pragma unroll
          for (int d = 0; d < kDims; ++d) o[d] *= f;
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            if (p0 + k * take >= parts) continue;
            const float fk = __builtin_amdgcn_exp2f(ml[k].x - ref);
            L += ml[k].y * fk;
#pragma unroll
            for (int d = 0; d < kDims / 2; ++d) {
              o[2 * d] += v[k][d].x * fk;
              o[2 * d + 1] += v[k][d].y * fk;
            }
          }
          M = top;
        }
      __syncthreads();
      float* const all = &so[0][0][0];  // [16][kStride]
#pragma unroll
      for (int d = 0; d < kDims; ++d) all[row * kStride + d0 + d] = o[d];
      if ((t & 15) == 0) {
        all[row * kStride + D] = M;
        all[row * kStride + D + 1] = L;
      }
      __syncthreads();
      if (g == 0 && mine < left) {
        float top = -__builtin_inff();
        for (int k = 0; k < take; ++k) top = fmaxf(top, all[(k * wide + mine) * kStride + D]);
        const float ref = top == -__builtin_inff() ? 0.0f : top;
        float total = 0.0f, r[kDims];
#pragma unroll
        for (int d = 0; d < kDims; ++d) r[d] = 0.0f;
        for (int k = 0; k < take; ++k) {
          const float* from_k = all + (k * wide + mine) * kStride;
          const float f = __builtin_amdgcn_exp2f(from_k[D] - ref);
          total += from_k[D + 1] * f;
#pragma unroll
          for (int d = 0; d < kDims; ++d) r[d] += from_k[d0 + d] * f;
        }
        write(row0 + 16 * j + mine, lo, top, total, r);
      }
    }
  }
}

}  // namespace

#define PAGES_ATTN(D, N, Q8, T)                                                        \
  extern "C" __global__ __launch_bounds__(256, T == 4 ? 1 : 2) void                    \
      pages_attn_##D##_##N##_##T(PagesAttnArgs A) {                                    \
    pages_attn<D, Q8, T>(A);                                                           \
  }
#define PAGES_ATTN_T(D, N, Q8) PAGES_ATTN(D, N, Q8, 1) PAGES_ATTN(D, N, Q8, 2) PAGES_ATTN(D, N, Q8, 4)
PAGES_ATTN_T(64, f16, false)
PAGES_ATTN_T(64, q8, true)
PAGES_ATTN_T(128, f16, false)
PAGES_ATTN_T(128, q8, true)

// ------------------------------------------------------------------ read ----
//
// A wave a row and layer, 8 values a lane at a time: bound by memory, one read of the
// pages and one write.  28 layers of 4096 rows from 8-bit pages, 713 MB, 136 us, 5.25 TB/s; one
// layer of 333 rows 4 us, the latency of starts, table, page and store.
namespace {

template <int D, bool Q8>
__device__ __forceinline__ void pages_read(const PagesReadArgs& A) {
  const int lane = threadIdx.x & 63, layer = blockIdx.y;
  const int row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (row >= A.b.rows) return;
  int lo, m, length = 0;
  const int s = seq_of_row(A.b, row, lo, m, A.b.length, length);
  if (s < 0) return;
  const int64_t slot = (int64_t)length - m + (row - lo);
  const int64_t rows = (int64_t)layer * A.b.pages * A.kv_heads * A.b.page_size;
  const int64_t to = layer * A.layer_stride + row * A.row_stride;
  for (int c = lane; c < A.kv_heads * (D / 8); c += 64) {
    int64_t at = pool_row(A.b, s, slot, A.kv_heads, c / (D / 8));
    const bool ok = at >= 0;
    at += rows;
    const int d = 8 * (c % (D / 8));
    auto copy = [&](const void* from, const float* scale, uint16_t* out) {
      u32x4 v = {0, 0, 0, 0};
      if (ok) {
        if constexpr (Q8) {
          const uint2 code = load_global(
              reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(from) + at * D + d));
          const float f = scale[at];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t w = (j < 2 ? code.x : code.y) >> (16 * (j & 1));
            v[j] = pack_f16x2((float)(int8_t)w * f, (float)(int8_t)(w >> 8) * f);
          }
        } else {
          v = load_global(
              reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(from) + at * D + d));
        }
      }
      *reinterpret_cast<u32x4*>(out + to + 8 * c) = v;
    };
    if (A.k_out) copy(A.k, A.k_scale, A.k_out);
    if (A.v_out) copy(A.v, A.v_scale, A.v_out);
  }
}

}  // namespace

#define PAGES_READ(D, N, Q8)                                                                     \
  extern "C" __global__ __launch_bounds__(256) void pages_read_##D##_##N(PagesReadArgs A) {      \
    pages_read<D, Q8>(A);                                                                        \
  }
PAGES_READ(64, f16, false)
PAGES_READ(64, q8, true)
PAGES_READ(128, f16, false)
PAGES_READ(128, q8, true)

// ---------------------------------------------------------------- verify ----
//
// verify_sums: a chunk of one row, its maximum, the maximum's lowest index and the
// sum of exp((x - maximum) / T); the last workgroup of a sequence joins the chunks of its
// rows and finds the accepted tokens and the row that decides.  verify_rest: a part of that
// row, the sums of max(p - q, 0) and of p; the last workgroup of a sequence finds the part
// and the index whose running sum passes the random number.  All in f64: next to a
// border of the running sums, one in 151936, f32 sums would give other tokens.  exp is
// 2^(n / 256) from a table in LDS times a polynomial of degree 4 in the rest, |rest| <= ln 2 /
// 512: 4e-17 of it is left out, for a fourth of the instructions of a full f64 exp (degree 3
// leaves out 1.4e-13 and took 0.8 us less of 49.6 for 185 rows).
// Bound by the f64 operations beside the memory: 185 rows of 151936 logits (56 MB) 31 us, of
// which 17 are VALU; the deciding rows of 64 sequences with the drafter's (58 MB) 23 us; one
// row 3 and 10 us, the last being a chain of loads and joins in one workgroup.  A wave that
// keeps its own chunk, without the workgroup's joins, was no faster (30 us).
namespace {

__constant__ double kExp2[16] = {  // 2^(n / 16)
    0x1.0000000000000p+0, 0x1.0b5586cf9890fp+0, 0x1.172b83c7d517bp+0, 0x1.2387a6e756238p+0,
    0x1.306fe0a31b715p+0, 0x1.3dea64c123422p+0, 0x1.4bfdad5362a27p+0, 0x1.5ab07dd485429p+0,
    0x1.6a09e667f3bcdp+0, 0x1.7a11473eb0187p+0, 0x1.8ace5422aa0dbp+0, 0x1.9c49182a3f090p+0,
    0x1.ae89f995ad3adp+0, 0x1.c199bdd85529cp+0, 0x1.d5818dcfba487p+0, 0x1.ea4afa2a490dap+0,
};

__constant__ double kFine2[16] = {  // 2^(n / 256)
    0x1.0000000000000p+0, 0x1.00b1afa5abcbfp+0, 0x1.0163da9fb3335p+0, 0x1.02168143b0281p+0,
    0x1.02c9a3e778061p+0, 0x1.037d42e11bbccp+0, 0x1.04315e86e7f85p+0, 0x1.04e5f72f654b1p+0,
    0x1.059b0d3158574p+0, 0x1.0650a0e3c1f89p+0, 0x1.0706b29ddf6dep+0, 0x1.07bd42b72a836p+0,
    0x1.0874518759bc8p+0, 0x1.092bdf66607e0p+0, 0x1.09e3ecac6f383p+0, 0x1.0a9c79b1f3919p+0,
};

// table[n] = 2^(n / 256), by 256 threads
__device__ __forceinline__ void fill_table(double* table) {
  const int t = threadIdx.x;
  table[t] = kExp2[t >> 4] * kFine2[t & 15];
}

// VerifyExp of values that may be infinite, over the table in LDS.  Where top is +inf, which
// alone has weight then, values go through near() first.
struct Exp : VerifyExp {
  using VerifyExp::VerifyExp;
  __device__ __forceinline__ float near(float x) const {
    return !far ? x : x == __builtin_inff() ? 0.0f : -__builtin_inff();
  }
  __device__ __forceinline__ u32x4 near(u32x4 v) const {
    if (far) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = ((v[i] & 0xffffu) == 0x7c00u ? 0u : 0xfc00u) |
               ((v[i] >> 16) == 0x7c00u ? 0u : 0xfc000000u);
    }
    return v;
  }
};

// The sum over the wave, in every lane: 16 lanes by DPP, then the four rows.
__device__ __forceinline__ double wave_sum64(double v) {
  v = over_head<128>(v, [](double a, double b) { return a + b; });
  auto halves = [](double v, auto&& swap) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    auto lo = swap((uint32_t)b), hi = swap((uint32_t)(b >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) +
           __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
  };
  v = halves(v, [](uint32_t w) { return __builtin_amdgcn_permlane16_swap(w, w, false, false); });
  return halves(v, [](uint32_t w) { return __builtin_amdgcn_permlane32_swap(w, w, false, false); });
}

// Running sums over the wave: rows of 16 by shifts, then the rows before.
__device__ __forceinline__ double wave_scan64(double v) {
  auto add = [&](auto ctrl, auto rows) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)b, decltype(ctrl)::value,
                                                    decltype(rows)::value, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(b >> 32), decltype(ctrl)::value,
                                                    decltype(rows)::value, 0xf, false);
    v += __builtin_bit_cast(double, lo | (uint64_t)hi << 32);
  };
  add(std::integral_constant<int, 0x111>(), std::integral_constant<int, 0xf>());
  add(std::integral_constant<int, 0x112>(), std::integral_constant<int, 0xf>());
  add(std::integral_constant<int, 0x114>(), std::integral_constant<int, 0xf>());
  add(std::integral_constant<int, 0x118>(), std::integral_constant<int, 0xf>());
  add(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());  // row 0 to 1, 2 to 3
  add(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());  // rows 0, 1 to 2, 3
  return v;
}

// 8 values from p on, the first `count` of them; rows start on any 2 (or 4) bytes.
__device__ __forceinline__ u32x4 logits8(const uint16_t* p, int count) {
  if (count >= 8) return load_words4(p);
  u32x4 v = {0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u};  // -inf
#pragma unroll
  for (int e = 0; e < 7; ++e)
    if (e < count) v[e >> 1] = e & 1 ? (v[e >> 1] & 0xffffu) | (uint32_t)p[e] << 16 : 0xfc000000u | p[e];
  return v;
}
__device__ __forceinline__ void probs8(const float* p, int count, float (&v)[8]) {
  typedef f32x4 __attribute__((aligned(4))) Any;
  if (count >= 8) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const f32x4 w = *(const GLOBAL_AS Any*)(p + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * h + e] = w[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < count ? p[e] : 0.0f;
  }
}
// the largest of 8, no NaN
__device__ __forceinline__ float top8(u32x4 v) {
  f16x2 a = as_f16x2(v[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) a = __builtin_elementwise_max(a, as_f16x2(v[i]));
  return fmaxf(fmaxf((float)a.x, (float)a.y), -__builtin_inff());
}

__device__ __forceinline__ void put_sum(double* p, double v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get_sum(const double* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
struct Top {  // a chunk's or row's maximum and, where it takes all, its lowest index
  float top;
  int first;
};

// Whether this workgroup is the last of `all` to come here with what it has left in memory
// (past the L2s); the counter is 0 again behind it.  Every thread gets the answer.
__device__ __forceinline__ bool last_here(int32_t* count, int all, int* arrived) {
  wait_vm<0>();
  __syncthreads();
  if (threadIdx.x == 0) {
    *arrived = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (*arrived == all - 1)
      __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *arrived == all - 1;
}

__device__ __forceinline__ float log_of(float x, float top, double log_total, float heat) {
  if (!(heat > 0.0f)) return 0.0f;
  return (float)((x == top ? 0.0 : ((double)x - (double)top) / (double)heat) - log_total);
}

// The last workgroup of a sequence in the first launch: its rows joined from their
// chunks, 16 lanes a row, the accepted tokens, and the row that decides.
__device__ __forceinline__ void verify_pick(const VerifyArgs& A, int s, int lo, int m, float heat,
                                            double unit, const double* table) {
  __shared__ VerifyStat st[256];
  __shared__ uint64_t stops[4];
  const int t = threadIdx.x, c16 = t & 15;
  // what the test of token t needs is requested ahead of the chunks
  int told = -1;
  float x = 0.0f, u = 0.0f, d = 1.0f;
  if (t < m) u = A.uniform[lo + t];
  if (t < m - 1) {
    told = A.tokens[lo + t + 1];
    if (told >= 0 && told < A.vocab) {
      x = (float)as_half(A.logits[(int64_t)(lo + t) * A.logits_stride + told]);
      if (A.draft) d = A.draft[(int64_t)(lo + t) * A.draft_stride + told];
    } else {
      told = -1;
    }
  }
  for (int i = t >> 4; i < m; i += 16) {
    const int64_t at = (int64_t)(lo + i) * A.chunks;
    auto top_of = [&](int c) { return __builtin_bit_cast(Top, get_sum(A.tops + at + c)); };
    float top = -__builtin_inff();
    for (int c = c16; c < A.chunks; c += 16) top = fmaxf(top, top_of(c).top);
    top = row_max16(top);
    double total = 0.0;
    int first = 0x7fffffff;
    const Exp weight(table, top, unit);
    for (int c = c16; c < A.chunks; c += 16) {
      const double sum = get_sum(A.sums + at + c);
      const Top v = top_of(c);
      if (v.top == -__builtin_inff()) continue;
      if (v.top == top && v.first < first) first = v.first;
      total += sum * weight(weight.near(v.top));
    }
    total = over_head<128>(total, [](double a, double b) { return a + b; });
    if (!(heat > 0.0f)) {
      total = 1.0;
#pragma unroll
      for (int k = 8; k > 0; k >>= 1) {
        const int other = __shfl_xor(first, k);
        first = other < first ? other : first;
      }
    }
    if (c16 == 0) st[i] = {total, top, first};
  }
  __syncthreads();
  bool no = t >= m - 1;
  if (!no) {
    const VerifyStat row = st[t];
    const Exp weight(table, row.top, unit);
    const double e = heat > 0.0f ? weight(weight.near(x)) : (told == row.first ? 1.0 : 0.0);
    no = !(told >= 0 && row.top > -__builtin_inff() &&
           (double)u * (d > 0.0f ? (double)d : 0.0) * row.sum < e);
  }
  const uint64_t mask = __builtin_amdgcn_ballot_w64(no);
  if ((t & 63) == 0) stops[t >> 6] = mask;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    if (n == 64 * g) n += stops[g] ? __builtin_ctzll(stops[g]) : 64;
  n = n < m - 1 ? n : m - 1;
  if (t == 0) A.accepted[s] = n;
  if (t == n) A.picks[s].told = told;
  if (t == m - 1) A.picks[s].u = u;
  if (t == 0) {
    VerifyPick& p = A.picks[s];
    p.row = st[n];
    p.unit = unit;
    p.heat = heat;
    p.n = n;
  }
  if (t < A.b.max_rows && t != n) {
    A.out[s * A.out_stride + t] = t < n ? told : -1;
    if (A.logprob)
      A.logprob[s * A.out_stride + t] = t < n ? log_of(x, st[t].top, log(st[t].sum), heat) : 0.0f;
  }
}

template <int V>
__device__ __forceinline__ void verify_sums(const VerifyArgs& A) {
  __shared__ double table[256], sums[4];
  __shared__ float tops[4];
  __shared__ int firsts[4], arrived;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int chunk = blockIdx.x, row = blockIdx.y;
  const int begin = chunk * 2048 * V;
  const uint16_t* x = A.logits + (int64_t)row * A.logits_stride + begin;
  u32x4 v[V];
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = logits8(x + (i * 256 + t) * 8, A.vocab - begin - (i * 256 + t) * 8);
  fill_table(table);
  int lo, m;
  float heat = 1.0f;
  const int s = seq_of_row(A.b, row, lo, m, A.temperature, heat);
  if (s < 0) return;
  if (!A.temperature) heat = 1.0f;
  const double unit = verify_unit(heat);
  float top = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < V; ++i) top = fmaxf(top, top8(v[i]));
  top = wave_max(top);
  if (lane == 0) tops[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  int first = 0x7fffffff;
  double sum = 0.0;
  if (!(heat > 0.0f)) {
#pragma unroll
    for (int i = V - 1; i >= 0; --i)
#pragma unroll
      for (int e = 7; e >= 0; --e)
        if (half_at(v[i], e) == top) first = begin + (i * 256 + t) * 8 + e;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      const int f = __shfl_xor(first, d);
      first = f < first ? f : first;
    }
  } else if (top > -__builtin_inff()) {
    const Exp weight(table, top, unit);
    // (read again, from the caches: 8 at a time in one code, or registers cost occupancy)
#pragma unroll 1
    for (int i = 0; i < V; ++i) {
      const u32x4 x8 = weight.near(logits8(x + (i * 256 + t) * 8, A.vocab - begin - (i * 256 + t) * 8));
      double w[2] = {0.0, 0.0}, to;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double one = weight.some(half_at(x8, e), to);
        w[e & 1] = fma(one, to, w[e & 1]);
      }
      sum += w[0] + w[1];
    }
    sum = wave_sum64(sum) * weight.norm;
  }
  if (lane == 0) {
    sums[wave] = sum;
    firsts[wave] = first;
  }
  __syncthreads();
  if (t == 0) {
#pragma unroll
    for (int w = 1; w < 4; ++w) first = firsts[w] < first ? firsts[w] : first;
    const int64_t at = (int64_t)row * A.chunks + chunk;
    put_sum(A.sums + at, (sums[0] + sums[1]) + (sums[2] + sums[3]));
    put_sum(A.tops + at, __builtin_bit_cast(double, Top{top, first}));
  }
  // (a sequence of one row has nothing to decide: the second launch joins its chunks)
  if (A.b.max_rows > 1 && last_here(A.count + s * kCountStep, m * A.chunks, &arrived)) verify_pick(A, s, lo, m, heat, unit, table);
}

// A row joined from its chunks by a wave, every lane getting it.
__device__ __forceinline__ VerifyStat join_row(const VerifyArgs& A, int row, int lane, double unit,
                                               float heat, const double* table) {
  const double *sums = A.sums + (int64_t)row * A.chunks, *tops = A.tops + (int64_t)row * A.chunks;
  float top = -__builtin_inff();
  for (int c = lane; c < A.chunks; c += 64) top = fmaxf(top, __builtin_bit_cast(Top, tops[c]).top);
  top = wave_max(top);
  double total = 0.0;
  int first = 0x7fffffff;
  const Exp weight(table, top, unit);
  for (int c = lane; c < A.chunks; c += 64) {
    const double sum = sums[c];
    const Top v = __builtin_bit_cast(Top, tops[c]);
    if (v.top == -__builtin_inff()) continue;
    if (v.top == top && v.first < first) first = v.first;
    total += sum * weight(weight.near(v.top));
  }
  if (heat > 0.0f) return {wave_sum64(total), top, first};
#pragma unroll
  for (int k = 32; k > 0; k >>= 1) {
    const int other = __shfl_xor(first, k);
    first = other < first ? other : first;
  }
  return {1.0, top, first};
}

// What an entry of the deciding row weighs: max(p - q, 0) and p.
struct Decide {
  Exp weight;
  double inv_total;  // with weight's norm
  bool greedy, drafted;
  int first, told;  // the maximum's lowest index, the refused token
  __device__ __forceinline__ double p(int j, float x) const {
    return greedy ? (j == first ? 1.0 : 0.0) : weight.raw(x) * inv_total;
  }
  __device__ __forceinline__ double rest(int j, double p, float d) const {
    return drafted ? fmax(p - (double)fmaxf(d, 0.0f), 0.0) : j == told ? 0.0 : p;
  }
};

// V parts of 2048 entries a workgroup.
template <int V>
__device__ __forceinline__ void verify_rest(const VerifyArgs& A) {
  __shared__ double table[256], sum[4][2], part_sum[4][V][2], base;
  __shared__ uint64_t over[4], some_over[4];
  __shared__ __attribute__((aligned(16))) uint16_t few[8];
  __shared__ float few_q[8];
  __shared__ int arrived;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6, s = blockIdx.y;
  const int lo = A.b.start ? A.b.start[s] : s;
  const int m = A.b.start ? rows_of(A.b, lo, A.b.start[s + 1]) : 1;
  const bool single = A.b.max_rows == 1;
  VerifyPick pick = {};
  if (!single) pick = A.picks[s];
  fill_table(table);
  int32_t* const out = A.out + s * A.out_stride;
  float* const logprob = A.logprob ? A.logprob + s * A.out_stride : nullptr;
  if (m == 0) {
    if (blockIdx.x > 0) return;
    if (t == 0) A.accepted[s] = 0;
    if (t < A.b.max_rows) {
      out[t] = -1;
      if (logprob) logprob[t] = 0.0f;
    }
    return;
  }
  if (single) {
    pick.heat = A.temperature ? A.temperature[s] : 1.0f;
    pick.u = A.uniform[lo];
    pick.told = -1;
  }
  // (starts that descend may have left a sequence without a pick)
  const int n = pick.n < 0 ? 0 : pick.n < m ? pick.n : m - 1;
  const bool refused = n < m - 1;
  const uint16_t* x = A.logits + (int64_t)(lo + n) * A.logits_stride;
  const float* q = A.draft && refused ? A.draft + (int64_t)(lo + n) * A.draft_stride : nullptr;
  // entries j .. j + 7
  auto request8 = [&](int j, u32x4& v, float (&d)[8]) {
    v = logits8(x + j, A.vocab - j);
    if (q) probs8(q + j, A.vocab - j, d);
  };
  const int part0 = blockIdx.x * V;
  u32x4 v[V];
  float d[V][8] = {};
#pragma unroll
  for (int i = 0; i < V; ++i) request8((part0 + i) * 2048 + t * 8, v[i], d[i]);
  __syncthreads();  // the table
  if (single) {
    pick.unit = verify_unit(pick.heat);
    pick.row = join_row(A, lo, lane, pick.unit, pick.heat, table);
    if (blockIdx.x == 0 && t == 0) A.accepted[s] = 0;
  }
  if (blockIdx.x == 0 && t == 0) A.count[s * kCountStep] = 0;
  const Exp weight(table, pick.row.top, pick.unit);
  const Decide w = {weight, weight.norm / pick.row.sum, !(pick.heat > 0.0f),
                    A.draft != nullptr, pick.row.first, pick.told};
  const bool some = pick.row.top > -__builtin_inff();
  auto sum8 = [&](int j, u32x4 v, const float (&d)[8], double& rest, double& all) {
    double r[8], p[8];
    v = w.weight.near(v);
    if (w.greedy) {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = j + e == w.first ? 1.0 : 0.0;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = w.weight.raw(half_at(v, e)) * w.inv_total;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = w.rest(j + e, p[e], d[e]);
    rest += ((r[0] + r[1]) + (r[2] + r[3])) + ((r[4] + r[5]) + (r[6] + r[7]));
    all += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
  };
  // Pairs of sums, one pair a thread: those of the threads before, and of all.
  auto running = [&](const double (&v)[2], double (&before)[2], double (&total)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const double c = wave_scan64(v[k]);
      if (lane == 63) sum[wave][k] = c;
      before[k] = c - v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      total[k] = 0.0;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g == wave) before[k] += total[k];
        total[k] += sum[g][k];
      }
    }
    __syncthreads();
  };
  double* const sums = A.rest + (int64_t)s * A.parts * 2;
  {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      double rest = 0.0, all = 0.0;
      if (some) {
        sum8((part0 + i) * 2048 + t * 8, v[i], d[i], rest, all);
        rest = wave_sum64(rest);
        all = wave_sum64(all);
      }
      if (lane == 0) {
        part_sum[wave][i][0] = rest;
        part_sum[wave][i][1] = all;
      }
    }
    __syncthreads();
    const double* const p = &part_sum[0][0][0];
    if (t < 2 * V && part0 + (t >> 1) < A.parts)
      put_sum(sums + 2 * part0 + t, (p[t] + p[2 * V + t]) + (p[4 * V + t] + p[6 * V + t]));
  }
  if (!last_here(A.count + (kSeqsMax + s) * kCountStep, gridDim.x, &arrived)) return;
  // The last workgroup of the sequence takes the token.
  double log_total = 0.0;
  auto give = [&](int token, float of) {
    out[n] = token;
    if (logprob) logprob[n] = token < 0 ? 0.0f : log_of(of, pick.row.top, log_total, pick.heat);
  };
  if (!some) {
    if (t == 0) give(-1, 0.0f);
    return;
  }
  auto request = [&](int c0, double (&v)[2]) {
    const bool is = c0 + t < A.parts;
    v[0] = is ? get_sum(sums + 2 * (c0 + t)) : 0.0;
    v[1] = is ? get_sum(sums + 2 * (c0 + t) + 1) : 0.0;
  };
  double here[2], before[2], total[2], all[2];
  request(0, here);
  log_total = log(pick.row.sum);
  asm volatile("" : "+v"(log_total));  // while the sums are on their way
  running(here, before, total);
  for (int c0 = 256; c0 < A.parts; c0 += 256) {
    request(c0, here);
    running(here, before, all);
    total[0] += all[0];
    total[1] += all[1];
  }
  const int k = refused && total[0] > 0.0 ? 0 : 1;
  const double goal = (double)pick.u * total[k];
  // The first thread whose sum takes the running sum past the goal (then passed), else
  // the last one that weighs anything, -1 where none does.
  bool passed = false;
  auto look = [&](double here, double before) {
    const uint64_t a = __builtin_amdgcn_ballot_w64(here > 0.0 && before + here > goal);
    const uint64_t b = __builtin_amdgcn_ballot_w64(here > 0.0);
    if (lane == 0) {
      over[wave] = a;
      some_over[wave] = b;
    }
    __syncthreads();
    int place = -1;
    passed = false;
#pragma unroll
    for (int g = 3; g >= 0; --g) {
      if (over[g]) {
        place = 64 * g + __builtin_ctzll(over[g]);
        passed = true;
      } else if (!passed && place < 0 && some_over[g]) {
        place = 64 * g + 63 - __builtin_clzll(some_over[g]);
      }
    }
    __syncthreads();
    return place;
  };
  int part = -1;
  double past = 0.0;
  for (int c0 = 0; c0 < A.parts && !passed; c0 += 256) {
    if (A.parts > 256) {
      request(c0, here);
      running(here, before, all);
    }
    const int place = look(here[k], past + before[k]);
    if (place >= 0) part = c0 + place;
    if (t == place) base = past + before[k];
    if (A.parts > 256) past += all[k];
    __syncthreads();
  }
  if (part < 0) {  // a sum that is no number: there is no such index
    if (t == 0) give(-1, 0.0f);
    return;
  }
  // 8 entries in a row a thread, then the one thread's, one entry a lane
  const int j0 = part * 2048 + t * 8;
  double mine[2] = {0.0, 0.0}, run[2];
  request8(j0, v[0], d[0]);
  sum8(j0, v[0], d[0], mine[0], mine[1]);
  running(mine, run, all);
  const double from = base + run[k];
  const int place = look(mine[k], from);
  if (t == place) {
    base = from;
    *reinterpret_cast<u32x4*>(few) = v[0];
#pragma unroll
    for (int e = 0; e < 8; ++e) few_q[e] = d[0][e];
  }
  __syncthreads();
  if (wave > 0) return;
  const int j = part * 2048 + place * 8 + lane;
  double f[2] = {0.0, 0.0};
  float of = 0.0f;
  if (place >= 0 && lane < 8 && j < A.vocab) {
    of = (float)as_half(few[lane]);
    f[1] = w.p(j, w.weight.near(of));
    f[0] = w.rest(j, f[1], few_q[lane]);
  }
  const double c = base + wave_scan64(f[k]);  // (every lane takes part)
  const uint64_t b = __builtin_amdgcn_ballot_w64(f[k] > 0.0);
  const uint64_t a = __builtin_amdgcn_ballot_w64(f[k] > 0.0 && c > goal);
  if (b == 0) {
    if (lane == 0) give(-1, 0.0f);
  } else if (lane == (a ? __builtin_ctzll(a) : 63 - __builtin_clzll(b))) {
    give(j, of);
  }
}

}  // namespace

#define VERIFY(V)                                                                              \
  extern "C" __global__ __launch_bounds__(256) void verify_sums_##V(VerifyArgs A) {            \
    verify_sums<V>(A);                                                                         \
  }                                                                                            \
  extern "C" __global__ __launch_bounds__(256) void verify_rest_##V(VerifyArgs A) {            \
    verify_rest<V>(A);                                                                         \
  }
VERIFY(1)
VERIFY(4)
