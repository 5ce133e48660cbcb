// Kernels of include/f16_cache.h: attention of a tree of drafted tokens over a
// KV cache, the attention weights positions got, eviction by them, and the
// vocabulary product over several token rows.
#include "cache_args.h"
#include "decode_device.h"

namespace {

__device__ __forceinline__ float half_lo(uint32_t v) { return (float)as_f16x2(v).x; }
__device__ __forceinline__ float half_hi(uint32_t v) { return (float)as_f16x2(v).y; }

// 8 products of f16 pairs, summed in f32
__device__ __forceinline__ float dot8(const u32x4& a, const u32x4& b) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s = fmaf(half_lo(a[i]), half_lo(b[i]), s);
    s = fmaf(half_hi(a[i]), half_hi(b[i]), s);
  }
  return s;
}

// the sum over L consecutive lanes (a power of two), in each of them
template <int L>
__device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
  for (int d = 1; d < L; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

}  // namespace

// ------------------------------------------------------------ tree mask ----

// One workgroup, thread i = node i.  Ancestor sets by pointer doubling: after
// round r, anc[i] holds the 2^r nearest nodes on the way up (i among them) and
// jump[i] the node 2^r steps up (-1 behind the root, -2 once padding was met),
// so ceil(log2 n) rounds close a chain of n nodes.
extern "C" __global__ __launch_bounds__(kTreeMax) void tree_mask_k(
    const int32_t* __restrict__ parents, int n, uint32_t* __restrict__ mask,
    int32_t* __restrict__ depth) {
  __shared__ uint32_t anc[kTreeMax][9];  // 8 words, one apart in banks
  __shared__ int32_t jump[kTreeMax];
  const int i = threadIdx.x;
  uint32_t mine[8];
#pragma unroll
  for (int w = 0; w < 8; ++w) mine[w] = w == (i >> 5) ? 1u << (i & 31) : 0u;
  int j = -2;
  if (i < n) {
    const int p = parents[i];
    j = p >= -1 && p < i ? p : -2;
  }
#pragma unroll
  for (int w = 0; w < 8; ++w) anc[i][w] = mine[w];
  jump[i] = j;
  __syncthreads();
  for (int reach = 1; reach < n; reach *= 2) {
    if (j >= 0) {
#pragma unroll
      for (int w = 0; w < 8; ++w) mine[w] |= anc[j][w];
      j = jump[j];
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) anc[i][w] = mine[w];
    jump[i] = j;
    __syncthreads();
  }
  if (i >= n) return;
  const bool live = j == -1;
  const int words = (n + 31) >> 5;
  int count = 0;
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    if (w < words) mask[i * words + w] = live ? mine[w] : 0u;
    count += __popc(mine[w]);
  }
  if (depth) depth[i] = live ? count - 1 : -1;
}

// ------------------------------------------------------- tree attention ----

// Whether row i sees slot len + a, and whether it sees anything at all.
namespace {
__device__ __forceinline__ bool row_sees(const AttnTreeArgs& A, int i, int a) {
  if (!A.mask) return a <= i;
  const int words = (A.n + 31) >> 5;
  return (A.mask[i * words + (a >> 5)] >> (a & 31)) & 1;
}
__device__ __forceinline__ bool row_empty(const AttnTreeArgs& A, int i) {
  if (!A.mask) return false;
  const int words = (A.n + 31) >> 5;
  uint32_t any = 0;
  for (int w = 0; w < words; ++w) {
    uint32_t m = A.mask[i * words + w];
    if (w == words - 1 && (A.n & 31)) m &= (1u << (A.n & 31)) - 1u;
    any |= m;
  }
  return any == 0;
}
}  // namespace

// One workgroup per (row, query head); D / 8 lanes hold a position's dims, each
// such group of lanes keeps a running maximum, sum and output over every
// (groups of the workgroup)th position, and the groups meet in LDS.
template <int D>
__device__ __forceinline__ void attn_tree(const AttnTreeArgs& A) {
  constexpr int L = D / 8, G = 256 / L;
  __shared__ float sm[G], sl[G], so[G][D];
  const int t = threadIdx.x;
  const int lane = t % L, grp = t / L;
  const int i = blockIdx.x / A.q_heads, h = blockIdx.x % A.q_heads;
  uint16_t* out = A.out + (int64_t)i * A.out_stride + h * D;
  if (row_empty(A, i)) {
    if (t < D) out[t] = 0;
    if (t == 0 && A.lse) A.lse[i * A.q_heads + h] = -__builtin_inff();
    return;
  }
  const int64_t row = (int64_t)A.kv_heads * D;
  const uint16_t* kb = A.k + (h / A.group) * D + 8 * lane;
  const uint16_t* vb = A.v + (h / A.group) * D + 8 * lane;
  const u32x4 q = *reinterpret_cast<const u32x4*>(A.q + (int64_t)i * A.q_stride + h * D + 8 * lane);
  float m = -__builtin_inff(), l = 0.0f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.0f;
  for (int p = grp; p < A.len + A.n; p += G) {
    if (p >= A.len && !row_sees(A, i, p - A.len)) continue;
    const u32x4 k = *reinterpret_cast<const u32x4*>(kb + p * row);
    const u32x4 v = *reinterpret_cast<const u32x4*>(vb + p * row);
    const float s = A.scale * sum_lanes<L>(dot8(q, k));
    const float mn = fmaxf(m, s);
    const float a = m == -__builtin_inff() ? 0.0f : expf(m - mn);
    const float w = expf(s - mn);
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      o[e] = o[e] * a + w * ((e & 1) ? half_hi(v[e >> 1]) : half_lo(v[e >> 1]));
    m = mn;
  }
  if (lane == 0) {
    sm[grp] = m;
    sl[grp] = l;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) so[grp][8 * lane + e] = o[e];
  __syncthreads();
  if (t < D) {
    float M = -__builtin_inff(), S = 0.0f, v = 0.0f;
    for (int g = 0; g < G; ++g) M = fmaxf(M, sm[g]);
    for (int g = 0; g < G; ++g) {
      const float w = sm[g] == -__builtin_inff() ? 0.0f : expf(sm[g] - M);
      S += sl[g] * w;
      v += so[g][t] * w;
    }
    out[t] = f32_to_f16_bits(v / S);
    if (t == 0 && A.lse) A.lse[i * A.q_heads + h] = M + logf(S);
  }
}
extern "C" __global__ __launch_bounds__(256) void attn_tree_64(AttnTreeArgs A) { attn_tree<64>(A); }
extern "C" __global__ __launch_bounds__(256) void attn_tree_128(AttnTreeArgs A) {
  attn_tree<128>(A);
}

// ---------------------------------------------------- attention weights ----

// D / 8 lanes per slot, 256 / (D / 8) slots per workgroup; grid.y = layer and
// kv head.  Each slot's sum runs over the rows in order.
template <int D>
__device__ __forceinline__ void weights_add(const WeightsArgs& A) {
  constexpr int L = D / 8, G = 256 / L;
  const int lane = threadIdx.x % L;
  const int p = blockIdx.x * G + threadIdx.x / L;
  const int layer = blockIdx.y / A.kv_heads, kvh = blockIdx.y % A.kv_heads;
  if (p >= A.len + A.n) return;
  const u32x4 k = *reinterpret_cast<const u32x4*>(
      A.k + ((layer * A.max_seq + p) * A.kv_heads + kvh) * D + 8 * lane);
  float sum = 0.0f;
  for (int i = p < A.len ? 0 : p - A.len; i < A.n; ++i) {
    const int r = A.path ? A.path[i] : i;
    if (r < 0 || r >= A.rows) continue;
    for (int g = 0; g < A.group; ++g) {
      const int h = kvh * A.group + g;
      const u32x4 q = *reinterpret_cast<const u32x4*>(A.q + layer * A.q_layer_stride +
                                                      r * A.q_stride + h * D + 8 * lane);
      const float lse = A.lse[layer * A.lse_layer_stride + (int64_t)r * A.q_heads + h];
      const float s = A.scale * sum_lanes<L>(dot8(q, k));
      if (lse != -__builtin_inff()) sum += expf(s - lse);
    }
  }
  if (lane == 0) {
    float* w = A.weights + ((int64_t)layer * A.kv_heads + kvh) * A.max_seq + p;
    *w = p < A.len ? *w + sum : sum;
  }
}
extern "C" __global__ __launch_bounds__(256) void weights_add_64(WeightsArgs A) {
  weights_add<64>(A);
}
extern "C" __global__ __launch_bounds__(256) void weights_add_128(WeightsArgs A) {
  weights_add<128>(A);
}

// ------------------------------------------------------------ selection ----

namespace {
// An unsigned number that orders as the weight does: -0 as 0, NaN below all.
__device__ __forceinline__ uint32_t weight_order(float w) {
  if (w != w) return 0u;
  uint32_t b = __float_as_uint(w);
  if (b == 0x80000000u) b = 0u;
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
}  // namespace

// One workgroup per layer and kv head.  The weight of the last slot that still
// fits is found digit by digit (8 bits of its order number at a time, a
// histogram of the slots that agree in the digits before); then the slots are
// walked in order and each thread's place comes from a prefix count, so the
// result has no order of arrival in it.
extern "C" __global__ __launch_bounds__(1024) void cache_select_k(SelectArgs A) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t wave_above[16], wave_equal[16];
  __shared__ uint32_t s_prefix, s_need;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const float* w = A.weights + (int64_t)blockIdx.x * A.max_seq;
  int32_t* keep = A.keep + (int64_t)blockIdx.x * A.budget;
  const int first = A.sinks, last = A.len - A.recent;
  const int middle = A.budget - A.sinks - A.recent;
  for (int j = t; j < A.sinks; j += 1024) keep[j] = j;
  for (int j = t; j < A.recent; j += 1024) keep[A.budget - A.recent + j] = last + j;
  if (middle == 0) return;
  if (t == 0) {
    s_prefix = 0;
    s_need = (uint32_t)middle;
  }
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (t < 256) hist[t] = 0;
    __syncthreads();
    const uint32_t prefix = s_prefix, need = s_need;
    for (int p = first + t; p < last; p += 1024) {
      const uint32_t o = weight_order(w[p]);
      if (shift == 24 || (o >> (shift + 8)) == prefix >> (shift + 8))
        atomicAdd(&hist[(o >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (t == 0) {
      uint32_t left = need;
      int d = 255;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      s_prefix = prefix | (uint32_t)d << shift;
      s_need = left;
    }
    __syncthreads();
  }
  // keep every slot above the bound, and the first s_need that equal it
  const uint32_t bound = s_prefix, ties = s_need;
  uint32_t above0 = 0, equal0 = 0;  // among the slots before this round
  for (int p0 = first; p0 < last; p0 += 1024) {
    const int p = p0 + t;
    const uint32_t o = p < last ? weight_order(w[p]) : 0u;
    const bool above = p < last && o > bound, equal = p < last && o == bound;
    const uint64_t ma = __ballot(above), me = __ballot(equal);
    const uint64_t below = ((uint64_t)1 << lane) - 1;
    if (lane == 0) {
      wave_above[wave] = (uint32_t)__popcll(ma);
      wave_equal[wave] = (uint32_t)__popcll(me);
    }
    __syncthreads();
    uint32_t a = above0, e = equal0;
    for (int v = 0; v < 16; ++v) {
      if (v < wave) {
        a += wave_above[v];
        e += wave_equal[v];
      }
      above0 += wave_above[v];
      equal0 += wave_equal[v];
    }
    a += (uint32_t)__popcll(ma & below);
    e += (uint32_t)__popcll(me & below);
    if (above || (equal && e < ties)) keep[A.sinks + a + (e < ties ? e : ties)] = p;
    __syncthreads();
  }
}

// ----------------------------------------------------------- compaction ----

// One workgroup per (layer, kv head, part): parts 0 .. head_dim / 64 - 1 move
// 128 bytes of every k row, the next head_dim / 64 the same of v, the last one
// the weights.  A workgroup walks the kept slots in order, 256 / 8 at a time,
// and waits until all of them are read before it writes: with ascending slots
// (keep[j] >= j) a write never meets a slot that is still to be read, so source
// and destination may be one.
extern "C" __global__ __launch_bounds__(256) void cache_compact_k(CompactArgs A) {
  const int t = threadIdx.x;
  const int halves = A.head_dim / 64;
  const int parts = 2 * halves + (A.w ? 1 : 0);
  const int part = blockIdx.x % parts, head = blockIdx.x / parts;
  const int layer = head / A.kv_heads, kvh = head % A.kv_heads;
  const int32_t* keep = A.keep + (A.per_head ? (int64_t)head * A.count : 0);
  const int64_t src_left = A.src_seq - A.base;
  if (part == 2 * halves) {
    const float* from = A.w + (int64_t)head * A.src_seq + A.base;
    float* to = A.w_to + (int64_t)head * A.dst_seq + A.base;
    for (int j0 = 0; j0 < A.count; j0 += 256) {
      const int j = j0 + t;
      const int64_t p = j < A.count ? keep[j] : -1;
      const bool ok = p >= 0 && p < src_left;
      const float x = ok ? from[p] : 0.0f;
      __syncthreads();
      if (ok) to[j] = x;
    }
    return;
  }
  const int64_t row = (int64_t)A.kv_heads * A.head_dim;
  const int col = kvh * A.head_dim + 64 * (part % halves) + 8 * (t & 7);
  const uint16_t* from = (part < halves ? A.k : A.v) + (layer * A.src_seq + A.base) * row + col;
  uint16_t* to = (part < halves ? A.k_to : A.v_to) + (layer * A.dst_seq + A.base) * row + col;
  for (int j0 = 0; j0 < A.count; j0 += 32) {
    const int j = j0 + (t >> 3);
    const int64_t p = j < A.count ? keep[j] : -1;
    const bool ok = p >= 0 && p < src_left;
    u32x4 x = {0, 0, 0, 0};
    if (ok) x = *reinterpret_cast<const u32x4*>(from + p * row);
    __syncthreads();
    if (ok) *reinterpret_cast<u32x4*>(to + j * row) = x;
  }
}

// ------------------------------------------------------ vocabulary rows ----

// One wave per vocabulary row and round, every token row in turn; the best
// (logit, row) of each token meets in LDS, then in the workspace.
extern "C" __global__ __launch_bounds__(256) void gemm_argmax_k(
    const uint16_t* __restrict__ w, int rows, const uint16_t* __restrict__ x, int n,
    uint16_t* __restrict__ logits, uint64_t* __restrict__ part) {
  __shared__ uint64_t best[4][kTreeMax];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  for (int i = lane; i < n; i += 64) best[wave][i] = 0;
  for (int64_t r = (int64_t)blockIdx.x * 4 + wave; r < rows; r += (int64_t)launch_wgs() * 4) {
    const u32x4* wr = reinterpret_cast<const u32x4*>(w + r * kHidden);
    const u32x4 w0 = wr[lane], w1 = wr[64 + lane];
    for (int i = 0; i < n; ++i) {
      const u32x4* xr = reinterpret_cast<const u32x4*>(x + i * kHidden);
      const float acc = wave_sum(f16_row_dot(w1, xr[64 + lane], f16_row_dot(w0, xr[lane], 0.0f)));
      const uint16_t h = f32_to_f16_bits(acc);
      if (lane == 0) {
        if (logits) logits[(int64_t)i * rows + r] = h;
        const float v = f16_bits_to_f32(h);
        const uint64_t key = v > -__builtin_inff() ? argmax_key(v, (int)r) : 0;
        if (key > best[wave][i]) best[wave][i] = key;
      }
    }
  }
  __syncthreads();
  for (int i = t; i < n; i += 256) {
    uint64_t key = best[0][i];
    for (int v = 1; v < 4; ++v) key = best[v][i] > key ? best[v][i] : key;
    part[(int64_t)blockIdx.x * n + i] = key;
  }
}

// tokens[i] from the workgroups' keys (argmax_key: the larger value, then the
// lower row; 0: none)
extern "C" __global__ __launch_bounds__(64) void gemm_argmax_final(
    const uint64_t* __restrict__ part, int wgs, int n, int32_t* __restrict__ tokens) {
  const int i = blockIdx.x;
  uint64_t key = 0;
  for (int g = threadIdx.x; g < wgs; g += 64) {
    const uint64_t k = part[(int64_t)g * n + i];
    key = k > key ? k : key;
  }
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t k = __shfl_xor((unsigned long long)key, d);
    key = k > key ? k : key;
  }
  if (threadIdx.x == 0)
    tokens[i] = key == 0 ? -1 : (int32_t)(0xffffffffu - (uint32_t)(key & 0xffffffffu));
}
