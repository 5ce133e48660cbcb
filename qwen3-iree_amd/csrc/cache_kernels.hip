// Kernels of include/f16_cache.h: attention of a tree of drafted tokens over a
// KV cache, the attention weights positions got, eviction by them, and the
// vocabulary product over several token rows.
#include "cache_args.h"
#include "decode_device.h"

#include <type_traits>

namespace {

constexpr float kLn2 = 0.693147180559945309f, kLog2e = 1.44269504088896341f;

}  // namespace

// ------------------------------------------------------------ tree mask ----

// One workgroup, thread i = node i.  Ancestor sets by pointer doubling: after
// round r, anc[i] holds the 2^r nearest nodes on the way up (i among them) and
// jump[i] the node 2^r steps up (-1 behind the root, -2 once padding was met),
// so ceil(log2 n) rounds close a chain of n nodes.  Latency only, a launch and the
// rounds' barriers: 1.4 us for 1 node, 1.9 for 13, 3.3-4.8 for 256.
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

// The RoPE table of a tree (as pf_rmsnorm writes a prompt's): row i the 64 cosines,
// then the 64 sines at position `position` + depth[i]; padding as depth 0.  One wave
// a node: once a pass, not once a layer, and the angles' few instructions bound it.
extern "C" __global__ __launch_bounds__(64) void tree_rope_k(const int32_t* __restrict__ depth,
                                                             int position,
                                                             float* __restrict__ table) {
  const int i = blockIdx.x, lane = threadIdx.x;
  const int d = depth[i];
  float c, s;
  rope_angle(position + (d > 0 ? d : 0), lane, c, s);
  table[i * 128 + lane] = c;
  table[i * 128 + 64 + lane] = s;
}

// ------------------------------------------------------- tree attention ----
//
// The rows of one kv head are its query heads' rows of all nodes, r = group
// node + head, in tiles of 16.  A wave works transposed, one row per lane
// column, on blocks of 32 slots:
//   S^T = K Q^T (v_mfma_f32_16x16x32_f16: exact f16 products, f32 sums), so lane
//     (c16, grp) holds the scores of row c16 at slots 4 grp + e and 16 + 4 grp + e;
//   softmax in one pass: a reference m per row (base-2 units), weights
//     2^(s - m), their sum l and the output O relative to the same m.  m is set
//     kRefRoom below the first block's maximum and moves only when the sum of a
//     lane's 8 weights passes kSumMax (then their maximum is 2^kRefMax above m),
//     so most blocks look for no maximum and rescale nothing, every weight fits
//     f16, and small ones are normal f16 numbers down to 2^-20 of the largest;
//   O^T += V^T P^T with the weights as they stand in the lanes: the MFMA's 32 k
//     slots mean slots 4 grp + e, 16 + 4 grp + e, and V^T is read from LDS in
//     that order (transposing reads).  A weight goes into the product as the sum of
//     two f16 values (2^-22 of itself at most; one alone, 2^-11, would show in the
//     outputs beside their own rounding).
// K and V blocks are copied from memory straight into LDS, the next one while one
// is computed.  RG waves share a block (RG row groups of T tiles:
// T = 2 halves the reads of LDS, but one tile's rounds are shorter, so it pays only
// where there is much to do);
// the 4 / RG position groups of a workgroup take blocks in turn and meet in LDS.
// With one row group no wave waits for another until the end: few rows are bound
// by the bytes in flight, 64 KiB a CU, many rows by MFMA and exp2.
// The slots are divided into splits of `blocks` blocks (grid: kv heads,
// row blocks, splits; kv head fastest, so that 8 kv heads keep to an XCD each); several
// splits leave (m, l, O) in the workspace and attn_merge combines them in order.
// 16 query heads over 8 kv heads of 128 (medians): 1 node, 300 slots 7.0 us (one
// workgroup a kv head: launch, masks, four rounds); 13 nodes, 1024 slots 7.1 and 3.5
// for the merge; 61, 8191 16.0 and 5.6; 256, 16384 57-60 (570-600 TFLOP/s of scores
// and outputs, the weights' second halves not counted; MFMA and VALU 49 and 43 % busy,
// in turn) and 8.6.  With one f16 a weight above 32 rows the last was 48.8, at outputs
// 3.1e-4 relative L2 from the rounded exact ones in place of 0.3e-4.
namespace {

constexpr float kRefRoom = 6.0f, kRefMax = 10.0f, kSumMax = 16384.0f;

// Word w of row i's mask: all ones in front of it (the cache), zeros behind.
__device__ __forceinline__ uint32_t mask_word(const AttnTreeArgs& A, int i, int w) {
  const int words = (A.n + 31) >> 5;
  if (w < 0) return ~0u;
  if (w >= words) return 0u;
  if (!A.mask) {
    const int d = i - 32 * w;
    return d >= 31 ? ~0u : (d < 0 ? 0u : (2u << d) - 1u);
  }
  uint32_t m = A.mask[i * words + w];
  if (w == words - 1 && (A.n & 31)) m &= (1u << (A.n & 31)) - 1u;
  return m;
}
__device__ __forceinline__ bool row_empty(const AttnTreeArgs& A, int i) {
  uint32_t any = 0;
  for (int w = 0; w < (A.n + 31) >> 5; ++w) any |= mask_word(A, i, w);
  return any == 0;
}

// The top bits of the halves that are infinities or NaN (an exponent of all ones
// carries into its top bit, and no further).
__device__ __forceinline__ uint32_t special_bits(uint32_t b) {
  return ((b & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
}
// v with its infinities and NaN replaced by 0
__device__ __forceinline__ f16x8 without_special(f16x8 v) {
  u32x4 b = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t one = special_bits(b[i]) >> 15;  // bits 0 and 16, then their halves
    b[i] &= ~((one << 16) - one);
  }
  return __builtin_bit_cast(f16x8, b);
}

template <int D, int RG, int T>
__device__ __forceinline__ void attn_tree(const AttnTreeArgs& A) {
  constexpr int PG = 4 / RG;
  constexpr int kTile = 64 * D;            // bytes of a block of k or v
  constexpr int kPieces = kTile / 1024;    // 1 KiB copies of a block
  constexpr int kChunks = D / 8;           // 16-byte chunks of a row
  constexpr int kRowsPerPiece = 64 / kChunks;
  constexpr int kRows = 16 * T * RG;       // rows of a workgroup
  // two buffers of each position group's K and V blocks, separate arrays so
  // that the compiler sees that reading one does not wait for copies into another
  __shared__ __attribute__((aligned(1024))) uint8_t k0[PG * kTile], k1[PG * kTile];
  __shared__ __attribute__((aligned(1024))) uint8_t v0[PG * kTile], v1[PG * kTile];
  // mask words -1 .. words of the workgroup's rows
  __shared__ uint32_t sees[kRows][kTreeMax / 32 + 3];
  const int t = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lane = t & 63, c16 = lane & 15, grp = lane >> 4;
  const int rg = wave % RG, pg = wave / RG;
  const int kvh = blockIdx.x, rb = blockIdx.y, split = blockIdx.z;
  const int R = A.n * A.group;
  const int row0 = rb * kRows + 16 * T * rg;  // this wave's first row
  const int slots = A.len + A.n;
  const int nb_all = (slots + 31) >> 5;
  const int b_lo = split * A.blocks;
  const int b_hi = b_lo + A.blocks < nb_all ? b_lo + A.blocks : nb_all;
  const int64_t row_elems = (int64_t)A.kv_heads * D;
  const uint16_t* kb = A.k + kvh * D;
  const uint16_t* vb = A.v + kvh * D;

  // Q as the B operand: column c16 is row row0 + 16 j + c16, dims 32 st + 8 grp
  int node[T];
  f16x8 qf[T][D / 32];
#pragma unroll
  for (int j = 0; j < T; ++j) {
    int r = row0 + 16 * j + c16;
    r = r < R ? r : R - 1;
    node[j] = A.group == 1 ? r : (int)__umulhi((uint32_t)r, A.group_inv);
    const uint16_t* q = A.q + (int64_t)node[j] * A.q_stride +
                        (kvh * A.group + r - node[j] * A.group) * D + 8 * grp;
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
      qf[j][st] =
          __builtin_bit_cast(f16x8, load_global(reinterpret_cast<const u32x4*>(q + 32 * st)));
  }
  float m[T], l[T];
  f32x4 o[T][D / 16];
#pragma unroll
  for (int j = 0; j < T; ++j) {
    m[j] = -__builtin_inff();
    l[j] = 0.0f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) o[j][d] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  }

  // K chunk c of row r sits in slot c ^ (r mod kChunks) of its row, V chunk c in
  // c ^ 2 (r mod kChunks / 2): the fragment reads below hit distinct banks
  uint32_t k_at[kPieces / RG], v_at[kPieces / RG];  // this lane's bytes of a block
#pragma unroll
  for (int i = 0; i < kPieces / RG; ++i) {
    const int row = kRowsPerPiece * (kPieces / RG * rg + i) + lane / kChunks, c = lane % kChunks;
    k_at[i] = row * (uint32_t)(2 * row_elems) + 16 * (c ^ (row & (kChunks - 1)));
    v_at[i] = row * (uint32_t)(2 * row_elems) + 16 * (c ^ (2 * (row & (kChunks / 2 - 1))));
  }
  // block b; in the last one, slots behind the last repeat it
  auto copy = [&](auto last_t, int b, uint8_t* kt, uint8_t* vt) {
    const uint8_t* kp = reinterpret_cast<const uint8_t*>(kb + 32 * b * row_elems);
    const uint8_t* vp = reinterpret_cast<const uint8_t*>(vb + 32 * b * row_elems);
    const uint32_t row_bytes = (uint32_t)(2 * row_elems);
    auto piece = [&](const uint8_t* from, uint32_t at, uint8_t* to, int i) {
      const int pc = kPieces / RG * rg + i;
      if constexpr (decltype(last_t)::value) {
        const int over = kRowsPerPiece * pc + lane / kChunks - (slots - 1 - 32 * b);
        at -= (over > 0 ? over : 0) * row_bytes;
      }
      __builtin_amdgcn_global_load_lds((const GLOBAL_AS void*)(from + at),
                                       (LDS_AS void*)(to + pg * kTile + 1024 * pc), 16, 0, 0);
    };
#pragma unroll
    for (int i = 0; i < kPieces / RG; ++i) piece(kp, k_at[i], kt, i);
#pragma unroll
    for (int i = 0; i < kPieces / RG; ++i) piece(vp, v_at[i], vt, i);
  };
  // 4 lanes of a 16-lane group address a row each time: lane j row vrow + j / 4,
  // dims 16 d + 4 (j mod 4); the read hands lane i V[vrow + e][16 d + i], e < 4
  const int vrow = 4 * grp + (c16 >> 2);
  auto v_off = [&](int row, int d) {
    return 2 * D * row + 16 * ((2 * d + ((c16 & 3) >> 1)) ^ (2 * (row & (kChunks / 2 - 1)))) +
           8 * (c16 & 1);
  };

  uint32_t bits[T];  // of a masked block: the lane's 8 slots
  // between() runs once the block's fragments have been requested
  auto block = [&](auto masked_t, const uint8_t* kt, const uint8_t* vt, auto&& between) {
    constexpr bool kMasked = decltype(masked_t)::value;
    kt += pg * kTile;
    vt += pg * kTile;
    f16x8 kf[D / 32][2], vf[D / 16];
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
        kf[st][nt] = *reinterpret_cast<const f16x8*>(
            kt + 2 * D * (16 * nt + c16) + 16 * ((4 * st + grp) ^ (c16 & (kChunks - 1))));
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
      const v4i16 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS v4i16*)(vt + v_off(vrow, d)));
      const v4i16 a1 =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS v4i16*)(vt + v_off(vrow + 16, d)));
      vf[d] = __builtin_bit_cast(f16x8, (v8i16){a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w});
    }
    between();
    f32x4 sc[T][2];
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int j = 0; j < T; ++j)
          sc[j][nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
              kf[st][nt], qf[j][st], st == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : sc[j][nt], 0, 0, 0);
    f16x8 ph[T], pl[T];
#pragma unroll
    for (int j = 0; j < T; ++j) {
      float s[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = sc[j][e >> 2][e & 3];
      if constexpr (kMasked) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!((bits[j] >> (16 * (e >> 2) + (e & 3))) & 1)) s[e] = -__builtin_inff();
      }
      float p[8];
      auto weigh = [&](float ref) {
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s[e], A.scale, -ref));
        return ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
      };
      // The sum says whether the reference still serves: it passes the bound (or
      // is no number) where a weight does, and in a row's first block, m = -inf.
      float sum = weigh(m[j]);
      if (__builtin_amdgcn_ballot_w64(!(sum <= kSumMax)) != 0) {
        float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])),
                         fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7])));
        mx = max_col4(mx) * A.scale;
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
      l[j] += sum;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        typedef float f32x2_t __attribute__((ext_vector_type(2)));
        const f16x2 hi = __builtin_convertvector((f32x2_t){p[e], p[e + 1]}, f16x2);
        ph[j][e] = hi.x;
        ph[j][e + 1] = hi.y;
        const f16x2 lo = f16_rest(hi, p[e], p[e + 1]);
        pl[j][e] = lo.x;
        pl[j][e + 1] = lo.y;
      }
    }
    // A masked weight of 0 times an infinity would reach every row: infinities
    // and NaN are left out of the product.
    bool any = false;
    if constexpr (kMasked) {
      uint32_t special = 0;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) {
        const u32x4 w = __builtin_bit_cast(u32x4, vf[d]);
#pragma unroll
        for (int i = 0; i < 4; ++i) special |= special_bits(w[i]);
      }
      any = __builtin_amdgcn_ballot_w64(special != 0) != 0;
      if (any) {
#pragma unroll
        for (int d = 0; d < D / 16; ++d) vf[d] = without_special(vf[d]);
      }
    }
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int j = 0; j < T; ++j)
        o[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d], ph[j], o[j][d], 0, 0, 0);
#pragma unroll
    for (int d = 0; d < D / 16; ++d)
#pragma unroll
      for (int j = 0; j < T; ++j)
        o[j][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf[d], pl[j], o[j][d], 0, 0, 0);
    // They go to the rows that see them, value by value.
    if (any) {
#pragma unroll 1
      for (int x = 0; x < 32; ++x) {
        // slot x: bit 16 (x / 16) + x mod 4 of the lanes with grp (x / 4) mod 4
#pragma unroll
        for (int j = 0; j < T; ++j) {
          const bool sees = (__shfl(bits[j], c16 + 16 * ((x >> 2) & 3)) >>
                             (16 * (x >> 4) + (x & 3))) & 1;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            const int c = 2 * d + (grp >> 1);
            const uint16_t* v = reinterpret_cast<const uint16_t*>(
                vt + 2 * D * x + 16 * (c ^ (2 * (x & (kChunks / 2 - 1)))) + 8 * (grp & 1));
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (sees && (v[e] & 0x7c00u) == 0x7c00u) o[j][d][e] += f16_bits_to_f32(v[e]);
          }
        }
      }
    }
  };

  // The split's masked blocks (from the one that holds slot len on), then the
  // others; position group pg takes every PG-th of either.  With several row
  // groups the waves keep in step, one barrier a round: it shows everyone's
  // copies of this round and frees the other buffer.
  const int b_tree = A.len >> 5;
  const int b_mid = b_hi < b_tree ? b_hi : (b_lo > b_tree ? b_lo : b_tree);
  const int masked = b_hi - b_mid, plain = b_mid - b_lo;
  const int first = b_lo + ((pg - masked) & (PG - 1));  // of the plain ones
  const std::true_type kMaskedBlock;
  const std::false_type kPlainBlock;
  auto masked_bits = [&](int b) {
#pragma unroll
    for (int j = 0; j < T; ++j) {
      // a block that is masked starts at most 31 slots before len
      const int a0 = 32 * b - A.len;
      const uint32_t* w = sees[16 * (T * rg + j) + c16] + (a0 >> 5) + 1;
      bits[j] = (uint32_t)((((uint64_t)w[1] << 32) | w[0]) >> (a0 & 31)) >> (4 * grp);
    }
  };
  // plain round i: block first + PG i
  auto plain_next = [&](int i) { return first + PG * i < b_mid ? first + PG * i : -1; };
  const int plain_rounds = (plain + PG - 1) / PG;
  // Masked blocks alternate between the buffers so that the last one is in k0 and
  // the first plain one in k1.  One code for both buffers: the next copy is issued
  // behind the block's own reads, or it would have to land before them.
  const int masked_rounds = (masked + PG - 1) / PG;
  const int b_tree0 = b_mid + pg;  // this group's first masked block
  auto start = [&](int i) {  // the copy for masked round i
    if (i < masked_rounds && b_tree0 + PG * i < b_hi) {
      const bool even = ((masked_rounds - i) & 1) != 0;
      copy(kMaskedBlock, b_tree0 + PG * i, even ? k0 : k1, even ? v0 : v1);
    } else if (i >= masked_rounds && plain_next(0) >= 0) {
      copy(kPlainBlock, plain_next(0), k1, v1);
    }
  };
  start(0);
  if (masked > 0 || A.splits == 1) {
    const int words = (A.n + 31) >> 5;
    const int row = t & (kRows - 1);
    int rr = rb * kRows + row;
    rr = rr < R ? rr : R - 1;
    const int i = A.group == 1 ? rr : (int)__umulhi((uint32_t)rr, A.group_inv);
    for (int w = t / kRows; w < words + 2; w += 256 / kRows) sees[row][w] = mask_word(A, i, w - 1);
    __syncthreads();
  }
  for (int i = 0; i < masked_rounds; ++i) {
    const bool live = b_tree0 + PG * i < b_hi;
    const bool even = ((masked_rounds - i) & 1) != 0;
    if (live) masked_bits(b_tree0 + PG * i);
    wait_vm<0>();
    if constexpr (RG > 1) __syncthreads();
    if (live)
      block(kMaskedBlock, even ? k0 : k1, even ? v0 : v1, [&] {
        wait_lds();
        start(i + 1);
      });
    else
      start(i + 1);
  }
  auto round = [&](int i, const uint8_t* kt, const uint8_t* vt, uint8_t* kn, uint8_t* vn) {
    wait_vm<0>();
    if constexpr (RG > 1) __syncthreads();
    if (plain_next(i + 1) >= 0) copy(kPlainBlock, plain_next(i + 1), kn, vn);
    if (plain_next(i) >= 0) block(kPlainBlock, kt, vt, [] {});
    if constexpr (RG == 1) wait_lds();  // the buffer's reads are done before its next copy
  };
  for (int i = 0; i < plain_rounds; i += 2) {
    round(i, k1, v1, k0, v0);
    if (i + 1 < plain_rounds) round(i + 1, k0, v0, k1, v1);
  }

#pragma unroll
  for (int j = 0; j < T; ++j) l[j] = sum_col4(l[j]);
  // o[j][d][e]: dim 16 d + 4 grp + e of row row0 + 16 j + c16.  The position
  // groups meet in LDS, (m, l) first, then O in parts that fit into k0; after
  // that o[j][0 .. D / 16 / PG - 1] are the sums of this group's share of the dims.
  if constexpr (PG > 1) {
    float* const sm = reinterpret_cast<float*>(v0);  // [2][PG][kRows]
    float* const so = reinterpret_cast<float*>(k0);  // [PG][RG][16][kPart]
    constexpr int kPart = PG * D / 4, kParts = D / kPart;
    // 16 bytes c of a row sit in slot c ^ (row mod 8), a row's lanes in other banks
    auto so_at = [&](int g, int c) {
      return so + ((g * RG + rg) * 16 + c16) * kPart + 4 * (c ^ (c16 & 7));
    };
    __syncthreads();
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const int r = 16 * (T * rg + j) + c16;
      if (grp == 0) {
        sm[pg * kRows + r] = m[j];
        sm[(PG + pg) * kRows + r] = l[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < T; ++j) {
      const int r = 16 * (T * rg + j) + c16;
      float M = -__builtin_inff(), L = 0.0f;
#pragma unroll
      for (int g = 0; g < PG; ++g) M = fmaxf(M, sm[g * kRows + r]);
      const float ref = M == -__builtin_inff() ? 0.0f : M;
#pragma unroll
      for (int g = 0; g < PG; ++g)
        L += sm[(PG + g) * kRows + r] * __builtin_amdgcn_exp2f(sm[g * kRows + r] - ref);
      const float w = __builtin_amdgcn_exp2f(m[j] - ref);
      m[j] = M;
      l[j] = L;
      f32x4 sum[D / 16 / PG];
#pragma unroll
      for (int part = 0; part < kParts; ++part) {
#pragma unroll
        for (int d = 0; d < kPart / 16; ++d)
          *reinterpret_cast<f32x4*>(so_at(pg, 4 * d + grp)) = o[j][kPart / 16 * part + d] * w;
        __syncthreads();
        constexpr int kMine = kPart / 16 / PG;  // of this part's pieces
#pragma unroll
        for (int dd = 0; dd < kMine; ++dd) {
          f32x4 s = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int g = 0; g < PG; ++g)
            s += *reinterpret_cast<const f32x4*>(so_at(g, 4 * (kMine * pg + dd) + grp));
          sum[kMine * part + dd] = s;
        }
        __syncthreads();
      }
#pragma unroll
      for (int d = 0; d < D / 16 / PG; ++d) o[j][d] = sum[d];
    }
  }
  // piece d of this wave's sums: dims 16 piece(d) .. + 15
  auto piece = [&](int d) {
    constexpr int kPer = PG * D / 4 / 16 / PG;  // a group's pieces of one part
    return d / kPer * (PG * D / 64) + kPer * pg + d % kPer;
  };
  constexpr int kDims = D / 16 / PG;  // pieces of 16 dims this wave writes
#pragma unroll
  for (int j = 0; j < T; ++j) {
    const int r = row0 + 16 * j + c16;
    if (r >= R) continue;
    if (A.splits > 1) {
      float* to = A.part + ((int64_t)(split * A.kv_heads + kvh) * R + r) * D + 4 * grp;
#pragma unroll
      for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4*>(to + 16 * piece(d)) = o[j][d];
      if (grp == 0 && pg == 0) {
        float* ml = A.part_ml + ((int64_t)kvh * R + r) * 2 * A.splits;
        ml[split] = m[j];
        ml[A.splits + split] = l[j];
      }
    } else {
      const int h = kvh * A.group + r - node[j] * A.group;
      uint32_t any = 0;
      for (int w = 1; w <= (A.n + 31) >> 5; ++w) any |= sees[16 * (T * rg + j) + c16][w];
      const bool none = any == 0;
      const float inv = 1.0f / l[j];
      uint16_t* to = A.out + (int64_t)node[j] * A.out_stride + h * D + 4 * grp;
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        const f32x4 x = o[j][d];
        const uint2 v = {pack_f16x2(x[0] * inv, x[1] * inv), pack_f16x2(x[2] * inv, x[3] * inv)};
        *reinterpret_cast<uint2*>(to + 16 * piece(d)) = none ? make_uint2(0, 0) : v;
      }
      if (grp == 0 && pg == 0 && A.lse)
        A.lse[(int64_t)node[j] * A.q_heads + h] =
            none ? -__builtin_inff() : kLn2 * (m[j] + __builtin_amdgcn_logf(l[j]));
    }
  }
}

}  // namespace

#define ATTN_TREE(D, RG, T)                                                \
  extern "C" __global__ __launch_bounds__(256, RG == 1 ? 1 : 2) void       \
      attn_tree_##D##_##RG##T(AttnTreeArgs A) {                            \
    attn_tree<D, RG, T>(A);                                                \
  }
ATTN_TREE(64, 1, 1)
ATTN_TREE(64, 2, 1)
ATTN_TREE(64, 4, 1)
ATTN_TREE(64, 4, 2)
ATTN_TREE(128, 1, 1)
ATTN_TREE(128, 2, 1)
ATTN_TREE(128, 4, 1)
ATTN_TREE(128, 4, 2)

// One wave per row: the splits' (m, l) one per lane (at most 64 splits), then
// sum_s O_s 2^(m_s - M), half a wave the even splits in order, the other half the
// odd ones, each lane D / 32 dims.  Bound by latency: everything that does not
// hang on the statistics is requested with them, 16 splits at a time after that
// (16384 slots, 28 splits: attention and merge 23.5 us before, 21.1 so).
namespace {
template <int D>
__device__ __forceinline__ void attn_merge(const AttnTreeArgs& A) {
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int R = A.n * A.group;
  const int kvh = blockIdx.y, r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= R) return;
  const int64_t row = (int64_t)kvh * R + r;
  const float* ml = A.part_ml + row * 2 * A.splits;
  const float ms = lane < A.splits ? ml[lane] : -__builtin_inff();
  const float ls = lane < A.splits ? ml[A.splits + lane] : 0.0f;
  typedef float Dims __attribute__((ext_vector_type(D / 32)));
  const int64_t step = (int64_t)A.kv_heads * R * D;
  const float* p = A.part + row * D + D / 32 * (lane & 31);
  constexpr int kAhead = 8;
  Dims v[kAhead];
  auto request = [&](int s0) {
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = s0 + 2 * k + half;
      v[k] = *reinterpret_cast<const Dims*>(p + (s < A.splits ? s : 0) * step);
    }
  };
  request(0);
  const int node = A.group == 1 ? r : (int)__umulhi((uint32_t)r, A.group_inv);
  const int h = kvh * A.group + r - node * A.group;
  const bool empty = row_empty(A, node);
  float M = ms;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) M = fmaxf(M, __shfl_xor(M, d));
  const float ref = M == -__builtin_inff() ? 0.0f : M;
  const float w = __builtin_amdgcn_exp2f(ms - ref);
  const float L = wave_sum(ls * w);
  Dims acc = 0.0f;
  for (int s0 = 0; s0 < A.splits; s0 += 2 * kAhead) {
    if (s0 > 0) request(s0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = s0 + 2 * k + half;
      const float x = __shfl(w, s & 63);
      acc = s < A.splits ? acc + v[k] * x : acc;
    }
  }
#pragma unroll
  for (int d = 0; d < D / 32; ++d) acc[d] += __shfl_xor(acc[d], 32);
  const float inv = 1.0f / L;
  if (half == 0) {
    uint16_t* to = A.out + (int64_t)node * A.out_stride + h * D + D / 32 * lane;
    uint32_t o[D / 64];
#pragma unroll
    for (int d = 0; d < D / 64; ++d)
      o[d] = empty ? 0u : pack_f16x2(acc[2 * d] * inv, acc[2 * d + 1] * inv);
    if constexpr (D == 128) *reinterpret_cast<uint2*>(to) = make_uint2(o[0], o[1]);
    else *reinterpret_cast<uint32_t*>(to) = o[0];
  }
  if (lane == 0 && A.lse)
    A.lse[(int64_t)node * A.q_heads + h] =
        empty ? -__builtin_inff() : kLn2 * (M + __builtin_amdgcn_logf(L));
}
}  // namespace
extern "C" __global__ __launch_bounds__(256) void attn_merge_64(AttnTreeArgs A) {
  attn_merge<64>(A);
}
extern "C" __global__ __launch_bounds__(256) void attn_merge_128(AttnTreeArgs A) {
  attn_merge<128>(A);
}

// ---------------------------------------------------- attention weights ----
//
// The scores of 32 slots and 16 rows are S^T = K Q^T as in the attention: lane
// (c16, grp) holds row c16's at slots 4 grp + e and 16 + 4 grp + e, adds
// exp2(s - lse) of every row tile to 8 sums, and the 16 lanes of a DPP row meet
// at the end.  K fragments come straight from memory (16 rows x 64 bytes a load)
// and are read once; the sums run in one fixed order.
namespace {

// One row as a lane's column: its query vector, log-sum-exp and the last slot it
// sees (-1: none).
template <int D>
struct WeightRow {
  f16x8 q[D / 32];
  float lse;  // base 2
  int last;

  // row r of the kv head (token r / group); src: the row of q that token has
  __device__ __forceinline__ void load(const WeightsArgs& A, int layer, int kvh, int r, int i,
                                       int src) {
    const int h = kvh * A.group + r - i * A.group;
    const bool ok = r < A.n * A.group && src >= 0 && src < A.rows;
    const int64_t at = ok ? src : 0;
    const uint16_t* p = A.q + layer * A.q_layer_stride + at * A.q_stride + (ok ? h : 0) * D +
                        8 * ((threadIdx.x & 63) >> 4);
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
      q[st] = __builtin_bit_cast(f16x8, load_global(reinterpret_cast<const u32x4*>(p + 32 * st)));
    const float x = A.lse[layer * A.lse_layer_stride + at * A.q_heads + (ok ? h : 0)];
    lse = x * kLog2e;
    last = ok && x != -__builtin_inff() ? A.len + i : -1;
  }
};

template <int D>
struct WeightKeys {
  f16x8 k[D / 32][2];
  // slots p0 .. p0 + 31; those behind `slots` repeat the last
  __device__ __forceinline__ void load(const uint16_t* base, int64_t row, int p0, int slots) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
      const int p = p0 + 16 * nt + (lane & 15);
      const uint16_t* from = base + (p < slots ? p : slots - 1) * row + 8 * (lane >> 4);
#pragma unroll
      for (int st = 0; st < D / 32; ++st)
        k[st][nt] = __builtin_bit_cast(
            f16x8, load_global(reinterpret_cast<const u32x4*>(from + 32 * st)));
    }
  }
};

// sum[e] += the weights of slots p0 + 16 (e / 4) + 4 grp + e mod 4
template <int D>
__device__ __forceinline__ void add_weights(const WeightRow<D>& R, const WeightKeys<D>& K, int p0,
                                            float scale, bool edge, float (&sum)[8]) {
  f32x4 sc[2];
#pragma unroll
  for (int st = 0; st < D / 32; ++st)
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
      sc[nt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
          K.k[st][nt], R.q[st], st == 0 ? (f32x4){0.0f, 0.0f, 0.0f, 0.0f} : sc[nt], 0, 0, 0);
  if (edge) {
    const int p = p0 + 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float w = __builtin_amdgcn_exp2f(fmaf(sc[e >> 2][e & 3], scale, -R.lse));
      sum[e] += p + 16 * (e >> 2) + (e & 3) <= R.last ? w : 0.0f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      sum[e] += __builtin_amdgcn_exp2f(fmaf(sc[e >> 2][e & 3], scale, -R.lse));
  }
}

// The lane's sums over all 16 rows; lanes c16 < 8 get that of slot
// 16 (c16 / 4) + 4 grp + c16 mod 4.
__device__ __forceinline__ float rows_sum(const float (&sum)[8]) {
  const int c16 = threadIdx.x & 15;
  float v = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float s = reduce_row16(sum[e]);
    v = c16 == e ? s : v;
  }
  return v;
}
__device__ __forceinline__ int sum_slot() {
  const int lane = threadIdx.x & 63, c16 = lane & 15;
  return 16 * (c16 >> 2) + 4 * (lane >> 4) + (c16 & 3);
}

__device__ __forceinline__ int weight_source(const WeightsArgs& A, int i) {
  return i >= A.n ? -1 : (A.path ? A.path[i] : i);
}

// Up to 16 NT rows, whose queries stay in registers: bound by the bytes of K,
// 5.0 TB/s (5 tokens, 16384 slots of 28 layers 194 us; 1 token, 1000 slots 15).
// A wave takes A.blocks consecutive blocks, the next one's keys requested before
// one is computed.
template <int D, int NT>
__device__ __forceinline__ void weights_add(const WeightsArgs& A) {
  const int lane = threadIdx.x & 63, c16 = lane & 15;
  const int kvh = blockIdx.y, layer = blockIdx.z;
  const int slots = A.len + A.n, nb = (slots + 31) >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int b0 = (4 * blockIdx.x + wave) * A.blocks;
  const int b1 = b0 + A.blocks < nb ? b0 + A.blocks : nb;
  if (b0 >= nb) return;
  const int64_t row = (int64_t)A.kv_heads * D;
  const uint16_t* kb = A.k + layer * A.max_seq * row + kvh * D;
  float* wb = A.weights + ((int64_t)layer * A.kv_heads + kvh) * A.max_seq;
  WeightKeys<D> keys[2];
  keys[0].load(kb, row, 32 * b0, slots);
  WeightRow<D> rows[NT];
  bool all = true;  // every row exists and counts
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = 16 * j + c16;
    const int i = A.group == 1 ? r : (int)__umulhi((uint32_t)r, A.group_inv);
    rows[j].load(A, layer, kvh, r, i, weight_source(A, i));
    all = all && rows[j].last >= 0;
  }
  const bool some = __builtin_amdgcn_ballot_w64(!all) != 0;
  auto block = [&](int b, const WeightKeys<D>& now, WeightKeys<D>& next) {
    if (b + 1 < b1) next.load(kb, row, 32 * b + 32, slots);
    const int p = 32 * b + sum_slot();
    const bool mine = c16 < 8 && p < slots;
    const float old = mine && p < A.len ? wb[p] : 0.0f;
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.0f;
#pragma unroll
    for (int j = 0; j < NT; ++j)
      add_weights<D>(rows[j], now, 32 * b, A.scale, some || 32 * b + 32 > A.len, sum);
    const float v = rows_sum(sum);
    if (mine) wb[p] = old + v;
  };
  for (int b = b0; b < b1; b += 2) {
    block(b, keys[0], keys[1]);
    if (b + 1 < b1) block(b + 1, keys[1], keys[0]);
  }
}

// Any number of rows: a workgroup holds the keys of 64 slots, its waves take the
// row tiles in turn (the next one's queries requested before one is computed)
// and meet in LDS.  Every wave needs all the keys, so they come by LDS, whole rows
// at a time: 256 tokens, 2047 slots of a layer 13.3 us against 15.8 with each wave's
// fragments (64 bytes of 16 rows a load) from memory, 4096 slots 18.0 against 21.8.
// The queries stay on that way: by LDS too 14.2.
template <int D>
__device__ __forceinline__ void weights_add_many(const WeightsArgs& A) {
  constexpr int kChunks = D / 8, kRowsPerPiece = 64 / kChunks, kPieces = D / 32;
  __shared__ int source[kTreeMax];
  __shared__ float part[4][64];
  __shared__ __attribute__((aligned(1024))) uint8_t kk[128 * D];
  const int t = threadIdx.x, lane = t & 63, c16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kvh = blockIdx.y, layer = blockIdx.z;
  const int slots = A.len + A.n, p0 = 64 * blockIdx.x;
  const int64_t row = (int64_t)A.kv_heads * D;
  const uint16_t* kb = A.k + layer * A.max_seq * row + kvh * D;
  float* wb = A.weights + ((int64_t)layer * A.kv_heads + kvh) * A.max_seq;
  // chunk c of slot r sits in place c ^ (r mod kChunks) of its row; slots behind the
  // last repeat it
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int r = kRowsPerPiece * (kPieces * wave + i) + lane / kChunks, p = p0 + r;
    const uint16_t* from = kb + (p < slots ? p : slots - 1) * row +
                           8 * ((lane % kChunks) ^ (r & (kChunks - 1)));
    __builtin_amdgcn_global_load_lds((const GLOBAL_AS void*)from,
                                     (LDS_AS void*)(kk + 1024 * (kPieces * wave + i)), 16, 0, 0);
  }
  source[t] = weight_source(A, t);
  wait_vm<0>();
  __syncthreads();
  const int tiles = (A.n * A.group + 15) >> 4;
  auto load = [&](int tile, WeightRow<D>& R) {
    const int r = 16 * tile + c16;
    const int i = A.group == 1 ? r : (int)__umulhi((uint32_t)r, A.group_inv);
    R.load(A, layer, kvh, r, i, i < A.n ? source[i] : -1);
  };
  WeightRow<D> rows[2];
  if (wave < tiles) load(wave, rows[0]);
  WeightKeys<D> keys[2];
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
      keys[x >> 1].k[st][x & 1] = *reinterpret_cast<const f16x8*>(
          kk + 2 * D * (16 * x + c16) + 16 * ((4 * st + grp) ^ (c16 & (kChunks - 1))));
  float sum[2][8];
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[x][e] = 0.0f;
  auto use = [&](const WeightRow<D>& R) {
    const bool edge = p0 + 64 > A.len || __builtin_amdgcn_ballot_w64(R.last < 0) != 0;
    add_weights<D>(R, keys[0], p0, A.scale, edge, sum[0]);
    add_weights<D>(R, keys[1], p0 + 32, A.scale, edge, sum[1]);
  };
  for (int tile = wave; tile < tiles; tile += 8) {
    if (tile + 4 < tiles) load(tile + 4, rows[1]);
    use(rows[0]);
    if (tile + 4 >= tiles) break;
    if (tile + 8 < tiles) load(tile + 8, rows[0]);
    use(rows[1]);
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const float v = rows_sum(sum[x]);
    if (c16 < 8) part[wave][32 * x + sum_slot()] = v;
  }
  __syncthreads();
  const int p = p0 + t;
  if (t < 64 && p < slots) {
    const float v = (part[0][t] + part[1][t]) + (part[2][t] + part[3][t]);
    wb[p] = p < A.len ? wb[p] + v : v;
  }
}

// The same for many slots: the four waves hold the keys of 32 slots each and share
// the row tiles, whose queries are copied into LDS one tile ahead: a query is read
// once per 128 slots, but the tiles come one behind another.  256 tokens, 16384 slots
// of a layer 42.1 us against 47.1 by weights_add_many, 2047 slots 29 against 13.3;
// 64 tokens, 2047 slots of 28 layers 46.2 against 53.8.
template <int D>
__device__ __forceinline__ void weights_add_stream(const WeightsArgs& A) {
  constexpr int kChunks = D / 8, kRowsPerPiece = 64 / kChunks;
  __shared__ int source[kTreeMax];
  __shared__ __attribute__((aligned(1024))) uint8_t q0[32 * D], q1[32 * D];
  const int t = threadIdx.x, lane = t & 63, c16 = lane & 15, grp = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int kvh = blockIdx.y, layer = blockIdx.z;
  const int slots = A.len + A.n, p0 = 128 * blockIdx.x + 32 * wave;
  const int64_t row = (int64_t)A.kv_heads * D;
  const uint16_t* kb = A.k + layer * A.max_seq * row + kvh * D;
  float* wb = A.weights + ((int64_t)layer * A.kv_heads + kvh) * A.max_seq;
  const int tiles = (A.n * A.group + 15) >> 4;
  source[t] = weight_source(A, t);
  WeightKeys<D> keys;
  keys.load(kb, row, p0, slots);
  __syncthreads();
  // row r of the kv head: its token, its row of q and lse (-1: none), its head
  auto find = [&](int r, int& i, int& h) {
    i = A.group == 1 ? r : (int)__umulhi((uint32_t)r, A.group_inv);
    const int src = i < A.n ? source[i] : -1;
    const bool ok = src >= 0 && src < A.rows;
    h = ok ? kvh * A.group + r - i * A.group : 0;
    return ok ? src : -1;
  };
  auto copy = [&](int tile, uint8_t* to) {
    const int q_row = kRowsPerPiece * wave + lane / kChunks;
    if (kRowsPerPiece * wave >= 16) return;
    int i, h;
    const int src = find(16 * tile + q_row, i, h);
    const uint16_t* from = A.q + layer * A.q_layer_stride +
                           (int64_t)(src < 0 ? 0 : src) * A.q_stride + h * D +
                           8 * ((lane % kChunks) ^ (q_row & (kChunks - 1)));
    __builtin_amdgcn_global_load_lds((const GLOBAL_AS void*)from, (LDS_AS void*)(to + 1024 * wave),
                                     16, 0, 0);
  };
  auto meta = [&](int tile, WeightRow<D>& R) {
    int i, h;
    const int src = find(16 * tile + c16, i, h);
    const float x =
        A.lse[layer * A.lse_layer_stride + (int64_t)(src < 0 ? 0 : src) * A.q_heads + h];
    R.lse = x * kLog2e;
    R.last = src >= 0 && x != -__builtin_inff() ? A.len + i : -1;
  };
  float sum[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) sum[e] = 0.0f;
  WeightRow<D> rows[2];
  auto round = [&](int tile, const uint8_t* now, uint8_t* next, WeightRow<D>& R, WeightRow<D>& S) {
    wait_vm<0>();
    __syncthreads();  // everyone's copies are there, and `next` has been read
    if (tile + 1 < tiles) {
      copy(tile + 1, next);
      meta(tile + 1, S);
    }
#pragma unroll
    for (int st = 0; st < D / 32; ++st)
      R.q[st] = *reinterpret_cast<const f16x8*>(now + 2 * D * c16 +
                                                16 * ((4 * st + grp) ^ (c16 & (kChunks - 1))));
    const bool edge = p0 + 32 > A.len || __builtin_amdgcn_ballot_w64(R.last < 0) != 0;
    add_weights<D>(R, keys, p0, A.scale, edge, sum);
  };
  copy(0, q0);
  meta(0, rows[0]);
  for (int tile = 0; tile < tiles; tile += 2) {
    round(tile, q0, q1, rows[0], rows[1]);
    if (tile + 1 < tiles) round(tile + 1, q1, q0, rows[1], rows[0]);
  }
  const int p = p0 + sum_slot();
  const float v = rows_sum(sum);
  if (c16 < 8 && p < slots) wb[p] = p < A.len ? wb[p] + v : v;
}

}  // namespace

#define WEIGHTS_ADD(D)                                                                      \
  extern "C" __global__ __launch_bounds__(256) void weights_add_##D##_1(WeightsArgs A) {    \
    weights_add<D, 1>(A);                                                                   \
  }                                                                                         \
  extern "C" __global__ __launch_bounds__(256) void weights_add_##D##_2(WeightsArgs A) {    \
    weights_add<D, 2>(A);                                                                   \
  }                                                                                         \
  extern "C" __global__ __launch_bounds__(256) void weights_add_##D##_4(WeightsArgs A) {    \
    weights_add<D, 4>(A);                                                                   \
  }                                                                                         \
  extern "C" __global__ __launch_bounds__(256) void weights_add_##D##_many(WeightsArgs A) { \
    weights_add_many<D>(A);                                                                 \
  }                                                                                         \
  extern "C" __global__ __launch_bounds__(256) void weights_add_##D##_stream(               \
      WeightsArgs A) {                                                                      \
    weights_add_stream<D>(A);                                                               \
  }
WEIGHTS_ADD(64)
WEIGHTS_ADD(128)

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

// One workgroup per layer and kv head.  The order number of the last slot that
// still fits is found in three digits (11, 11 and 10 bits): a histogram in LDS of
// the slots that agree in the digits before, then a count from its top down.  A
// wave holds consecutive slots, 64 at a time, up to E of them a lane in registers,
// so the places of the kept slots come from one prefix count over the waves and
// ballots: nothing depends on an order of arrival.  E = 0 reads the weights again
// for each of the five passes.
// Bound by the chain of barriers, then by the passes' instructions, all of a head on
// one CU: 601 slots of a layer (8 workgroups) 4.3 us, of 28 layers 2048 5.6, 16384
// 12.8 (20 where the weights come from memory), 30000 26.5, 48000 37.8; E = 0 by the re-reads, 60000 128, 100000 221.
namespace {
template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
// the sum over the lanes up to this one
__device__ __forceinline__ uint32_t scan_u32(uint32_t v) {
  v += dpp_u32<0x111>(v);       // row_shr 1, 2, 4, 8
  v += dpp_u32<0x112>(v);
  v += dpp_u32<0x114>(v);
  v += dpp_u32<0x118>(v);
  v += dpp_u32<0x142, 0xA>(v);  // lane 15 of rows 0 and 2 to the row behind
  v += dpp_u32<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
  return v;
}
// the sum of v[0 .. wave - 1], 16 words in LDS
__device__ __forceinline__ uint32_t waves_before(const uint32_t* v, int wave) {
  const int lane = threadIdx.x & 63;
  uint32_t x = lane < wave ? v[lane & 15] : 0u;
  x += dpp_u32<0x111>(x);
  x += dpp_u32<0x112>(x);
  x += dpp_u32<0x114>(x);
  x += dpp_u32<0x118>(x);
  return (uint32_t)__builtin_amdgcn_readlane((int)x, 15);
}

// the set bits of m below this lane, and base
__device__ __forceinline__ uint32_t bits_below(uint64_t m, uint32_t base) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)m, base));
}

template <int E, int kCopies>
__device__ __forceinline__ void cache_select(const SelectArgs& A) {
  constexpr int kBins = 2048;
  constexpr int kStep = E == 4 ? 1 : E ? 4 : 16;  // slots of a thread at a time
  // a lane counts in copy lane mod kCopies: equal weights meet in one word less often
  __shared__ __attribute__((aligned(16))) uint32_t hist[kCopies][kBins + 8];
  __shared__ uint32_t wave_sum_[16], wave_above[16], wave_equal[16];
  __shared__ uint32_t s_digit, s_left;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const float* w = A.weights + (int64_t)blockIdx.x * A.max_seq;
  int32_t* keep = A.keep + (int64_t)blockIdx.x * A.budget;
  const int first = A.sinks, last = A.len - A.recent;
  const int middle = A.budget - A.sinks - A.recent;
  for (int j = t; j < A.sinks; j += 1024) keep[j] = j;
  for (int j = t; j < A.recent; j += 1024) keep[A.budget - A.recent + j] = last + j;
  if (middle == 0) return;
  // this wave's slots: p0 + 64 e + lane, e < count; behind `last` number 0, the
  // lowest and in the last places, so that none of them is ever kept
  const int count = (((last - first + 1023) >> 10) + kStep - 1) / kStep * kStep;
  const int p0 = first + wave * 64 * count + lane;
  uint32_t own[E ? E : kStep];
#pragma unroll
  for (int e = 0; e < E; ++e)
    own[e] = e < count && p0 + 64 * e < last ? weight_order(w[p0 + 64 * e]) : 0u;
  // use(slot, number) for every slot of the wave in order
  auto each = [&](auto&& use) {
    if constexpr (E != 0) {
#pragma unroll
      for (int e0 = 0; e0 < E; e0 += kStep) {
        if (e0 >= count) break;
#pragma unroll
        for (int e = e0; e < e0 + kStep; ++e) use(p0 + 64 * e, own[e]);
      }
    } else {
      for (int e0 = 0; e0 < count; e0 += kStep) {
#pragma unroll
        for (int u = 0; u < kStep; ++u) {
          const int p = p0 + 64 * (e0 + u);
          const float x = w[p < last ? p : last - 1];
          own[u] = p < last ? weight_order(x) : 0u;
        }
#pragma unroll
        for (int u = 0; u < kStep; ++u) use(p0 + 64 * (e0 + u), own[u]);
      }
    }
  };
  uint32_t prefix = 0, need = (uint32_t)middle;
#pragma unroll
  for (int digit = 0; digit < 3; ++digit) {
    const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
    const int bits = digit == 2 ? 10 : 11;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) *reinterpret_cast<uint2*>(&hist[c][2 * t]) = make_uint2(0, 0);
    __syncthreads();
    each([&](int p, uint32_t o) {
      if (digit == 0 ? p < last : (o ^ prefix) >> (shift + bits) == 0)
        atomicAdd(&hist[lane % kCopies][(o >> shift) & ((1u << bits) - 1)], 1u);
    });
    __syncthreads();
    // thread t: bins 2047 - 2 t and 2046 - 2 t, counted from the top
    uint32_t c0 = 0, c1 = 0;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      const uint2 two = *reinterpret_cast<const uint2*>(&hist[c][2046 - 2 * t]);
      c0 += two.y;
      c1 += two.x;
    }
    uint32_t up = scan_u32(c0 + c1);  // of the threads up to this one
    if (lane == 63) wave_sum_[wave] = up;
    __syncthreads();
    up += waves_before(wave_sum_, wave);
    const uint32_t before = up - c0 - c1;
    if (before < need && need <= up) {
      const bool high = need <= before + c0;
      s_digit = high ? 2047 - 2 * t : 2046 - 2 * t;
      s_left = need - before - (high ? 0u : c0);
    }
    __syncthreads();
    prefix |= s_digit << shift;
    need = s_left;
  }
  // every slot above the bound, and the first `need` that equal it
  uint32_t above = 0, equal = 0;
  each([&](int, uint32_t o) {
    above += (uint32_t)__popcll(__ballot(o > prefix));
    equal += (uint32_t)__popcll(__ballot(o == prefix));
  });
  if (lane == 0) {
    wave_above[wave] = above;
    wave_equal[wave] = equal;
  }
  __syncthreads();
  above = waves_before(wave_above, wave);
  equal = waves_before(wave_equal, wave);
  each([&](int p, uint32_t o) {
    const uint64_t ma = __ballot(o > prefix), me = __ballot(o == prefix);
    const uint32_t a = bits_below(ma, above), q = bits_below(me, equal);
    if (o > prefix || (o == prefix && q < need)) keep[A.sinks + a + (q < need ? q : need)] = p;
    above += (uint32_t)__popcll(ma);
    equal += (uint32_t)__popcll(me);
  });
}
}  // namespace
extern "C" __global__ __launch_bounds__(1024) void cache_select_4(SelectArgs A) {
  cache_select<4, 1>(A);
}
extern "C" __global__ __launch_bounds__(1024) void cache_select_16(SelectArgs A) {
  cache_select<16, 4>(A);
}
extern "C" __global__ __launch_bounds__(1024) void cache_select_48(SelectArgs A) {
  cache_select<48, 4>(A);
}
extern "C" __global__ __launch_bounds__(1024) void cache_select_any(SelectArgs A) {
  cache_select<0, 4>(A);
}

// ----------------------------------------------------------- compaction ----

// One workgroup per part and range of the kept slots, kv head and layer: parts 0 ..
// head_dim / 64 - 1 move 128 bytes of every k row, the next head_dim / 64 the same
// of v, the last one the weights.  A workgroup walks its slots in order, 256 (of
// the weights 2048) at a time, and waits until all of them are read before it
// writes.  Source and destination may be one (then with one range): keep ascends
// strictly, so keep[j] - j never falls, and the entries that move a slot up
// (keep[j] < j, which takes negative ones in front) come before those that do not.
// The latter are walked upwards, where a write never meets a slot still to be read,
// the former, if there are any, downwards; neither part reads or writes a slot of
// the other's.
// Bound by the bytes moved, 128 at a time from scattered slots: 28 layers, 4096 of
// 16384 slots 192 us, 4.9 TB/s read and written, in place 199; 1024 of 2048 51, over
// and over 43 and in place 32; 512 of one layer 3.6 (two rounds).
extern "C" __global__ __launch_bounds__(256) void cache_compact_k(CompactArgs A) {
  constexpr int U = 8;
  const int t = threadIdx.x;
  const int halves = A.head_dim / 64;
  const int parts = 2 * halves + (A.w ? 1 : 0);
  const int part = blockIdx.x % parts, range = blockIdx.x / parts;
  const int kvh = blockIdx.y, layer = blockIdx.z;
  const int head = layer * A.kv_heads + kvh;
  const int32_t* keep = A.keep + (A.per_head ? (int64_t)head * A.count : 0);
  const int64_t src_left = A.src_seq - A.base;
  const int j_lo = range * A.range;
  const int j_hi = j_lo + A.range < A.count ? j_lo + A.range : A.count;
  const int lead = A.in_place ? keep[0] : 0;
  // the number of entries that move a slot up
  auto moved_up = [&] {
    int lo = 0, hi = A.count;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (keep[mid] < mid) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  if (part == 2 * halves) {
    const float* from = A.w + (int64_t)head * A.src_seq + A.base;
    float* to = A.w_to + (int64_t)head * A.dst_seq + A.base;
    auto round = [&](int j0, int hi, bool up) {
      float x[U];
      bool ok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + 256 * u + t;
        const int p = j < hi ? keep[j] : -1;
        ok[u] = p >= (A.in_place && !up ? j : 0) && p < src_left;
        x[u] = from[ok[u] ? p : 0];  // (slot base is there: count > 0)
      }
#pragma unroll
      for (int u = 0; u < U; ++u) asm volatile("" : "+v"(x[u]));  // the loads are back
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (ok[u]) to[j0 + 256 * u + t] = x[u];
    };
    for (int j0 = j_lo; j0 < j_hi; j0 += 256 * U) round(j0, j_hi, false);
    if (lead < 0) {
      const int up = moved_up();
      for (int j0 = (up - 1) / (256 * U) * (256 * U); j0 >= 0; j0 -= 256 * U) round(j0, up, true);
    }
    return;
  }
  const int64_t row = (int64_t)A.kv_heads * A.head_dim;
  const int col = kvh * A.head_dim + 64 * (part % halves) + 8 * (t & 7);
  const uint16_t* from = (part < halves ? A.k : A.v) + (layer * A.src_seq + A.base) * row + col;
  uint16_t* to = (part < halves ? A.k_to : A.v_to) + (layer * A.dst_seq + A.base) * row + col;
  // rounds j0, j0 + step .. that start in [lo, hi)
  auto walk = [&](int lo, int hi, int j0, int step, bool up) {
    int next[U];
    auto places = [&] {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + 32 * u + (t >> 3);
        next[u] = j >= lo && j < hi ? keep[j] : -1;
      }
    };
    places();
    while (j0 >= lo && j0 < hi) {
      const int now = j0 + (t >> 3);
      u32x4 x[U];
      bool ok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ok[u] = next[u] >= (A.in_place && !up ? now + 32 * u : 0) && next[u] < src_left;
        x[u] = load_global(reinterpret_cast<const u32x4*>(from + (ok[u] ? next[u] : 0) * row));
      }
      j0 += step;
      places();
#pragma unroll
      for (int u = 0; u < U; ++u) asm volatile("" : "+v"(x[u]));  // the loads are back
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (ok[u]) *reinterpret_cast<u32x4*>(to + (now + 32 * u) * row) = x[u];
    }
  };
  walk(j_lo, j_hi, j_lo, 32 * U, false);
  if (lead < 0) {
    const int up = moved_up();
    walk(0, up, (up - 1) / (32 * U) * (32 * U), -32 * U, true);
  }
}

// ------------------------------------------------------ vocabulary rows ----
//
// Logits^T = W X^T, a tile of 128 vocabulary rows and all tokens (64 MS) per
// workgroup and round, eight waves 2 (rows) x 4 (tokens) of 64 x 16 MS, one chain
// of v_mfma_f32_16x16x32_f16 over K for every output.  The matrix is read from
// memory once; the bound is its bytes up to about 128 tokens, its bytes and the
// logits' beyond.  A stage is 64 k of the tile's W rows and of the X rows (those
// out of L2), copied straight into one of NBUF LDS buffers NBUF - 1 stages ahead,
// on into the workgroup's next tile, so that only its first tile waits for
// memory.  Lane (c16, g) holds rows 4 g + e of token c16: 8 bytes of logits a
// store, and the token's best row in two registers.  151,936 rows: 13 tokens 56 us
// (5.6 TB/s), 256 tokens 118 (675 TFLOP/s; 17 of them the logits, which all
// workgroups store at once; 134-140 under a profiler).
namespace {

// byte offset of row r's 16-byte chunk c (of 8) in a stage: two rows a 256-byte
// line, position p of the 16 in slot p ^ (line mod 16), so that neither the 16
// rows of a fragment read nor the copies meet in a bank
__device__ __forceinline__ int stage_off(int r, int c) {
  const int line = r >> 1;
  return 256 * line + 16 * ((((r & 1) << 3) | c) ^ (line & 15));
}

template <int MS, int NBUF>
__device__ __forceinline__ void gemm_argmax(const GemmArgmaxArgs& A) {
  constexpr int BM = 64 * MS, BN = 128, NS = 4;
  constexpr int kStages = kHidden / 64;
  constexpr int kBuf = (BM + BN) * 128;
  constexpr int J = kBuf / 1024 / 8;  // copies of a wave and stage
  static_assert(BM % 64 == 0 && kBuf % 8192 == 0, "copy pieces");
  __shared__ __attribute__((aligned(1024))) uint8_t b0[kBuf];
  __shared__ __attribute__((aligned(1024))) uint8_t b1[kBuf];
  __shared__ __attribute__((aligned(1024))) uint8_t b2[kBuf];
  __shared__ __attribute__((aligned(1024))) uint8_t b3[NBUF > 3 ? kBuf : 16];
  // the buffer of a stage s = I (mod NBUF); a table of them would hide from the
  // compiler which one a copy fills
  auto buf = [&](auto i) -> uint8_t* {
    constexpr int I = decltype(i)::value % NBUF;
    if constexpr (I == 0) return b0;
    else if constexpr (I == 1) return b1;
    else if constexpr (I == 2) return b2;
    else return b3;
  };
  const int t = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int lane = t & 63, c16 = lane & 15, g = lane >> 4;
  const int wr = wave & 1, wt = wave >> 1;  // rows, tokens
  const int wgs = (int)launch_wgs();
  const int tiles = (A.rows + BN - 1) / BN;
  const int mine = (tiles - (int)blockIdx.x + wgs - 1) / wgs;  // tiles of this workgroup
  const int total = mine * kStages;

  // Copy j of this wave fills lines 4 (J wave + j) .. + 3 of a buffer (W rows
  // first, then X rows); at: its lane's bytes from the tile's (X: matrix's) start.
  uint32_t at[J];
  int w_row[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int line = 4 * (J * wave + j) + (lane >> 4);
    const int p = (lane & 15) ^ (line & 15);
    const int row = 2 * line + (p >> 3);
    w_row[j] = row;
    int r = row;
    if (row >= BN) r = row - BN < A.n ? row - BN : A.n - 1;
    at[j] = (uint32_t)r * (2 * kHidden) + 16 * (p & 7);
  }
  // Every step copies a stage, the last ones the last stage once more: then one
  // wait count serves them all.
  auto issue = [&](int stage, uint8_t* to) {
    const int s = stage < total ? stage : total - 1;
    const int tile = (int)blockIdx.x + (s / kStages) * wgs, k = s % kStages;
    const uint8_t* wp = reinterpret_cast<const uint8_t*>(A.w) + (int64_t)tile * BN * 2 * kHidden + 128 * k;
    const uint8_t* xp = reinterpret_cast<const uint8_t*>(A.x) + 128 * k;
    const int last = A.rows - 1 - tile * BN;  // of the tile's rows
#pragma unroll
    for (int j = 0; j < J; ++j) {
      // a piece of 8 rows is all W or all X
      const bool is_w = 8 * (J * wave + j) < BN;
      uint32_t o = at[j];
      if (is_w && last < BN - 1 && w_row[j] > last) o -= (uint32_t)(w_row[j] - last) * (2 * kHidden);
      __builtin_amdgcn_global_load_lds((const GLOBAL_AS void*)((is_w ? wp : xp) + o),
                                       (LDS_AS void*)(to + 1024 * (J * wave + j)), 16, 0, 0);
    }
  };
  // fragments: row base + c16, chunk 4 kb + g
  int off[2][2];
#pragma unroll
  for (int hb = 0; hb < 2; ++hb)
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
      off[hb][kb] = stage_off(16 * hb + c16, 4 * kb + g) - 2048 * hb;
  int off_x[2];  // MS = 1: the wave's X rows start at an odd half for odd wt
#pragma unroll
  for (int kb = 0; kb < 2; ++kb)
    off_x[kb] = stage_off(16 * (wt & 1) + c16, 4 * kb + g) - 2048 * (wt & 1);
  f32x4 acc[NS][MS];
  auto clear = [&] {
#pragma unroll
    for (int ns = 0; ns < NS; ++ns)
#pragma unroll
      for (int ms = 0; ms < MS; ++ms) acc[ns][ms] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  };
  clear();
  float best[MS];
  int best_row[MS];
#pragma unroll
  for (int ms = 0; ms < MS; ++ms) {
    best[ms] = -__builtin_inff();
    best_row[ms] = -1;
  }
  auto finish = [&](int tile) {
    const int r0 = tile * BN + 64 * wr + 4 * g;  // + 16 ns + e
#pragma unroll
    for (int ms = 0; ms < MS; ++ms) {
      const int tok = 16 * (MS * wt + ms) + c16;
#pragma unroll
      for (int ns = 0; ns < NS; ++ns) {
        const int r = r0 + 16 * ns;
        const uint2 v = {pack_f16x2(acc[ns][ms][0], acc[ns][ms][1]),
                         pack_f16x2(acc[ns][ms][2], acc[ns][ms][3])};
        const uint16_t h[4] = {(uint16_t)v.x, (uint16_t)(v.x >> 16), (uint16_t)v.y,
                               (uint16_t)(v.y >> 16)};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = f16_bits_to_f32(h[e]);
          const bool up = x > best[ms] && r + e < A.rows;
          best[ms] = up ? x : best[ms];
          best_row[ms] = up ? r + e : best_row[ms];
        }
        if (A.logits && tok < A.n) {
          uint16_t* to = A.logits + (int64_t)tok * A.rows + r;
          if (A.whole8 && r + 4 <= A.rows) {
            *reinterpret_cast<uint2*>(to) = v;
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (r + e < A.rows) to[e] = h[e];
          }
        }
      }
    }
    clear();
  };
  auto step = [&](int s, const uint8_t* cur, uint8_t* refill) {
    // the copies of stage s have landed, those of the NBUF - 2 behind it may be out
    wait_vm<J * (NBUF - 2)>();
    wait_lds();  // this wave's reads of the buffer that is filled next
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue(s + NBUF - 1, refill);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      f16x8 wf[NS], xf[MS];
#pragma unroll
      for (int ns = 0; ns < NS; ++ns)
        wf[ns] = *reinterpret_cast<const f16x8*>(cur + (64 * wr + 16 * ns) * 128 + off[ns & 1][kb]);
#pragma unroll
      for (int ms = 0; ms < MS; ++ms)
        xf[ms] = *reinterpret_cast<const f16x8*>(cur + (BN + 16 * (MS * wt + ms)) * 128 +
                                                 (MS == 1 ? off_x[kb] : off[ms & 1][kb]));
#pragma unroll
      for (int ns = 0; ns < NS; ++ns)
#pragma unroll
        for (int ms = 0; ms < MS; ++ms)
          acc[ns][ms] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wf[ns], xf[ms], acc[ns][ms], 0, 0, 0);
    }
    if (s % kStages == kStages - 1 && s < total) finish((int)blockIdx.x + (s / kStages) * wgs);
  };
  using std::integral_constant;
  auto step_at = [&](auto i, int s) {
    constexpr int I = decltype(i)::value;
    step(s + I, buf(i), buf(integral_constant<int, I + NBUF - 1>{}));
  };
  issue(0, b0);
  issue(1, b1);
  if constexpr (NBUF > 3) issue(2, b2);
  // (with three buffers up to two steps too many, whose sums nobody reads)
  for (int s = 0; s < total; s += NBUF) {
    step_at(integral_constant<int, 0>{}, s);
    step_at(integral_constant<int, 1>{}, s);
    step_at(integral_constant<int, 2>{}, s);
    if constexpr (NBUF > 3) step_at(integral_constant<int, 3>{}, s);
  }
  wait_vm<0>();

  // a token's candidates: four lanes of each of the two row waves
  __syncthreads();
  uint64_t* const keys = reinterpret_cast<uint64_t*>(b0);  // [8][BM]
#pragma unroll
  for (int ms = 0; ms < MS; ++ms)
    keys[(4 * wr + g) * BM + 16 * (MS * wt + ms) + c16] =
        best_row[ms] >= 0 ? argmax_key(best[ms], best_row[ms]) : 0;
  __syncthreads();
  for (int i = t; i < A.n; i += 512) {
    uint64_t key = 0;
#pragma unroll
    for (int v = 0; v < 8; ++v) key = keys[v * BM + i] > key ? keys[v * BM + i] : key;
    A.part[(int64_t)i * wgs + blockIdx.x] = key;
  }
}

}  // namespace

extern "C" __global__ __launch_bounds__(512) void gemm_argmax_64(GemmArgmaxArgs A) {
  gemm_argmax<1, 4>(A);
}
extern "C" __global__ __launch_bounds__(512) void gemm_argmax_128(GemmArgmaxArgs A) {
  gemm_argmax<2, 4>(A);
}
extern "C" __global__ __launch_bounds__(512) void gemm_argmax_256(GemmArgmaxArgs A) {
  gemm_argmax<4, 3>(A);
}

// tokens[i] from the workgroups' keys (argmax_key: the larger value, then the
// lower row; 0: none): a launch and one round trip, 4-5 us
extern "C" __global__ __launch_bounds__(64) void gemm_argmax_final(
    const uint64_t* __restrict__ part, int wgs, int32_t* __restrict__ tokens) {
  const int i = blockIdx.x;
  uint64_t key = 0;
  for (int g = threadIdx.x; g < wgs; g += 64) {
    const uint64_t k = part[(int64_t)i * wgs + g];
    key = k > key ? k : key;
  }
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t k = __shfl_xor((unsigned long long)key, d);
    key = k > key ? k : key;
  }
  if (threadIdx.x == 0)
    tokens[i] = key == 0 ? -1 : (int32_t)(0xffffffffu - (uint32_t)(key & 0xffffffffu));
}
