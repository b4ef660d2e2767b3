// Attention of few query rows over the 4-bit cache: decoding, drafted tokens,
// shared kv heads.  All queries of one kv head that fit in 8 rows are one block
// of work (more rows: more blocks).
//
// What bounds it: the cache is read once, 5 bits per element (D / 2 bytes of
// codes and D / 8 of scales per row for k and again for v), so the floor is HBM
// bandwidth; the work per byte is the conversion of 4-bit codes to bf16
// operands, 1.5 instructions per element.  Hence:
//   * the codes become matrix operands in registers (mma.sync m16n8k16): the
//     tensor cores take the dot products off the fp32 pipe, and the dequantised
//     tile is never stored.  tcgen05 takes operands from shared memory only,
//     which would add a store and a barrier per element for a product whose 8
//     useful rows leave that unit idle either way.
//   * scores: A = queries (rows 0-7), B = 8 cache rows.  The contraction order is
//     free, so lane t of a quad owns whole 16-byte pieces of a row.
//   * output: A = probabilities, B = v.  A probability is split into two bf16
//     numbers, hi + lo; hi goes in A's rows 0-7 and lo in rows 8-15, which are idle
//     otherwise, so P carries 16 significant bits at no cost.
//   * each warp streams its own 32-row tiles through a private ring of
//     shared-memory stages (cp.async), with no CTA barrier until the end.
//   * the long axis is split over the warps of a CTA and the CTAs of a cluster;
//     partial results join in shared memory, across the cluster by distributed
//     shared memory: one launch, no workspace.
// The softmax runs online: running maximum and sum in fp32, log2 units.
#include <cooperative_groups.h>

#include "kv4_mma.cuh"
#include "launch.h"

namespace hrm {
namespace {

namespace cg = cooperative_groups;

constexpr int kTileRows = 32;
constexpr int kWarps = 4;
constexpr int kStages = 3;
constexpr int kBlockRows = 8;  // query rows per block

template <int D>
struct Shape {
  static constexpr int kCodeBytes = D / 2;             // per row
  static constexpr int kGroups = D / kKv4Group;        // words of scales per row
  static constexpr int kStageBytes = kTileRows * 2 * (kCodeBytes + 4 * kGroups);
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  // After the loop the ring holds the partial results of each warp.
  static constexpr int kPartial = kWarps * kBlockRows * D * 4;
  static constexpr int kSmem = (kRing > kPartial ? kRing : kPartial);
  static constexpr int kLaneWords = D / 32;  // 32-bit words of k codes per lane and row
};

// Where tile row r of k goes: the mma's column 2t + e of an 8-row tile is row
// t + 4e, so that the rows of a lane's probabilities are 4 apart and a warp's
// reads of v cover 4 adjacent rows.
__device__ __forceinline__ int k_place(int r) { return (r & ~7) | ((r & 3) << 1) | ((r >> 2) & 1); }
// 16-byte piece c of row r of v, moved so that 4 adjacent rows' pieces lie in different banks.
template <int D>
__device__ __forceinline__ int v_piece(int r, int c) {
  return D == 128 ? c ^ (r & 2) : (D == 256 ? c ^ ((r & 3) << 1) : c);
}
// Index of the k word that lane t owns as its i-th: 16-byte pieces i/4 * 4 + t,
// and for D = 64 and 192 a last 8-byte one.
template <int D>
__device__ __forceinline__ int k_word(int i, int t) {
  constexpr int kWhole = Shape<D>::kLaneWords / 4 * 4;
  return i < kWhole ? (i / 4) * 16 + 4 * t + i % 4 : kWhole * 4 + 2 * t + (i - kWhole);
}

template <int D>
__device__ __forceinline__ void load_tile(uint32_t stage, const Kv4View& c, int64_t head_row, int first, int limit,
                                          int lane) {
  using T = Shape<D>;
  constexpr int kPieces = T::kCodeBytes / 16;
  constexpr int kScaleUnit = D % 128 == 0 ? 16 : 8;
  constexpr int kScalePieces = 4 * T::kGroups / kScaleUnit;
  const uint32_t kc = stage, vc = stage + kTileRows * T::kCodeBytes;
  const uint32_t ks = stage + 2 * kTileRows * T::kCodeBytes, vs = ks + kTileRows * 4 * T::kGroups;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int idx = i * 32 + lane, r = idx / kPieces, p = idx % kPieces;
    const bool ok = first + r < limit;
    const int64_t at = (head_row + (ok ? first + r : 0)) * T::kCodeBytes + 16 * p;
    cp_async_zfill<16>(kc + k_place(r) * T::kCodeBytes + 16 * p, c.k_codes + at, ok);
    cp_async_zfill<16>(vc + r * T::kCodeBytes + 16 * v_piece<D>(r, p), c.v_codes + at, ok);
  }
#pragma unroll
  for (int i = 0; i < kScalePieces; ++i) {
    const int idx = i * 32 + lane, r = idx / kScalePieces, p = idx % kScalePieces;
    const bool ok = first + r < limit;
    const int64_t at = (head_row + (ok ? first + r : 0)) * T::kGroups + p * (kScaleUnit / 4);
    cp_async_zfill<kScaleUnit>(ks + k_place(r) * 4 * T::kGroups + p * kScaleUnit, c.k_scales + at, ok);
    cp_async_zfill<kScaleUnit>(vs + r * 4 * T::kGroups + p * kScaleUnit, c.v_scales + at, ok);
  }
}

// The two mma steps of one k word: 8 elements of 8 cache rows.
__device__ __forceinline__ void k_steps(float (&acc)[4], uint32_t w, uint32_t s2, uint32_t z2, const uint32_t* q) {
  mma_bf16(acc, q[0], 0, q[1], 0, fma_bf16x2(kv4_pair<0>(w), s2, z2), fma_bf16x2(kv4_pair<1>(w), s2, z2));
  mma_bf16(acc, q[2], 0, q[3], 0, fma_bf16x2(kv4_pair<2>(w), s2, z2), fma_bf16x2(kv4_pair<3>(w), s2, z2));
}

// Four output columns (elements P = 0..3 of a half word) for one 16-row step:
// `a` and `b` hold that half word of rows (0, 1) and (2, 3) of the lane.
template <int P>
__device__ __forceinline__ void v_step(float (*o)[4], uint32_t a, uint32_t b, const uint32_t (&s2)[2],
                                       const uint32_t (&z2)[2], const uint32_t (&p)[4]) {
  mma_bf16(o[P], p[0], p[1], p[2], p[3], fma_bf16x2(kv4_pair<P>(a), s2[0], z2[0]),
           fma_bf16x2(kv4_pair<P>(b), s2[1], z2[1]));
}

__device__ __forceinline__ float sigmoid_gate(uint16_t g) { return 1.0f / (1.0f + __expf(-bf16_to_f32(g))); }

template <int D>
__global__ void __launch_bounds__(kWarps * 32) kv4_decode_kernel(const AttnArgs a, const int splits) {
  using T = Shape<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][kBlockRows], s_l[kWarps][kBlockRows];
  __shared__ float c_m[kBlockRows], c_l[kBlockRows];  // this CTA's
  __shared__ uint32_t s_bad[kWarps][kBlockRows], c_bad[kBlockRows];
  grid_dependency_begin();

  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.x % splits;
  const int64_t rows = a.group * a.seq;  // query rows of one kv head
  const int64_t blocks = (rows + kBlockRows - 1) / kBlockRows;
  const int64_t item = blockIdx.x / splits;
  const int64_t bh = item / blocks, b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
  const int64_t row0 = (item - bh * blocks) * kBlockRows;
  const int nrows = (int)(rows - row0 < kBlockRows ? rows - row0 : kBlockRows);

  // the rows' limits; this lane's row is row0 + g
  __shared__ int s_limit[kBlockRows];
  int limit = 0, lowest = INT32_MAX, my_limit = 0;
  for (int r = 0; r < nrows; ++r) {
    const int l = visible_rows(a, b, (row0 + r) % a.seq);
    limit = max(limit, l);
    lowest = min(lowest, l);
    if (r == g) my_limit = l;
    if (threadIdx.x == r) s_limit[r] = l;
  }
  const int tiles = (limit + kTileRows - 1) / kTileRows;
  const int t0 = (int)((int64_t)tiles * rank / splits), t1 = (int)((int64_t)tiles * (rank + 1) / splits);
  const int64_t head_row = bh * a.c.cache_len;

  const uint32_t ring = smem_addr(smem) + warp * kStages * T::kStageBytes;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    const int tile = t0 + warp + i * kWarps;
    if (tile < t1) load_tile<D>(ring + i * T::kStageBytes, a.c, head_row, tile * kTileRows, limit, lane);
    cp_async_commit();
  }

  // queries as A operands: the words' 8 elements in the order in which kv4_pair yields them
  uint32_t q[T::kLaneWords][4];
  {
    const int64_t r = row0 + (g < nrows ? g : 0);
    const uint4* src = a.q + ((b * a.heads + hk * a.group + r / a.seq) * a.seq + r % a.seq) * (D / 8);
#pragma unroll
    for (int i = 0; i < T::kLaneWords; ++i) {
      uint4 v = ld_keep(src + k_word<D>(i, t));
      if (g >= nrows) v = make_uint4(0, 0, 0, 0);
      q[i][0] = __byte_perm(v.x, v.z, 0x5410);
      q[i][1] = __byte_perm(v.x, v.z, 0x7632);
      q[i][2] = __byte_perm(v.y, v.w, 0x5410);
      q[i][3] = __byte_perm(v.y, v.w, 0x7632);
    }
  }

  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  float m = -INFINITY, l = 0.0f;
  uint32_t bad = 0;  // groups of v that are not finite in a row that query g sees
  float* scores = nullptr;
  if (a.scores != nullptr && g < nrows) scores = a.scores + (bh * rows + row0 + g) * a.c.cache_len;

  int stage = 0;
  for (int tile = t0 + warp; tile < t1; tile += kWarps) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    const uint8_t* st = smem + (warp * kStages + stage) * T::kStageBytes;
    const uint8_t* kc = st;
    const uint8_t* vc = st + kTileRows * T::kCodeBytes;
    const uint32_t* ks = reinterpret_cast<const uint32_t*>(st + 2 * kTileRows * T::kCodeBytes);
    uint32_t* vs = reinterpret_cast<uint32_t*>(smem + (warp * kStages + stage) * T::kStageBytes +
                                               2 * kTileRows * T::kCodeBytes + kTileRows * 4 * T::kGroups);
    const int first = tile * kTileRows;

    // scores of 32 cache rows: c0, c1 of 8-row tile n are rows 8n + t and 8n + t + 4
    float acc[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
      const uint8_t* row = kc + (8 * n + g) * T::kCodeBytes;
      const uint32_t* sz = ks + (8 * n + g) * T::kGroups;
#pragma unroll
      for (int i = 0; i < T::kLaneWords / 4; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + 64 * i + 16 * t);
        const uint32_t x = sz[4 * i + t], s2 = kv4_scale2(x), z2 = kv4_base2(x);
        k_steps(acc[n], w.x, s2, z2, q[4 * i]);
        k_steps(acc[n], w.y, s2, z2, q[4 * i + 1]);
        k_steps(acc[n], w.z, s2, z2, q[4 * i + 2]);
        k_steps(acc[n], w.w, s2, z2, q[4 * i + 3]);
      }
      if (T::kLaneWords % 4) {
        constexpr int i = T::kLaneWords / 4;
        const uint2 w = *reinterpret_cast<const uint2*>(row + 64 * i + 8 * t);
        const uint32_t x = sz[4 * i + t / 2], s2 = kv4_scale2(x), z2 = kv4_base2(x);
        k_steps(acc[n], w.x, s2, z2, q[4 * i]);
        k_steps(acc[n], w.y, s2, z2, q[4 * i + 1]);
      }
    }

    float top = m;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = first + 8 * n + t + 4 * e;
        const float s = acc[n][e] * a.scale_log2;
        acc[n][e] = at < my_limit ? s : -INFINITY;
        if (scores != nullptr && at < my_limit) scores[at] = s;
        top = max_nan(top, acc[n][e]);
      }
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, 2));
    if (__any_sync(0xffffffffu, top != m)) {
      const float f = m == -INFINITY ? 0.0f : exp2_approx(m - top);
      l *= f;
#pragma unroll
      for (int j = 0; j < D / 8; ++j) {
        o[j][0] *= f;
        o[j][1] *= f;
        o[j][2] *= f;
        o[j][3] *= f;
      }
      m = top;
    }
    const float shift = m == -INFINITY ? 0.0f : m;

    // A row that some of the queries must not see, holding a value that is not
    // finite: 0 * NaN would reach them.  Such groups are read as zeros here and
    // the queries that do see them are marked.
    if (lowest < limit && first + kTileRows > lowest) {
      for (int r = 0; r < kTileRows; ++r) {
        const bool mine = lane < T::kGroups && kv4_not_finite(vs[r * T::kGroups + lane]);
        const uint32_t found = __ballot_sync(0xffffffffu, mine);
        if (mine) vs[r * T::kGroups + lane] = 0;
        if (first + r < my_limit) bad |= found;
      }
      __syncwarp();
    }

#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t p[4];  // hi and lo of columns (2t, 2t+1), then of (2t+8, 2t+9)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float p0 = exp2_approx(acc[2 * i + e][0] - shift), p1 = exp2_approx(acc[2 * i + e][1] - shift);
        l += p0 + p1;
        p[2 * e] = pack_bf16x2(p0, p1);
        p[2 * e + 1] = pack_bf16x2(p0 - bf16_lo(p[2 * e]), p1 - bf16_hi(p[2 * e]));
      }
      constexpr int kWords = D / 64;  // words of v codes per lane and row
      uint32_t w[4][kWords], sz[4][kWords];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * i + 4 * r + t;
        const uint8_t* base = vc + row * T::kCodeBytes;
        if (D == 64) {
          w[r][0] = *reinterpret_cast<const uint32_t*>(base + 4 * g);
        } else if (D == 128) {
          const uint2 x = *reinterpret_cast<const uint2*>(base + 16 * v_piece<D>(row, g >> 1) + 8 * (g & 1));
          w[r][0] = x.x;
          w[r][kWords > 1 ? 1 : 0] = x.y;
        } else if (D == 192) {
#pragma unroll
          for (int x = 0; x < kWords; ++x) w[r][x] = *reinterpret_cast<const uint32_t*>(base + 12 * g + 4 * x);
        } else {
          const uint4 x = *reinterpret_cast<const uint4*>(base + 16 * v_piece<D>(row, g));
#pragma unroll
          for (int y = 0; y < kWords; ++y) w[r][y] = vget(x, y);
        }
#pragma unroll
        for (int x = 0; x < kWords; ++x) sz[r][x] = vs[row * T::kGroups + (kWords * g + x) / 4];
      }
#pragma unroll
      for (int x = 0; x < kWords; ++x) {
        const uint32_t s2[2] = {__byte_perm(sz[0][x], sz[1][x], 0x5410), __byte_perm(sz[2][x], sz[3][x], 0x5410)};
        const uint32_t z2[2] = {__byte_perm(sz[0][x], sz[1][x], 0x7632), __byte_perm(sz[2][x], sz[3][x], 0x7632)};
        const uint32_t a0 = __byte_perm(w[0][x], w[1][x], 0x5410), b0 = __byte_perm(w[2][x], w[3][x], 0x5410);
        const uint32_t a1 = __byte_perm(w[0][x], w[1][x], 0x7632), b1 = __byte_perm(w[2][x], w[3][x], 0x7632);
        // the pairs of kv4_pair are nibbles P of both halves: element 8x + P (a0, b0) and 8x + 4 + P (a1, b1)
        const uint32_t pa[4] = {p[0], p[1], p[2], p[3]};
        v_step<0>(o + 8 * x, a0, b0, s2, z2, pa);
        v_step<1>(o + 8 * x, a0, b0, s2, z2, pa);
        v_step<2>(o + 8 * x, a0, b0, s2, z2, pa);
        v_step<3>(o + 8 * x, a0, b0, s2, z2, pa);
        v_step<0>(o + 8 * x + 4, a1, b1, s2, z2, pa);
        v_step<1>(o + 8 * x + 4, a1, b1, s2, z2, pa);
        v_step<2>(o + 8 * x + 4, a1, b1, s2, z2, pa);
        v_step<3>(o + 8 * x + 4, a1, b1, s2, z2, pa);
      }
    }

    __syncwarp();  // every lane is done with this stage's buffers
    const int next = tile + (kStages - 1) * kWarps;
    const int into = stage == 0 ? kStages - 1 : stage - 1;
    if (next < t1) load_tile<D>(ring + into * T::kStageBytes, a.c, head_row, next * kTileRows, limit, lane);
    cp_async_commit();
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();

  // ---- join the warps
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);  // [warp][row][D]
  if (t == 0) {
    s_m[warp][g] = m;
    s_l[warp][g] = l;
    s_bad[warp][g] = bad;
  }
  if (g < nrows) {
    float* dst = part + (warp * kBlockRows + g) * D + (D / 4) * t;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {  // lane t's columns 2t and 2t + 1 are D / 8 elements each
      dst[j] = o[j][0] + o[j][2];
      dst[D / 8 + j] = o[j][1] + o[j][3];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < nrows * D; e += kWarps * 32) {
    const int r = e / D, d = e % D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max_nan(top, s_m[w][r]);
    float sum = 0.0f, norm = 0.0f;
    uint32_t any = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s_m[w][r] == -INFINITY ? 0.0f : exp2_approx(s_m[w][r] - top);
      sum += f * part[(w * kBlockRows + r) * D + d];
      norm += f * s_l[w][r];
      any |= s_bad[w][r];
    }
    part[r * D + d] = sum;  // warp 0's element of the same thread's own (r, d)
    if (d == 0) {
      c_m[r] = top;
      c_l[r] = norm;
      c_bad[r] = any;
    }
  }
  cg::cluster_group cluster = cg::this_cluster();
  if (splits > 1)
    cluster.sync();
  else
    __syncthreads();

  // ---- join the cluster's CTAs; each writes its share of the output
  __shared__ float f_inv[kBlockRows], f_m[kBlockRows], f_w[16][kBlockRows];
  __shared__ uint32_t f_bad[kBlockRows];
  if (threadIdx.x < nrows) {
    const int r = threadIdx.x;
    float top = -INFINITY, sum = 0.0f;
    uint32_t any = 0;
    for (int x = 0; x < splits; ++x) top = max_nan(top, *cluster.map_shared_rank(&c_m[r], x));
    for (int x = 0; x < splits; ++x) {
      const float cm = *cluster.map_shared_rank(&c_m[r], x);
      const float f = cm == -INFINITY ? 0.0f : exp2_approx(cm - top);
      f_w[x][r] = f;
      sum += f * *cluster.map_shared_rank(&c_l[r], x);
      any |= *cluster.map_shared_rank(&c_bad[r], x);
    }
    f_m[r] = top;
    f_inv[r] = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing: 0
    f_bad[r] = any;
    if (a.lse != nullptr && rank == 0)
      a.lse[(b * a.heads + hk * a.group + (row0 + r) / a.seq) * a.seq + (row0 + r) % a.seq] =
          top == -INFINITY ? -INFINITY : top + log2f(sum);
  }
  __syncthreads();
  for (int e = rank * kWarps * 32 + threadIdx.x; e < nrows * (D / 2); e += splits * kWarps * 32) {
    const int r = e / (D / 2), d = 2 * (e % (D / 2));
    float x0 = 0.0f, x1 = 0.0f;
    for (int x = 0; x < splits; ++x) {
      const float2 v = *reinterpret_cast<const float2*>(cluster.map_shared_rank(part, x) + r * D + d);
      x0 += f_w[x][r] * v.x;
      x1 += f_w[x][r] * v.y;
    }
    x0 *= f_inv[r];
    x1 *= f_inv[r];
    if (f_bad[r] >> (d / kKv4Group) & 1u) x0 = x1 = __int_as_float(0x7fc00000);
    const int64_t h = hk * a.group + (row0 + r) / a.seq, s = (row0 + r) % a.seq;
    const int64_t at = ((b * a.seq + s) * a.heads + h) * D + d;
    if (a.gate != nullptr) {
      x0 *= sigmoid_gate(a.gate[at]);
      x1 *= sigmoid_gate(a.gate[at + 1]);
    }
    *reinterpret_cast<uint32_t*>(a.out + at) = pack_bf16x2(x0, x1);
  }

  // ---- add each cache row's probabilities to its weight: this CTA's rows, whose
  // scores this CTA wrote, summed over the query rows in order
  if (a.scores != nullptr) {
    const float* sc = a.scores + (bh * rows + row0) * a.c.cache_len;
    const int end = min(t1 * kTileRows, limit);
    for (int at = t0 * kTileRows + threadIdx.x; at < end; at += kWarps * 32) {
      float sum = 0.0f;
      for (int r = 0; r < nrows; ++r)
        if (at < s_limit[r])
          sum += exp2_approx(sc[(int64_t)r * a.c.cache_len + at] - f_m[r]) * f_inv[r];
      a.c.weights[head_row + at] += sum;
    }
  }
  if (splits > 1) cluster.sync();  // the shares are read: no CTA may leave before
}

template <int D>
cudaError_t launch_decode(const AttnArgs& a, int64_t longest, cudaStream_t s) {
  using T = Shape<D>;
  const int64_t items = a.batch * a.kv_heads * ((a.group * a.seq + kBlockRows - 1) / kBlockRows);
  // CTAs that fit on the GPU at once, by shared memory (228 KB per SM, 1 KB of it
  // reserved per CTA) and registers.
  const int per_sm = D <= 128 ? 3 : 1;
  const int64_t slots = (int64_t)device_sm_count() * per_sm;
  int splits = 1;
  while (splits < 8 && items * (splits + 1) <= slots && (int64_t)kTileRows * kWarps * (splits + 1) <= longest) ++splits;
  if (items * splits > INT32_MAX) return cudaErrorInvalidConfiguration;

  cudaError_t e = allow_shared(kv4_decode_kernel<D>, T::kSmem);
  if (e != cudaSuccess) return e;
  return launch_cluster(kv4_decode_kernel<D>, items * splits, kWarps * 32, T::kSmem, splits, s, a, splits);
}

}  // namespace

cudaError_t launch_kv4_decode(const AttnArgs& a, int64_t head_dim, int64_t longest, cudaStream_t s) {
  switch (head_dim) {
    case 64: return launch_decode<64>(a, longest, s);
    case 128: return launch_decode<128>(a, longest, s);
    case 192: return launch_decode<192>(a, longest, s);
    default: return launch_decode<256>(a, longest, s);
  }
}

}  // namespace hrm
