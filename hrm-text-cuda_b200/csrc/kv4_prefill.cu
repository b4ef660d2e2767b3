// Attention of many query rows over the 4-bit cache on tcgen05, head_dim 64 and
// 128: prompts and further turns of a chat.
//
// A CTA owns NQ x 128 query rows of one kv head and walks its share of the cache in
// tiles of 128 rows.  Three kinds of warps work at once, handing tiles over by
// mbarriers:
//   * 4 warps dequantise: codes and scales from global memory (the next tile's are
//     loaded while this one is converted), bf16 operands to shared memory, two
//     stages.  k is stored as it lies, [row][element]; v transposed, [element][row],
//     two cache rows' half words put together before the conversion, so that both
//     operands are K-major.
//   * one thread issues the products: S = Q K^T (128 x 128, accumulated in tensor
//     memory) and O += P V with P read from tensor memory, where it replaces S.
//     With NQ = 2 the products of one query tile run while the other's softmax does.
//   * 4 warps per query tile do the softmax, a thread per row: no shuffles.  O is
//     rescaled only when a row's maximum has grown by more than 8 (in log2 units)
//     since its last rescale: until then probabilities may be as large as 2^8,
//     which neither the bf16 P nor the fp32 sums mind.
// What bounds it: a tile costs 128 exponentials per row on a unit of 16 per clock,
// as long as its two products on the tensor cores; the conversion, 1.6 instructions
// per element, is a quarter of that for 256 query rows.
// P is rounded to bf16 (2^-8 of itself, the sum l is of the unrounded ones): the
// operand's type; the error it adds to an output is that of the output's own
// rounding at most.
// A long cache with few query tiles is split over CTAs; the partial results go to
// the workspace and kv4_prefill_join_kernel joins them.
#include "kv4_mma.cuh"
#include "launch.h"
#include "tcgen05.cuh"

namespace hrm {
namespace {

constexpr int kM = 128;  // query rows of a tile
constexpr int kN = 128;  // cache rows of a tile
constexpr float kSlack = 8.0f;

template <int D, int NQ>
struct Pre {
  static constexpr int kGroups = D / kKv4Group;
  static constexpr int kSoftmax = NQ * 128, kFill = 128;
  static constexpr int kThreads = kSoftmax + kFill + 32;
  static constexpr int kQ = 0, kQBytes = kM * D * 2;              // per query tile
  static constexpr int kK = NQ * kQBytes, kKBytes = kN * D * 2;   // per stage
  static constexpr int kV = kK + 2 * kKBytes, kVBytes = D * kN * 2;
  static constexpr int kSmem = kV + 2 * kVBytes + 1024;  // + alignment of the panels
  static constexpr uint32_t kColumns = NQ == 2 ? 512 : 256;  // S of each tile, then O of each
};

// Barriers, in order.
enum { kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPFull = 10, kOFull = 12, kBars = 14 };

struct PrefillSplit {
  int count;     // CTAs per item (kv head x block of query rows)
  float* parts;  // per (item, split): NQ * 128 rows of D sums, then the maxima, the sums and the masks
};
__host__ __device__ inline int64_t prefill_part(int nq, int64_t head_dim) { return nq * kM * (head_dim + 4); }

// Element x of a row's order of elements in shared memory: within 8, kv4_pair's order.
__device__ __forceinline__ uint4 paired_order(const uint4& v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                    __byte_perm(v.y, v.w, 0x7632));
}

// A filling thread's share of a tile: D / 32 pieces (16 bytes of codes, one group) of
// k, and one piece of 4 adjacent rows of v (D = 64: half the threads).  The lanes'
// rows are such that a warp's loads fill whole sectors and its stores fall into
// different banks.
template <int D>
struct Codes {
  static constexpr int kK = D / 32;
  uint4 k[kK], v[4];
  uint32_t ks[kK], vs[4];

  __device__ __forceinline__ static int k_row(int i, int t) { return (t >> 5) * 32 + i / (D / 64) * 16 + (t & 15); }
  __device__ __forceinline__ static int k_piece(int i, int t) { return i % (D / 64) * 2 + ((t >> 4) & 1); }
  __device__ __forceinline__ static bool v_works(int t) { return D == 128 || t < 64; }
  __device__ __forceinline__ static int v_quad(int t) { return ((t >> 5) & 1) * 16 + (t & 15); }
  __device__ __forceinline__ static int v_piece(int t) { return (t >> 6) * 2 + ((t >> 4) & 1); }

  // codes, scales: at the head's first row
  __device__ __forceinline__ void fetch_k(const uint8_t* codes, const uint32_t* scales, int first, int limit, int t) {
#pragma unroll
    for (int i = 0; i < kK; ++i) {
      const int row = first + k_row(i, t), p = k_piece(i, t);
      const bool in = row < limit;
      k[i] = in ? ld_l2(reinterpret_cast<const uint4*>(codes + (int64_t)row * (D / 2)) + p) : make_uint4(0, 0, 0, 0);
      ks[i] = in ? __ldcg(scales + (int64_t)row * (D / 32) + p) : 0u;
    }
  }
  __device__ __forceinline__ void fetch_v(const uint8_t* codes, const uint32_t* scales, int first, int limit, int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = first + 4 * v_quad(t) + i, p = v_piece(t);
      const bool in = v_works(t) && row < limit;
      v[i] = in ? ld_l2(reinterpret_cast<const uint4*>(codes + (int64_t)row * (D / 2)) + p) : make_uint4(0, 0, 0, 0);
      vs[i] = in ? __ldcg(scales + (int64_t)row * (D / 32) + p) : 0u;
    }
  }
  // bf16 k to the panels at dst, [row][element]
  __device__ __forceinline__ void store_k(uint8_t* dst, int t) const {
#pragma unroll
    for (int i = 0; i < kK; ++i) {
      const int row = k_row(i, t), p = k_piece(i, t);
      const uint32_t s2 = kv4_scale2(ks[i]), z2 = kv4_base2(ks[i]);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t x = vget(k[i], w);
        const int piece = 4 * p + w;
        *reinterpret_cast<uint4*>(dst + (piece / 8) * (kN * 128) + panel_piece(row, piece % 8)) =
            make_uint4(fma_bf16x2(kv4_pair<0>(x), s2, z2), fma_bf16x2(kv4_pair<1>(x), s2, z2),
                       fma_bf16x2(kv4_pair<2>(x), s2, z2), fma_bf16x2(kv4_pair<3>(x), s2, z2));
      }
    }
  }
  // bf16 v to the panels at dst, [element][row].  With `flags`, groups that are not
  // finite are stored as zeros and marked there.
  __device__ __forceinline__ void store_v(uint8_t* dst, int t, uint8_t (*flags)[4]) {
    if (!v_works(t)) return;
    const int q = v_quad(t), p = v_piece(t);
    if (flags != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool bad = kv4_not_finite(vs[i]);
        flags[4 * q + i][p] = bad;
        if (bad) vs[i] = 0;
      }
    }
    const uint32_t sa = __byte_perm(vs[0], vs[1], 0x5410), za = __byte_perm(vs[0], vs[1], 0x7632);
    const uint32_t sb = __byte_perm(vs[2], vs[3], 0x5410), zb = __byte_perm(vs[2], vs[3], 0x7632);
    uint8_t* panel = dst + (q / 16) * (D * 128) + 8 * (q & 1);
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int sel = h == 0 ? 0x5410 : 0x7632;
        const uint32_t xa = __byte_perm(vget(v[0], w), vget(v[1], w), sel), xb = __byte_perm(vget(v[2], w), vget(v[3], w), sel);
        const int d = 32 * p + 8 * w + 4 * h;
        auto put = [&](int e, uint32_t ya, uint32_t yb) {
          *reinterpret_cast<uint2*>(panel + panel_piece(d + e, (q & 15) / 2)) =
              make_uint2(fma_bf16x2(ya, sa, za), fma_bf16x2(yb, sb, zb));
        };
        put(0, kv4_pair<0>(xa), kv4_pair<0>(xb));
        put(1, kv4_pair<1>(xa), kv4_pair<1>(xb));
        put(2, kv4_pair<2>(xa), kv4_pair<2>(xb));
        put(3, kv4_pair<3>(xa), kv4_pair<3>(xb));
      }
  }
};

template <int D, int NQ>
__global__ void __launch_bounds__(Pre<D, NQ>::kThreads, 1)
    kv4_prefill_kernel(const AttnArgs a, const PrefillSplit split, const int blocks_q) {
  using T = Pre<D, NQ>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[kBars];
  __shared__ uint32_t s_tmem;
  __shared__ int s_limit[NQ * kM];
  __shared__ __align__(16) uint8_t s_bad[2][kN][4];  // per stage and cache row: groups of v that are not finite
  uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const uint32_t base = smem_addr(smem), bar0 = smem_addr(bars);
  auto bar = [&](int i) -> uint32_t { return bar0 + 8 * i; };
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int kMmaWarp = (T::kSoftmax + T::kFill) / 32;
  grid_dependency_begin();

  const unsigned rows = a.group * a.seq;
  const unsigned item = blockIdx.x / split.count;
  const int rank = (int)(blockIdx.x - item * split.count);
  const int bh = (int)(item / blocks_q), b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
  // the last rows first: under a causal mask they have the most tiles
  const unsigned row0 = (blocks_q - 1 - (item - bh * blocks_q)) * (NQ * kM);

  // ---- set-up: limits, queries, barriers, tensor memory
  for (int r = tid; r < NQ * kM; r += T::kThreads) {
    const unsigned row = row0 + r;
    s_limit[r] = row < rows ? visible_rows(a, b, row % a.seq) : -1;
  }
  {
    const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;  // the softmax takes |scale|
    const uint32_t keep = a.scale_log2 == 0.0f ? 0u : 0xffffffffu;  // scale 0: all scores 0
    for (int i = tid; i < NQ * kM * (D / 8); i += T::kThreads) {
      const int r = i / (D / 8), p = i % (D / 8);
      const unsigned row = row0 + r;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (row < rows) {
        const unsigned g = row / a.seq, s = row - g * a.seq;
        v = ld_keep(a.q + (((int64_t)b * a.heads + hk * a.group + g) * a.seq + s) * (D / 8) + p);
      }
      v = paired_order(v);
      v = make_uint4((v.x ^ flip) & keep, (v.y ^ flip) & keep, (v.z ^ flip) & keep, (v.w ^ flip) & keep);
      *reinterpret_cast<uint4*>(smem + (r / kM) * T::kQBytes + (p / 8) * (kM * 128) + panel_piece(r % kM, p % 8)) = v;
    }
  }
  for (int i = tid; i < 2 * kN; i += T::kThreads) *reinterpret_cast<uint32_t*>(s_bad[i / kN][i % kN]) = 0;
  if (warp == kMmaWarp) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(bar(kKFull + i), T::kFill);
        mbar_init(bar(kKEmpty + i), 1);
        mbar_init(bar(kVFull + i), T::kFill);
        mbar_init(bar(kVEmpty + i), 1);
        mbar_init(bar(kSFull + i), 1);
        mbar_init(bar(kPFull + i), kM);
        mbar_init(bar(kOFull + i), 1);
      }
      mbar_init_fence();
    }
    __syncwarp();
    tmem_alloc(smem_addr(&s_tmem), T::kColumns);
  }
  fence_proxy_async_smem();  // the queries, before the products read them
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  const uint32_t tmem = s_tmem;

  int limit = 0, lowest = INT32_MAX;
  for (int r = lane; r < NQ * kM; r += 32) {
    limit = max(limit, s_limit[r]);
    if (s_limit[r] >= 0) lowest = min(lowest, s_limit[r]);
  }
  limit = __reduce_max_sync(0xffffffffu, limit);
  lowest = __reduce_min_sync(0xffffffffu, lowest);
  const int tiles = (limit + kN - 1) / kN;
  const int j0 = (int)((int64_t)tiles * rank / split.count), j1 = (int)((int64_t)tiles * (rank + 1) / split.count);
  const int n = j1 - j0;

  if (warp < T::kSoftmax / 32) {
    // ---------------------------------------------------------------- softmax
    const int qt = warp / 4, r = qt * kM + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + lanes + qt * kN, o_at = tmem + lanes + NQ * kN + qt * D;
    const int lim = s_limit[r];
    const float scale = a.scale_log2 == 0.0f ? 1.0f : fabsf(a.scale_log2);
    float m = -INFINITY, l = 0.0f;  // m: of the unscaled scores, as of the last rescale
    uint32_t bad = 0;
    bool ok = true;
    for (int j = 0; j < n && ok; ++j) {
      const int first = (j0 + j) * kN;
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar(kSFull + qt), j & 1));
      if (!ok) break;
      tcgen05_after_sync();
      const bool whole = __all_sync(0xffffffffu, first + kN <= lim);  // no masked score in the warp's rows
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kN / 32; ++c) {
        uint32_t s[32];
        tmem_load32(s, s_at + 32 * c);
        tmem_wait_load();
        if (whole) {
          float x[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i & 3] = max_nan(x[i & 3], __uint_as_float(s[i]));
          top = max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3]));
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (first + 32 * c + i < lim) top = max_nan(top, __uint_as_float(s[i]));
        }
      }
      // Grown by more than the slack (or from nothing, or NaN): rescale.  S of this
      // tile is complete, so every product issued before it is, O's among them.
      const bool grown = !(top <= m + kSlack / scale);
      if (__any_sync(0xffffffffu, grown)) {
        const float to = grown ? max_nan(top, m) : m;
        const float f = m == -INFINITY ? 0.0f : exp2_approx((m - to) * scale);
        if (grown) {
          l *= f;
          m = to;
        }
        if (j > 0) {
          const float by = grown ? f : 1.0f;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_load32(o, o_at + 32 * c);
            tmem_wait_load();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
            tmem_store32(o_at + 32 * c, o);
          }
        }
      }
      const float shift = m == -INFINITY ? 0.0f : m * scale;
      float sum[2] = {0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < kN / 32; ++c) {
        uint32_t s[32], p[16];
        tmem_load32(s, s_at + 32 * c);
        tmem_wait_load();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x = exp2_approx(fmaf(__uint_as_float(s[2 * i]), scale, -shift));
          float y = exp2_approx(fmaf(__uint_as_float(s[2 * i + 1]), scale, -shift));
          if (!whole) {
            if (first + 32 * c + 2 * i >= lim) x = 0.0f;
            if (first + 32 * c + 2 * i + 1 >= lim) y = 0.0f;
          }
          sum[i & 1] += x + y;
          p[i] = pack_bf16x2(x, y);
        }
        tmem_store16(s_at + 16 * c, p);  // columns whose scores have been read
      }
      tmem_wait_store();
      tcgen05_before_sync();
      mbar_arrive(bar(kPFull + qt));
      l += sum[0] + sum[1];
      if (first + kN > lowest && lowest < limit) {
        // rows that some query must not see: the groups of v that are not finite were read as zeros
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar(kVFull + (j & 1)), (j >> 1) & 1));
        if (!ok) break;
        const uint4* flags = reinterpret_cast<const uint4*>(s_bad[j & 1]);
        for (int i = 0; i < kN / 4; ++i) {
          const uint4 f = flags[i];
          if ((f.x | f.y | f.z | f.w) == 0) continue;
#pragma unroll
          for (int w = 0; w < 4; ++w)
            if (first + 4 * i + w < lim) bad |= vget(f, w);
        }
      }
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar(kOFull + qt), 0));
    tcgen05_after_sync();
    const unsigned row = row0 + r;
    const unsigned g = row / a.seq, sq = row - g * a.seq;
    const int64_t head = hk * a.group + g;
    if (split.count == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (row < rows && a.lse != nullptr)
        a.lse[((int64_t)b * a.heads + head) * a.seq + sq] = m == -INFINITY ? -INFINITY : m * scale + log2f(l);
      const int64_t at = (((int64_t)b * a.seq + sq) * a.heads + head) * D;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_load32(o, o_at + 32 * c);
          tmem_wait_load();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0;
        }
        const bool nan = bad >> (8 * c) & 1u;
#pragma unroll
        for (int i = 0; i < 4 && row < rows && ok; ++i) {
          uint4 y, gate = make_uint4(0, 0, 0, 0);
          if (a.gate != nullptr) gate = ld_l2(reinterpret_cast<const uint4*>(a.gate + at + 32 * c) + i);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float v0 = __uint_as_float(o[8 * i + 2 * w]) * inv, v1 = __uint_as_float(o[8 * i + 2 * w + 1]) * inv;
            if (nan) v0 = v1 = __int_as_float(0x7fc00000);
            if (a.gate != nullptr) {
              v0 *= 1.0f / (1.0f + __expf(-bf16_lo(vget(gate, w))));
              v1 *= 1.0f / (1.0f + __expf(-bf16_hi(vget(gate, w))));
            }
            vset(y, w, pack_bf16x2(v0, v1));
          }
          st_l2(reinterpret_cast<uint4*>(a.out + at + 32 * c) + i, y);
        }
        __syncwarp();
      }
    } else {
      float* part = split.parts + (int64_t)blockIdx.x * prefill_part(NQ, D);
#pragma unroll 1
      for (int c = 0; c < D / 32 && n > 0; ++c) {
        uint32_t o[32];
        tmem_load32(o, o_at + 32 * c);
        tmem_wait_load();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          reinterpret_cast<uint4*>(part + (int64_t)r * D + 32 * c)[i] =
              make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
      }
      float* tail = part + NQ * kM * D + r;
      tail[0] = m == -INFINITY ? -INFINITY : m * scale;  // log2 units
      tail[NQ * kM] = l;
      tail[2 * NQ * kM] = __uint_as_float(bad);
    }
  } else if (warp < kMmaWarp) {
    // --------------------------------------------------------------- filling
    const int t = tid - T::kSoftmax;
    const int64_t head_row = (int64_t)bh * a.c.cache_len;
    const uint8_t* kc = a.c.k_codes + head_row * (D / 2);
    const uint8_t* vc = a.c.v_codes + head_row * (D / 2);
    const uint32_t* ks = a.c.k_scales + head_row * T::kGroups;
    const uint32_t* vs = a.c.v_scales + head_row * T::kGroups;
    Codes<D> c;
    if (n > 0) {
      c.fetch_k(kc, ks, j0 * kN, limit, t);
      c.fetch_v(vc, vs, j0 * kN, limit, t);
    }
    for (int j = 0; j < n; ++j) {
      const int first = (j0 + j) * kN, s = j & 1, phase = (j >> 1) & 1;
      if (!mbar_wait_bounded(bar(kKEmpty + s), phase ^ 1)) break;
      c.store_k(smem + T::kK + s * T::kKBytes, t);
      fence_proxy_async_smem();
      mbar_arrive(bar(kKFull + s));
      if (j + 1 < n) c.fetch_k(kc, ks, first + kN, limit, t);
      if (!mbar_wait_bounded(bar(kVEmpty + s), phase ^ 1)) break;
      const bool border = first + kN > lowest && lowest < limit;
      c.store_v(smem + T::kV + s * T::kVBytes, t, border ? s_bad[s] : nullptr);
      fence_proxy_async_smem();
      mbar_arrive(bar(kVFull + s));
      if (j + 1 < n) c.fetch_v(vc, vs, first + kN, limit, t);
    }
  } else if (lane == 0) {
    // -------------------------------------------------------------- products
    constexpr uint32_t kShapeS = mma_shape(kM, kN), kShapeO = mma_shape(kM, D);
    auto scores = [&](int q, int s) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t at = (k / 4) * (kM * 128) + 32 * (k % 4);
        tcgen05_mma(tmem + q * kN, panel_desc(base + T::kQ + q * T::kQBytes + at),
                    panel_desc(base + T::kK + s * T::kKBytes + at), kShapeS, k > 0);
      }
      tcgen05_commit(bar(kSFull + q));
    };
    bool ok = n > 0 && mbar_wait_bounded(bar(kKFull), 0);
    if (ok) {
      tcgen05_after_sync();
      for (int q = 0; q < NQ; ++q) scores(q, 0);
      tcgen05_commit(bar(kKEmpty));
    }
    for (int j = 0; j < n && ok; ++j) {
      const int s = j & 1, next = (j + 1) & 1;
      ok = mbar_wait_bounded(bar(kVFull + s), (j >> 1) & 1);
      for (int q = 0; q < NQ && ok; ++q) {
        ok = mbar_wait_bounded(bar(kPFull + q), j & 1);
        if (!ok) break;
        tcgen05_after_sync();
#pragma unroll
        for (int k = 0; k < kN / 16; ++k)
          tcgen05_mma_ta(tmem + NQ * kN + q * D, tmem + q * kN + 8 * k,
                         panel_desc(base + T::kV + s * T::kVBytes + (k / 4) * (D * 128) + 32 * (k % 4)), kShapeO,
                         j > 0 || k > 0);
        // the next scores replace P once it has been read: products run in the order of their issue
        if (j + 1 < n) {
          if (q == 0) ok = mbar_wait_bounded(bar(kKFull + next), ((j + 1) >> 1) & 1);
          if (!ok) break;
          tcgen05_after_sync();
          scores(q, next);
        } else {
          tcgen05_commit(bar(kOFull + q));
        }
      }
      if (!ok) break;
      tcgen05_commit(bar(kVEmpty + s));
      if (j + 1 < n) tcgen05_commit(bar(kKEmpty + next));
    }
  }
  __syncwarp();
  tcgen05_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) tmem_free(tmem, T::kColumns);
}

// Joins the split items' partial results: a warp per query row.
template <int D, int NQ>
__global__ void __launch_bounds__(256) kv4_prefill_join_kernel(const AttnArgs a, const PrefillSplit split,
                                                               const int blocks_q) {
  grid_dependency_begin();
  const unsigned rows = a.group * a.seq;
  const unsigned line = blockIdx.x * 8 + threadIdx.x / 32;  // item * 128 NQ + r
  const unsigned item = line / (NQ * kM), r = line % (NQ * kM);
  const int bh = (int)(item / blocks_q), b = bh / a.kv_heads, hk = bh - b * a.kv_heads, lane = threadIdx.x & 31;
  const unsigned row = (blocks_q - 1 - (item - bh * blocks_q)) * (NQ * kM) + r;
  if (row >= rows) return;
  const float* parts = split.parts + (int64_t)item * split.count * prefill_part(NQ, D);
  float top = -INFINITY, norm = 0.0f;
  uint32_t bad = 0;
  for (int i = 0; i < split.count; ++i) top = max_nan(top, parts[i * prefill_part(NQ, D) + NQ * kM * D + r]);
  float sum[D / 32];
#pragma unroll
  for (int x = 0; x < D / 32; ++x) sum[x] = 0.0f;
  for (int i = 0; i < split.count; ++i) {
    const float* part = parts + i * prefill_part(NQ, D);
    const float m = part[NQ * kM * D + r];
    if (m == -INFINITY) continue;
    const float f = exp2_approx(m - top);
    norm += f * part[NQ * kM * D + NQ * kM + r];
    bad |= __float_as_uint(part[NQ * kM * D + 2 * NQ * kM + r]);
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
      const float2 v = *reinterpret_cast<const float2*>(part + (int64_t)r * D + 64 * x + 2 * lane);
      sum[2 * x] += f * v.x;
      sum[2 * x + 1] += f * v.y;
    }
  }
  const unsigned g = row / a.seq, s = row - g * a.seq;
  const int64_t head = hk * a.group + g;
  if (a.lse != nullptr && lane == 0)
    a.lse[((int64_t)b * a.heads + head) * a.seq + s] = top == -INFINITY ? -INFINITY : top + log2f(norm);
  const float inv = norm == 0.0f ? 0.0f : 1.0f / norm;
  const int64_t at = (((int64_t)b * a.seq + s) * a.heads + head) * D;
#pragma unroll
  for (int x = 0; x < D / 64; ++x) {
    const int d = 64 * x + 2 * lane;
    float v0 = sum[2 * x] * inv, v1 = sum[2 * x + 1] * inv;
    if (bad >> (8 * (d / kKv4Group)) & 1u) v0 = v1 = __int_as_float(0x7fc00000);
    if (a.gate != nullptr) {
      const uint32_t y = *reinterpret_cast<const uint32_t*>(a.gate + at + d);
      v0 *= 1.0f / (1.0f + __expf(-bf16_lo(y)));
      v1 *= 1.0f / (1.0f + __expf(-bf16_hi(y)));
    }
    *reinterpret_cast<uint32_t*>(a.out + at + d) = pack_bf16x2(v0, v1);
  }
}

struct PrefillShape {
  int nq, blocks_q;
  int64_t items;
};
PrefillShape prefill_shape(int64_t batch_kv_heads, int64_t rows) {
  PrefillShape s;
  s.nq = rows > kM ? 2 : 1;
  s.blocks_q = (int)((rows + s.nq * kM - 1) / (s.nq * kM));
  s.items = batch_kv_heads * s.blocks_q;
  return s;
}

template <int D, int NQ>
cudaError_t launch_prefill(const AttnArgs& a, const PrefillShape& p, int64_t longest, float* parts, cudaStream_t s) {
  using T = Pre<D, NQ>;
  // One CTA per SM: items that leave SMs idle are split, to 4 tiles at least.
  PrefillSplit split{1, parts};
  while (p.items * (split.count + 1) <= device_sm_count() && (split.count + 1) * 4 * kN <= longest) ++split.count;
  if (p.items * split.count > INT32_MAX) return cudaErrorInvalidConfiguration;
  cudaError_t e = allow_shared<kv4_prefill_kernel<D, NQ>>(T::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_kernel(kv4_prefill_kernel<D, NQ>, p.items * split.count, T::kThreads, T::kSmem, s, a, split, p.blocks_q);
  if (e != cudaSuccess || split.count == 1) return e;
  return launch_kernel(kv4_prefill_join_kernel<D, NQ>, p.items * NQ * kM / 8, 256, 0, s, a, split, p.blocks_q);
}

}  // namespace

int64_t kv4_prefill_workspace(int64_t batch_kv_heads, int64_t rows, int64_t head_dim) {
  const PrefillShape p = prefill_shape(batch_kv_heads, rows);
  const int64_t most = device_sm_count() / (p.items > 0 ? p.items : 1);  // CTAs per item, for any cache length
  return most < 2 ? 0 : p.items * most * prefill_part(p.nq, head_dim) * (int64_t)sizeof(float);
}

cudaError_t launch_kv4_prefill(const AttnArgs& a, int64_t head_dim, int64_t longest, float* parts, cudaStream_t s) {
  const PrefillShape p = prefill_shape(a.batch * a.kv_heads, (int64_t)a.group * a.seq);
  if (head_dim == 64)
    return p.nq == 1 ? launch_prefill<64, 1>(a, p, longest, parts, s) : launch_prefill<64, 2>(a, p, longest, parts, s);
  return p.nq == 1 ? launch_prefill<128, 1>(a, p, longest, parts, s) : launch_prefill<128, 2>(a, p, longest, parts, s);
}

cudaError_t kv4_prefill_wait_timeouts(unsigned int* count, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(count, g_wait_timeouts, sizeof(*count));
  if (e == cudaSuccess && reset) {
    const unsigned int zero = 0;
    e = cudaMemcpyToSymbol(g_wait_timeouts, &zero, sizeof(zero));
  }
  return e;
}

}  // namespace hrm
