// Attention of many query rows over the 4-bit cache on tcgen05 (prompts and further
// turns of a chat), and the pass that adds the probabilities of many query rows to
// the cache rows' weights.
//
// A CTA owns NQ x 128 query rows of one kv head and walks its share of the cache in
// tiles of N rows: NQ = 2 and N = 128 up to head_dim 128, 1 and 64 above, where the
// operands of two stages fill the shared memory.  Three kinds of warps work at once, handing tiles over by
// mbarriers:
//   * 4 warps dequantise (with NQ = 1 4 for k and 4 for v): codes and scales from global
//     memory (the next tile's are loaded while this one is converted), bf16 operands
//     to shared memory, two stages.  k is stored as it lies, [row][element]; v transposed, [element][row],
//     two cache rows' half words put together before the conversion, so that both
//     operands are K-major.
//   * 4 warps per query tile do the softmax, a thread per row, the row in registers:
//     no shuffles.  P goes to tensor memory, over S, in two halves.  O is
//     rescaled only when a row's maximum has grown by more than 8 (in log2 units)
//     since its last rescale: until then probabilities may be as large as 2^8,
//     which neither the bf16 P nor the fp32 sums mind.
//   * one thread issues the products, S = Q K^T (128 x N, accumulated in tensor memory)
//     and O += P V with P read from tensor memory: with NQ = 2 those of one query tile
//     run while the other's softmax does, with NQ = 1 S of the next cache tile does.
// What bounds it: a tile costs 128 exponentials per row on a unit of 16 per clock
// (2048 cycles for 256 rows), as long as its products on the tensor cores; but a query
// tile's softmax waits for its own products, P being where S was, so that a tile takes
// 3400 cycles of softmax and products in turn, the other query tile's in between.
// Measured (D = 128): 512 queries of 16 heads over 8192 rows 50 us (710 TFLOP/s); 2 x
// 4096 queries of 12 heads with gate, causal past a prefix of 1000, 133 us (820), with
// the weights' kernel below 224.  With NQ = 1 a tile takes 3300 cycles: the
// stores of the operands and the products share the shared memory's bandwidth (8 x 64 queries
// of 12 heads over 8192 rows 121 us; k and v filled by 4 warps in turns 135, with one buffer
// of S 153; codes loaded two tiles ahead 136).
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
constexpr float kSlack = 8.0f;

template <int D>
constexpr int tile_rows() { return D <= 128 ? 128 : 64; }
constexpr uint32_t tmem_columns(int used) { return used <= 128 ? 128 : used <= 256 ? 256 : 512; }

template <int D, int NQ>
struct Pre {
  static constexpr int kN = tile_rows<D>();  // cache rows of a tile
  static constexpr int kGroups = D / kKv4Group;
  // Warpgroups: NQ of softmax; one that fills k and v, or (NQ = 1, where a tile has half
  // the softmax but all the filling) one for each; one for the products' thread.
  static constexpr int kSoftmax = NQ * 128, kFill = (3 - NQ) * 128;
  static constexpr int kThreads = kSoftmax + kFill + 128;
  // 4 warps on each scheduler leave a thread 128 registers, too few for a row of 128
  // scores.  The warpgroups share the launch's registers out again (NQ = 2, chunk of 512
  // over 8192: 51 us; 168 + 104 + 72: 60; 152 + 120 + 88: 60).
  static constexpr int kLaunchRegs = 128, kSoftmaxRegs = NQ == 2 ? 160 : 184, kFillRegs = 120, kMmaRegs = 72;
  static_assert(NQ * kSoftmaxRegs + (3 - NQ) * kFillRegs + kMmaRegs <= 4 * kLaunchRegs);
  static_assert(kSoftmaxRegs >= kLaunchRegs && kFillRegs <= kLaunchRegs && kMmaRegs <= kLaunchRegs);  // taken, given
  static constexpr int kQ = 0, kQBytes = kM * D * 2;              // per query tile
  static constexpr int kK = NQ * kQBytes, kKBytes = kN * D * 2;   // per stage
  static constexpr int kV = kK + 2 * kKBytes, kVBytes = D * kN * 2;
  static constexpr int kSmem = kV + 2 * kVBytes + 1024;  // + alignment of the panels
  // A single query tile has two buffers of S, which take turns: S of the next cache tile
  // is computed during the softmax of this one.
  static constexpr int kSBufs = 3 - NQ;
  static constexpr int kOAt = NQ * kSBufs * kN;
  static constexpr uint32_t kColumns = tmem_columns(kOAt + NQ * D);  // S of each tile, then O of each
};

// Barriers, in order: pairs by stage; S and P by query tile, or by buffer of S; O by query tile;
// the last products, where a wait ran out.
enum {
  kKFull = 0, kKEmpty = 2, kVFull = 4, kVEmpty = 6, kSFull = 8, kPHalf = 10, kPFull = 12, kOFull = 14, kDone = 16,
  kBars = 17
};

// What is left by rows whose waits ran out: in a partial result's mask of groups this bit,
// so that the joining kernel does not write them; as the log of their sum +inf, so
// that the weights' kernel finds all their probabilities 0.
constexpr uint32_t kTimedOut = 1u << 31;

struct PrefillSplit {
  int count;     // CTAs per item (kv head x block of query rows)
  float* parts;  // per (item, split), [D][rows] sums, then the rows' maxima, sums and masks; rows = NQ * 128
};
__host__ __device__ inline int64_t prefill_part(int nq, int64_t head_dim) { return nq * kM * (head_dim + 3); }

// Element x of a row's order of elements in shared memory: within 8, kv4_pair's order.
__device__ __forceinline__ uint4 paired_order(const uint4& v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                    __byte_perm(v.y, v.w, 0x7632));
}

// Query rows [r0, + count) of a kv head: the highest and the lowest number of cache
// rows that one of them sees (rows past the last: none).
__device__ __forceinline__ int2 row_limits(const Visible& see, unsigned seq, unsigned rows, unsigned r0,
                                           unsigned count) {
  const unsigned r1 = min(r0 + count, rows) - 1;
  const unsigned g0 = r0 / seq, s0 = r0 - g0 * seq, g1 = r1 / seq, s1 = r1 - g1 * seq;
  return make_int2(see.rows((int)(g0 == g1 ? s1 : seq - 1)),
                   r0 + count > rows ? 0 : see.rows((int)(g0 == g1 ? s0 : 0)));
}

// A filling thread's share of a tile of N rows: pieces (16 bytes of codes, one group)
// of k, and one piece of 4 adjacent rows of v (where there are fewer of those than
// threads, some threads have none).  The lanes' rows are such that a warp's loads
// fill whole sectors and its stores fall into different banks: 16 lanes have 16
// rows (or quads of rows) of one piece, the other 16 the next piece.
template <int D, int N>
struct Codes {
  static constexpr int kPieces = D / 32;  // per row
  static constexpr int kK = N * kPieces / 128;
  uint4 k[kK], v[4];
  uint32_t ks[kK], vs[4];

  // of the half warp number h, in order: first the pieces, then the rows
  __device__ __forceinline__ static int piece(int h) { return (h & 1) + 2 * ((h >> 1) % (kPieces / 2)); }
  __device__ __forceinline__ static int sixteen(int h) { return (h >> 1) / (kPieces / 2); }
  __device__ __forceinline__ static int k_row(int i, int t) { return sixteen(8 * i + (t >> 4)) * 16 + (t & 15); }
  __device__ __forceinline__ static int k_piece(int i, int t) { return piece(8 * i + (t >> 4)); }
  __device__ __forceinline__ static bool v_works(int t) { return (t >> 4) < N / 64 * kPieces; }
  __device__ __forceinline__ static int v_quad(int t) { return sixteen(t >> 4) * 16 + (t & 15); }
  __device__ __forceinline__ static int v_piece(int t) { return piece(t >> 4); }

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
        const int c = 4 * p + w;  // 16-byte piece of the row in bf16
        *reinterpret_cast<uint4*>(dst + (c / 8) * (N * 128) + panel_piece(row, c % 8)) =
            make_uint4(fma_bf16x2(kv4_pair<0>(x), s2, z2), fma_bf16x2(kv4_pair<1>(x), s2, z2),
                       fma_bf16x2(kv4_pair<2>(x), s2, z2), fma_bf16x2(kv4_pair<3>(x), s2, z2));
      }
    }
  }
  // bf16 v to the panels at dst, [element][row].  With `flags`, groups that are not
  // finite are stored as zeros and marked there.
  __device__ __forceinline__ void store_v(uint8_t* dst, int t, uint8_t (*flags)[8]) {
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
        const uint32_t xa = __byte_perm(vget(v[0], w), vget(v[1], w), sel);
        const uint32_t xb = __byte_perm(vget(v[2], w), vget(v[3], w), sel);
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
  constexpr int kN = T::kN;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[kBars];
  __shared__ uint32_t s_tmem;
  __shared__ __align__(16) uint8_t s_bad[2][kN][8];  // per stage and cache row: groups of v that are not finite
  uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const uint32_t base = smem_addr(smem), bar0 = smem_addr(bars);
  auto bar = [&](int i) -> uint32_t { return bar0 + 8 * i; };
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  grid_dependency_begin();

  const unsigned rows = a.group * a.seq;
  const unsigned item = blockIdx.x / split.count;
  const int rank = (int)(blockIdx.x - item * split.count);
  // all heads' last rows first: under a causal mask they have the most tiles
  const unsigned heads_all = (unsigned)(a.batch * a.kv_heads), back = item / heads_all;
  const int bh = (int)(item - back * heads_all), b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
  const unsigned row0 = (blocks_q - 1 - back) * (NQ * kM);
  // query row r of the kv head is query r % seq of its head r / seq: they lie one after
  // another (worked out where it is needed: the softmax has no register to spare)
  auto q_row0 = [&]() -> int64_t { return ((int64_t)b * a.heads + hk * a.group) * a.seq; };

  // ---- set-up: limits, queries, barriers, tensor memory
  {
    const uint32_t flip = a.scale_log2 < 0.0f ? 0x80008000u : 0u;  // the softmax takes |scale|
    const uint32_t keep = a.scale_log2 == 0.0f ? 0u : 0xffffffffu;  // scale 0: all scores 0
    constexpr int kAhead = 8;  // pieces in flight at once per thread
    const uint4* src = a.q + (q_row0() + row0) * (D / 8);
    for (int i0 = tid; i0 < NQ * kM * (D / 8); i0 += kAhead * T::kThreads) {
      uint4 v[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = i0 + x * T::kThreads, r = i / (D / 8);
        v[x] = make_uint4(0, 0, 0, 0);
        if (i < NQ * kM * (D / 8) && row0 + r < rows) v[x] = ld_keep(src + i);
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = i0 + x * T::kThreads, r = i / (D / 8), p = i % (D / 8);
        const uint4 y = paired_order(v[x]);
        if (i < NQ * kM * (D / 8))
          *reinterpret_cast<uint4*>(smem + (r / kM) * T::kQBytes + (p / 8) * (kM * 128) + panel_piece(r % kM, p % 8)) =
              make_uint4((y.x ^ flip) & keep, (y.y ^ flip) & keep, (y.z ^ flip) & keep, (y.w ^ flip) & keep);
      }
    }
  }
  const Visible see(a, b);
  const int2 limits = row_limits(see, a.seq, rows, row0, NQ * kM);
  const int limit = limits.x, lowest = limits.y;
  const int tiles = (limit + kN - 1) / kN;
  int j0 = 0, j1 = tiles;
  if (split.count > 1) {
    j0 = (int)((int64_t)tiles * rank / split.count);
    j1 = (int)((int64_t)tiles * (rank + 1) / split.count);
  }
  const int n = j1 - j0;
  constexpr int kFillFirst = T::kSoftmax / 32, kMmaWarp = kFillFirst + T::kFill / 32;
  const bool fills = warp >= kFillFirst && warp < kMmaWarp;
  for (int i = tid; i < 2 * kN; i += T::kThreads) *reinterpret_cast<uint2*>(s_bad[i / kN][i % kN]) = make_uint2(0, 0);
  if (warp == 0) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(bar(kKFull + i), 128);
        mbar_init(bar(kKEmpty + i), 1);
        mbar_init(bar(kVFull + i), 128);
        mbar_init(bar(kVEmpty + i), 1);
        mbar_init(bar(kSFull + i), 1);
        mbar_init(bar(kPHalf + i), kM);
        mbar_init(bar(kPFull + i), kM);
        mbar_init(bar(kOFull + i), 1);
      }
      mbar_init(bar(kDone), 1);
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

  if (warp < kFillFirst) {
    // ---------------------------------------------------------------- softmax
    take_registers<T::kSoftmaxRegs>();
    const int qt = warp / 4, r = qt * kM + (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_at = tmem + lanes + T::kOAt + qt * D;
    const int lim = row0 + r < rows ? see.rows((int)((row0 + r) % a.seq)) : -1;
    const float scale = a.scale_log2 == 0.0f ? 1.0f : fabsf(a.scale_log2);
    float m = -INFINITY, l = 0.0f;  // m: of the unscaled scores, as of the last rescale
    uint32_t bad = 0;  // bit g: group g of v
    bool ok = true;
    for (int j = 0; j < n; ++j) {
      const int first = (j0 + j) * kN;
      const int buf = T::kSBufs == 2 ? j & 1 : qt, turn = T::kSBufs == 2 ? (j >> 1) & 1 : j & 1;
      const uint32_t s_at = tmem + lanes + buf * kN;
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar(kSFull + buf), turn));
      if (!ok) break;
      tcgen05_after_sync();
      uint32_t s[kN];
#pragma unroll
      for (int c = 0; c < kN / 32; ++c) tmem_load32(s + 32 * c, s_at + 32 * c);
      tmem_wait_load<kN>(s);
      if (!__all_sync(0xffffffffu, first + kN <= lim)) {  // some score of the warp's rows is masked
#pragma unroll
        for (int i = 0; i < kN; ++i)
          if (first + i >= lim) s[i] = 0xff800000u;
      }
      float top;
      {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(s[i]);
#pragma unroll
        for (int i = 4; i + 1 < kN; i += 2)
          x[(i >> 1) & 3] = max3_nan(x[(i >> 1) & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        top = max3_nan(x[0], x[1], max_nan(x[2], x[3]));
      }
      // Grown by more than the slack (or from nothing, or NaN): rescale.  With one buffer
      // of S, S of this tile is complete, so every product issued before it is, O's among
      // them; with two, O's of the tile before may still run.
      const bool grown = !(top <= m + kSlack / scale);
      if (__any_sync(0xffffffffu, grown)) {
        const float to = grown ? max_nan(top, m) : m;
        const float f = m == -INFINITY ? 0.0f : exp2_approx((m - to) * scale);
        if (grown) {
          l *= f;
          m = to;
        }
        if (T::kSBufs == 2 && j > 0) {
          ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar(kVEmpty + ((j - 1) & 1)), ((j - 1) >> 1) & 1));
          if (!ok) break;
          tcgen05_after_sync();
        }
        if (j > 0) {
          const float by = grown ? f : 1.0f;
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_load16(o, o_at + 16 * c);
            tmem_wait_load<16>(o);
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
            tmem_store16(o_at + 16 * c, o);
          }
        }
      }
      if (first + kN > lowest && lowest < limit) {
        // rows that some query must not see: the groups of v that are not finite were read
        // as zeros (before P is handed over: the products free the flags' buffer)
        ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar(kVFull + (j & 1)), (j >> 1) & 1));
        if (!ok) {
          tmem_wait_store();  // O's, before its memory is given back
          break;
        }
        const uint2* flags = reinterpret_cast<const uint2*>(s_bad[j & 1]);
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < kN / 32; ++i) any |= flags[32 * i + lane].x | flags[32 * i + lane].y;
        if (__any_sync(0xffffffffu, any != 0)) {
#pragma unroll 1
          for (int i = 0; i < kN && first + i < lim; ++i) {
            const uint2 f = flags[i];
#pragma unroll
            for (int x = 0; x < 4; ++x) bad |= (f.x >> (8 * x) & 1u) << x | (f.y >> (8 * x) & 1u) << (4 + x);
          }
          __syncwarp();
        }
      }
      const float shift = m == -INFINITY ? 0.0f : m * scale;
      const uint64_t scale2 = pack_f32x2(__float_as_uint(scale), __float_as_uint(scale));
      const uint64_t shift2 = pack_f32x2(__float_as_uint(-shift), __float_as_uint(-shift));
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < kN / 32; ++c) {
        uint32_t p[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint64_t y = fma_f32x2(pack_f32x2(s[32 * c + 2 * i], s[32 * c + 2 * i + 1]), scale2, shift2);
          const float p0 = exp2_approx(lo_f32(y)), p1 = exp2_approx(hi_f32(y));
          sum[i & 1] = add_f32x2(sum[i & 1], pack_f32x2(__float_as_uint(p0), __float_as_uint(p1)));
          p[i] = pack_bf16x2(p0, p1);
        }
        tmem_store16(s_at + 16 * c, p);  // over scores that this thread has in registers
        if (c + 1 == kN / 64 || c + 1 == kN / 32) {
          tmem_wait_store();
          tcgen05_before_sync();
          mbar_arrive(bar((c + 1 == kN / 64 ? kPHalf : kPFull) + buf));
        }
      }
      const uint64_t both = add_f32x2(sum[0], sum[1]);
      l += lo_f32(both) + hi_f32(both);
    }
    const unsigned row = row0 + r;
    const unsigned g = row / a.seq, sq = row - g * a.seq;
    const int64_t head = hk * a.group + g;
    const int64_t out_at = row < rows ? (((int64_t)b * a.seq + sq) * a.heads + head) * D : -1;
    // A thread has a row, but 32 rows' pieces of 16 bytes lie 32 heads' rows apart: gate
    // and output pass through the warp's 32 rows of the query tile, free since the last S,
    // so that a warp's access covers whole rows.  (Accesses by row took 28000 cycles
    // for 256 rows of 128 elements with a gate, as long as 8 tiles.)
    uint8_t* const mine = smem + T::kQ + qt * T::kQBytes;
    const int warp_row = (warp & 3) * 32;
    auto each_piece = [&](auto&& f) {  // f(place in the output or -1, place in the tile)
#pragma unroll 4
      for (int i = 0; i < D / 8; ++i) {
        const int x = 32 * i + lane, in_warp = x / (D / 8), p = x % (D / 8);
        const int64_t at = __shfl_sync(0xffffffffu, out_at, in_warp);
        f(at < 0 ? at : at + 8 * p, mine + (p / 8) * (kM * 128) + panel_piece(warp_row + in_warp, p % 8));
      }
    };
    if (ok && split.count == 1 && a.gate != nullptr) {
      each_piece([&](int64_t at, uint8_t* place) {
        cp_async_zfill<16>(smem_addr(place), a.gate + (at < 0 ? 0 : at), at >= 0);
      });
      cp_async_commit();
    }
    if (ok && n > 0) ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar(kOFull + qt), 0));
    tcgen05_after_sync();
    if (split.count == 1) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      if (row < rows && a.lse != nullptr)
        a.lse[q_row0() + row] = !ok ? INFINITY : (m == -INFINITY ? -INFINITY : m * scale + log2f(l));
      cp_async_wait_all();
      __syncwarp();
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_load32(o, o_at + 32 * c);
          tmem_wait_load<32>(o);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0;
        }
        const bool nan = bad >> c & 1u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int p = 4 * c + i;
          uint4* const place = reinterpret_cast<uint4*>(mine + (p / 8) * (kM * 128) + panel_piece(r % kM, p % 8));
          uint4 y, gate = make_uint4(0, 0, 0, 0);
          if (a.gate != nullptr) gate = *place;
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float v0 = __uint_as_float(o[8 * i + 2 * w]) * inv, v1 = __uint_as_float(o[8 * i + 2 * w + 1]) * inv;
            if (nan) v0 = v1 = __int_as_float(0x7fc00000);
            if (a.gate != nullptr) {
              v0 *= gate_factor(bf16_lo(vget(gate, w)));
              v1 *= gate_factor(bf16_hi(vget(gate, w)));
            }
            vset(y, w, pack_bf16x2(v0, v1));
          }
          *place = y;
        }
      }
      __syncwarp();
      if (ok)
        each_piece([&](int64_t at, const uint8_t* place) {
          if (at >= 0) st_l2(reinterpret_cast<uint4*>(a.out + at), *reinterpret_cast<const uint4*>(place));
        });
    } else {
      float* part = split.parts + (int64_t)blockIdx.x * prefill_part(NQ, D);
#pragma unroll 1
      for (int c = 0; c < D / 32 && n > 0; ++c) {
        uint32_t o[32];
        tmem_load32(o, o_at + 32 * c);
        tmem_wait_load<32>(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) part[(32 * c + i) * (NQ * kM) + r] = __uint_as_float(o[i]);
      }
      float* tail = part + NQ * kM * D + r;
      tail[0] = m == -INFINITY ? -INFINITY : m * scale;  // log2 units
      tail[NQ * kM] = l;
      tail[2 * NQ * kM] = __uint_as_float(ok ? bad : kTimedOut);
    }
  } else if (fills) {
    // --------------------------------------------------------------- filling
    give_registers<T::kFillRegs>();
    const int t = tid & 127;
    const bool fills_k = NQ == 2 || warp < kFillFirst + 4, fills_v = NQ == 2 || !fills_k;
    const int64_t head_row = (int64_t)bh * a.c.cache_len;
    const uint8_t* kc = a.c.k_codes + head_row * (D / 2);
    const uint8_t* vc = a.c.v_codes + head_row * (D / 2);
    const uint32_t* ks = a.c.k_scales + head_row * T::kGroups;
    const uint32_t* vs = a.c.v_scales + head_row * T::kGroups;
    Codes<D, kN> c;
    if (n > 0) {
      if (fills_k) c.fetch_k(kc, ks, j0 * kN, limit, t);
      if (fills_v) c.fetch_v(vc, vs, j0 * kN, limit, t);
    }
    for (int j = 0; j < n; ++j) {
      const int first = (j0 + j) * kN, s = j & 1, phase = (j >> 1) & 1;
      if (fills_k) {
        if (!mbar_wait_bounded(bar(kKEmpty + s), phase ^ 1)) break;
        c.store_k(smem + T::kK + s * T::kKBytes, t);
        fence_proxy_async_smem();
        mbar_arrive(bar(kKFull + s));
        if (j + 1 < n) c.fetch_k(kc, ks, first + kN, limit, t);
      }
      if (fills_v) {
        if (!mbar_wait_bounded(bar(kVEmpty + s), phase ^ 1)) break;
        const bool border = first + kN > lowest && lowest < limit;
        c.store_v(smem + T::kV + s * T::kVBytes, t, border ? s_bad[s] : nullptr);
        fence_proxy_async_smem();
        mbar_arrive(bar(kVFull + s));
        if (j + 1 < n) c.fetch_v(vc, vs, first + kN, limit, t);
      }
    }
  } else {
    // -------------------------------------------------------------- products
    // By one thread; they run in the order of their issue.
    give_registers<T::kMmaRegs>();
    if (warp == kMmaWarp && elect_one()) {
      constexpr uint32_t kShapeS = mma_shape(kM, kN), kShapeO = mma_shape(kM, D);
      auto scores = [&](int qt, int buf, int s) {  // of the keys of stage s
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tcgen05_mma(tmem + buf * kN, panel_desc(base + T::kQ + qt * T::kQBytes + (k / 4) * (kM * 128) + 32 * (k % 4)),
                      panel_desc(base + T::kK + s * T::kKBytes + (k / 4) * (kN * 128) + 32 * (k % 4)), kShapeS, k > 0);
        tcgen05_commit(bar(kSFull + buf));
      };
      bool run = n > 0 && mbar_wait_bounded(bar(kKFull), 0);
      if (run) {
        tcgen05_after_sync();
#pragma unroll
        for (int qt = 0; qt < NQ; ++qt) scores(qt, qt, 0);
        tcgen05_commit(bar(kKEmpty));
      }
      for (int j = 0; j < n && run; ++j) {
        const int s = j & 1, phase = (j >> 1) & 1;
        if (T::kSBufs == 1) run = mbar_wait_bounded(bar(kVFull + s), phase);
        if (j + 1 < n) run = run && mbar_wait_bounded(bar(kKFull + (s ^ 1)), ((j + 1) >> 1) & 1);
        if (!run) break;
        if (T::kSBufs == 2) {
          if (j + 1 < n) {  // over P of the tile before, which its products have read by then
            tcgen05_after_sync();
            scores(0, s ^ 1, s ^ 1);
            tcgen05_commit(bar(kKEmpty + (s ^ 1)));
          }
          run = mbar_wait_bounded(bar(kVFull + s), phase);
        }
#pragma unroll
        for (int qt = 0; qt < NQ; ++qt) {
          const int buf = T::kSBufs == 2 ? s : qt, turn = T::kSBufs == 2 ? phase : j & 1;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            run = run && mbar_wait_bounded(bar((half == 0 ? kPHalf : kPFull) + buf), turn);
            if (!run) break;
            tcgen05_after_sync();
#pragma unroll
            for (int k = half * (kN / 32); k < (half + 1) * (kN / 32); ++k)
              tcgen05_mma_ta(tmem + T::kOAt + qt * D, tmem + buf * kN + 8 * k,
                             panel_desc(base + T::kV + s * T::kVBytes + (k / 4) * (D * 128) + 32 * (k % 4)), kShapeO,
                             j > 0 || k > 0);
          }
          if (!run) break;
          if (qt == NQ - 1) tcgen05_commit(bar(kVEmpty + s));
          if (j + 1 == n) {
            tcgen05_commit(bar(kOFull + qt));
          } else if (T::kSBufs == 1) {
            scores(qt, qt, s ^ 1);  // replace P, which the products before them have read by then
            if (qt == NQ - 1) tcgen05_commit(bar(kKEmpty + (s ^ 1)));
          }
        }
      }
      if (n > 0 && !run) {  // a wait ran out: what was issued ends before its memory is given back
        tcgen05_commit(bar(kDone));
        mbar_wait_bounded(bar(kDone), 0);
      }
    }
  }
  __syncwarp();
  tcgen05_before_sync();
  __syncthreads();
  if (warp == 0) tmem_free(tmem, T::kColumns);
}

// Joins the split items' partial results: a thread per query row and 16 elements.
constexpr int kJoinElements = 16;
template <int D, int NQ>
__global__ void __launch_bounds__(kM) kv4_prefill_join_kernel(const AttnArgs a, const PrefillSplit split,
                                                              const int blocks_q) {
  grid_dependency_begin();
  constexpr int kRows = NQ * kM, kCuts = D / kJoinElements;
  const unsigned rows = a.group * a.seq;
  const unsigned tile = blockIdx.x / kCuts, item = tile / NQ;  // query tile of 128 rows
  const int d0 = (int)(blockIdx.x - tile * kCuts) * kJoinElements, r = (int)(tile - item * NQ) * kM + threadIdx.x;
  const unsigned heads_all = (unsigned)(a.batch * a.kv_heads), back = item / heads_all;
  const int bh = (int)(item - back * heads_all), b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
  const unsigned row = (blocks_q - 1 - back) * kRows + r;
  if (row >= rows) return;
  const float* parts = split.parts + (int64_t)item * split.count * prefill_part(NQ, D);
  auto tail = [&](int i) -> const float* { return parts + i * prefill_part(NQ, D) + kRows * D + r; };
  // online over the parts; the loads of 4 parts are in flight at once
  constexpr int kAhead = 4;
  float top = -INFINITY, norm = 0.0f, sum[kJoinElements];
  uint32_t bad = 0;
#pragma unroll
  for (int x = 0; x < kJoinElements; ++x) sum[x] = 0.0f;
  for (int i0 = 0; i0 < split.count; i0 += kAhead) {
    float m[kAhead], l[kAhead], v[kAhead][kJoinElements];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const bool in = i0 + i < split.count;
      const float* t = tail(in ? i0 + i : 0);
      const float* part = parts + (in ? i0 + i : 0) * prefill_part(NQ, D) + d0 * kRows + r;
      m[i] = in ? t[0] : -INFINITY;
      l[i] = t[kRows];
      if (in) bad |= __float_as_uint(t[2 * kRows]);
#pragma unroll
      for (int x = 0; x < kJoinElements; ++x) v[i][x] = part[x * kRows];
    }
    float now = top;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) now = max_nan(now, m[i]);
    const float back_by = top == -INFINITY ? 0.0f : exp2_approx(top - now);
    norm *= back_by;
#pragma unroll
    for (int x = 0; x < kJoinElements; ++x) sum[x] *= back_by;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (m[i] == -INFINITY) continue;  // a part without rows left only this mark
      const float f = exp2_approx(m[i] - now);
      norm += f * l[i];
#pragma unroll
      for (int x = 0; x < kJoinElements; ++x) sum[x] += f * v[i][x];
    }
    top = now;
  }
  const bool timed_out = bad & kTimedOut;
  const unsigned g = row / a.seq, s = row - g * a.seq;
  const int64_t head = hk * a.group + g;
  if (a.lse != nullptr && d0 == 0)
    a.lse[((int64_t)b * a.heads + hk * a.group) * a.seq + row] =
        timed_out ? INFINITY : (top == -INFINITY ? -INFINITY : top + log2f(norm));
  if (timed_out) return;  // unwritten, as without a split
  const float inv = norm == 0.0f ? 0.0f : 1.0f / norm;
  const bool nan = bad >> (d0 / kKv4Group) & 1u;
  const int64_t at = (((int64_t)b * a.seq + s) * a.heads + head) * D + d0;
#pragma unroll
  for (int i = 0; i < kJoinElements / 8; ++i) {
    uint4 y, gate = make_uint4(0, 0, 0, 0);
    if (a.gate != nullptr) gate = ld_l2(reinterpret_cast<const uint4*>(a.gate + at) + i);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      float v0 = sum[8 * i + 2 * w] * inv, v1 = sum[8 * i + 2 * w + 1] * inv;
      if (nan) v0 = v1 = __int_as_float(0x7fc00000);
      if (a.gate != nullptr) {
        v0 *= gate_factor(bf16_lo(vget(gate, w)));
        v1 *= gate_factor(bf16_hi(vget(gate, w)));
      }
      vset(y, w, pack_bf16x2(v0, v1));
    }
    st_l2(reinterpret_cast<uint4*>(a.out + at) + i, y);
  }
}

// weights[j] += the probabilities of cache row j, summed over the query rows in
// their order: S^T = K Q^T, recomputed, so that a thread has a cache row and sums
// over its columns by itself -- no atomics, no shuffles, the same sum from call to
// call.  A CTA owns 128 cache rows, dequantised once; 4 warps copy the query tiles
// to shared memory (cp.async, two stages), one thread issues the products into two
// buffers of tensor memory, 4 warps take the exponentials, 128 per row and tile.  Up
// to head_dim 128 two CTAs share an SM: a pair of tiles takes them 2600 cycles, 2048 of
// exponentials.  2 x 4096 queries of 12 heads of 128: 96 us (one CTA of 256 cache rows
// instead of two of 128, with half the copies: 116; every third or fourth pair of exponentials
// by a polynomial: 94 to 95).
template <int D>
struct Wgt {
  static constexpr int kK = 0, kBytes = 128 * D * 2, kQ = kBytes;  // keys; two stages of queries
  // (at least so much that no third CTA comes to an SM, whose tensor memory two fill)
  static constexpr int kSmem = D == 64 ? 80 * 1024 : 3 * kBytes + 1024;
  static constexpr int kThreads = 128 + 128 + 32;
  static constexpr uint32_t kColumns = 256;
};
enum { kWFull = 0, kWEmpty = 2, kWSFull = 4, kWSEmpty = 6, kWDone = 8, kWBars = 9 };

// The query tiles of a kv head with a row that sees cache row `first` or one after it,
// in order.  (Asking each tile in turn for its limits, divisions and all, took 750
// cycles a tile.)
struct QueryTiles {
  const Visible see;
  const unsigned seq, rows;
  const int first;
  unsigned row = 0, s = 0;  // the tile's first row, and which query of its head that is
  int lowest = 0;           // cache rows that the one of its rows with the fewest sees
  __device__ __forceinline__ QueryTiles(const Visible& see, unsigned seq, unsigned rows, int first)
      : see(see), seq(seq), rows(rows), first(first) {}
  __device__ __forceinline__ bool find() {  // from the present tile on; false past the last
    while (row < rows) {
      const bool more = s + 128 > seq;  // heads than one (or the end)
      if (see.rows((int)(more ? seq - 1 : s + 127)) > first) {
        lowest = row + 128 > rows ? 0 : see.rows((int)(more ? 0 : s));
        return true;
      }
      // a head's last query sees `first`: on to the tile of the first query that does
      step((unsigned)(first - see.off - s) / 128u);
    }
    return false;
  }
  __device__ __forceinline__ void step(unsigned tiles) {
    row += 128 * tiles;
    s += 128 * tiles;
    if (s >= seq) s %= seq;
  }
};

template <int D>
__global__ void __launch_bounds__(Wgt<D>::kThreads) kv4_weights_kernel(const AttnArgs a) {
  using T = Wgt<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[kWBars];
  __shared__ uint32_t s_tmem;
  __shared__ __align__(16) float s_lse[4][128];  // negated
  __shared__ int s_lim[4][128];
  __shared__ int s_whole[4], s_more[4];  // all of the tile's queries see all of the rows; another tile follows
  uint8_t* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  const uint32_t base = smem_addr(smem), bar0 = smem_addr(bars);
  auto bar = [&](int i) -> uint32_t { return bar0 + 8 * i; };
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  grid_dependency_begin();
  const unsigned rows = a.group * a.seq;
  // all heads' first rows first: under a causal mask most queries see them
  const unsigned heads_all = (unsigned)(a.batch * a.kv_heads), tile = blockIdx.x / heads_all;
  const int bh = (int)(blockIdx.x - tile * heads_all), b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
  const int first = (int)tile * 128;
  const Visible see(a, b);
  const int limit = see.rows(a.seq - 1);  // of the last query: the highest
  if (first >= limit) return;

  const int64_t head_row = (int64_t)bh * a.c.cache_len;
  {  // the keys, elements in kv4_pair's order put back: the queries are copied as they are
    const uint8_t* kc = a.c.k_codes + head_row * (D / 2);
    const uint32_t* ks = a.c.k_scales + head_row * (D / 32);
    for (int i = tid; i < 128 * (D / 32); i += T::kThreads) {
      const int row = i / (D / 32), p = i % (D / 32);
      uint4 c = make_uint4(0, 0, 0, 0);
      uint32_t sz = 0;
      if (first + row < limit) {
        c = ld_l2(reinterpret_cast<const uint4*>(kc + (int64_t)(first + row) * (D / 2)) + p);
        sz = __ldcg(ks + (int64_t)(first + row) * (D / 32) + p);
      }
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int at = 4 * p + w;
        *reinterpret_cast<uint4*>(smem + T::kK + (at / 8) * (128 * 128) + panel_piece(row, at % 8)) =
            kv4_values(vget(c, w), sz);
      }
    }
  }
  if (warp == 8) {
    if (lane == 0) {
      for (int i = 0; i < 2; ++i) {
        mbar_init(bar(kWFull + i), 128);
        mbar_init(bar(kWEmpty + i), 1);
        mbar_init(bar(kWSFull + i), 1);
        mbar_init(bar(kWSEmpty + i), 128);
      }
      mbar_init(bar(kWDone), 1);
      mbar_init_fence();
    }
    __syncwarp();
    tmem_alloc(smem_addr(&s_tmem), T::kColumns);
  }
  fence_proxy_async_smem();
  tcgen05_before_sync();
  __syncthreads();
  tcgen05_after_sync();
  const uint32_t tmem = s_tmem;

  if (warp < 4) {
    // ----------------------------------------------------------- probabilities
    const int at = first + tid;
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    uint64_t sum[2] = {0, 0};
    float extra = 0.0f;  // of tiles with masked probabilities
    const uint64_t scale2 = pack_f32x2(__float_as_uint(a.scale_log2), __float_as_uint(a.scale_log2));
    int n = 0, more = 1;  // (`first` < limit: there is a tile)
    bool ok = true;
    while (more) {
      const int s = n & 1, phase = (n >> 1) & 1, entry = n & 3;
      ++n;
      ok = __all_sync(0xffffffffu, mbar_wait_bounded(bar(kWSFull + s), phase));
      if (!ok) break;
      tcgen05_after_sync();
      const bool whole = s_whole[entry] != 0;
      more = s_more[entry];
      uint32_t x[2][32];  // 32 columns are loaded while the 32 before them are worked on
      tmem_load32(x[0], tmem + lanes + 128 * s);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        tmem_wait_load<32>(x[c & 1]);
        if (c < 3) tmem_load32(x[(c + 1) & 1], tmem + lanes + 128 * s + 32 * (c + 1));
        if (whole) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint4 lse = *reinterpret_cast<const uint4*>(&s_lse[entry][32 * c + 4 * i]);
            const uint32_t* u = &x[c & 1][4 * i];
            const uint64_t y0 = fma_f32x2(pack_f32x2(u[0], u[1]), scale2, pack_f32x2(lse.x, lse.y));
            const uint64_t y1 = fma_f32x2(pack_f32x2(u[2], u[3]), scale2, pack_f32x2(lse.z, lse.w));
            sum[0] = add_f32x2(sum[0], pack_f32x2(__float_as_uint(exp2_approx(lo_f32(y0))),
                                                  __float_as_uint(exp2_approx(hi_f32(y0)))));
            sum[1] = add_f32x2(sum[1], pack_f32x2(__float_as_uint(exp2_approx(lo_f32(y1))),
                                                  __float_as_uint(exp2_approx(hi_f32(y1)))));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (at < s_lim[entry][32 * c + i])
              extra += exp2_approx(fmaf(__uint_as_float(x[c & 1][i]), a.scale_log2, s_lse[entry][32 * c + i]));
        }
      }
      tcgen05_before_sync();
      mbar_arrive(bar(kWSEmpty + s));
    }
    const uint64_t both = add_f32x2(sum[0], sum[1]);
    if (ok && at < limit) a.c.weights[head_row + at] += lo_f32(both) + hi_f32(both) + extra;
  } else if (warp < 8) {
    // ----------------------------------------------------------------- queries
    const int t = tid - 128;
    const int64_t q_row0 = ((int64_t)b * a.heads + hk * a.group) * a.seq;  // the head's query rows lie one after another
    const uint4* src = a.q + q_row0 * (D / 8);
    auto fetch = [&](unsigned row0, int s) {
      const int64_t at = (int64_t)row0 * (D / 8);
#pragma unroll
      for (int x = t; x < 128 * (D / 8); x += 128) {
        const int r = x / (D / 8), p = x % (D / 8);
        const bool in = row0 + r < rows;
        cp_async_zfill<16>(base + T::kQ + s * T::kBytes + (p / 8) * (128 * 128) + panel_piece(r, p % 8),
                           in ? src + at + x : src, in);
      }
    };
    QueryTiles q(see, a.seq, rows, first);
    int n = 0;
    bool more = q.find();
    while (more) {
      const int s = n & 1, phase = (n >> 1) & 1;
      if (!mbar_wait_bounded(bar(kWEmpty + s), phase ^ 1)) break;
      fetch(q.row, s);
      cp_async_commit();
      // (entry n & 3 of lse and limits: its last reader freed the scores' buffer that the
      // products of tile n - 2, now done, went to)
      const unsigned row = q.row + t, sq = q.s + t;
      s_lse[n & 3][t] = row < rows ? -a.lse[q_row0 + row] : 0.0f;
      s_lim[n & 3][t] = row < rows ? see.rows((int)(sq < q.seq ? sq : sq % q.seq)) : -1;
      const bool whole = first + 128 <= q.lowest;
      q.step(1);
      more = q.find();
      if (t == 0) {
        s_whole[n & 3] = whole;
        s_more[n & 3] = more;
      }
      ++n;
      cp_async_wait_all();
      fence_proxy_async_smem();
      mbar_arrive(bar(kWFull + s));
    }
  } else if (elect_one()) {
    // ---------------------------------------------------------------- products
    constexpr uint32_t kShape = mma_shape(128, 128);
    int n = 0, more = 1;
    bool run = true;
    while (more) {
      const int s = n & 1, phase = (n >> 1) & 1;
      run = mbar_wait_bounded(bar(kWFull + s), phase) && mbar_wait_bounded(bar(kWSEmpty + s), phase ^ 1);
      if (!run) break;
      more = s_more[n++ & 3];
      tcgen05_after_sync();
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t from = (k / 4) * (128 * 128) + 32 * (k % 4);
        tcgen05_mma(tmem + 128 * s, panel_desc(base + T::kK + from), panel_desc(base + T::kQ + s * T::kBytes + from),
                    kShape, k > 0);
      }
      tcgen05_commit(bar(kWSFull + s));
      tcgen05_commit(bar(kWEmpty + s));
    }
    if (!run) {  // as in the attention's kernel
      tcgen05_commit(bar(kWDone));
      mbar_wait_bounded(bar(kWDone), 0);
    }
  }
  __syncwarp();
  tcgen05_before_sync();
  __syncthreads();
  if (warp == 8) tmem_free(tmem, T::kColumns);
}

template <int D>
cudaError_t launch_weights(const AttnArgs& a, int64_t longest, cudaStream_t s) {
  const int64_t tiles = (longest + 127) / 128, grid = a.batch * a.kv_heads * tiles;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  const cudaError_t e = allow_shared<kv4_weights_kernel<D>>(Wgt<D>::kSmem);
  if (e != cudaSuccess) return e;
  return launch_kernel(kv4_weights_kernel<D>, grid, Wgt<D>::kThreads, Wgt<D>::kSmem, s, a);
}

struct PrefillShape {
  int nq, blocks_q;
  int64_t items;
};
PrefillShape prefill_shape(int64_t batch_kv_heads, int64_t rows, int64_t head_dim) {
  PrefillShape s;
  s.nq = rows > kM && head_dim <= 128 ? 2 : 1;
  s.blocks_q = (int)((rows + s.nq * kM - 1) / (s.nq * kM));
  s.items = batch_kv_heads * s.blocks_q;
  return s;
}

template <int D, int NQ>
cudaError_t launch_prefill(const AttnArgs& a, const PrefillShape& p, int64_t longest, float* parts, cudaStream_t s) {
  using T = Pre<D, NQ>;
  // One CTA per SM: items that leave SMs idle are split, to 2 tiles at least (12 heads, 64
  // queries over 2048 rows: 15.0 us, to 4 tiles 17.6, 256 over 1024 15.8 and 19.4; to 1 tile 256
  // over 2048 24.6 against 18.3), and into more than 8 parts, whose joining waits for
  // more reads, only past 64 tiles (256 queries over 4096 rows in 8 parts 22.4, in 12
  // 26.6; over 16384 47.0 and 43.9).
  const int64_t most = longest <= 64 * T::kN ? 8 : INT32_MAX;
  PrefillSplit split{1, parts};
  while (split.count < most && p.items * (split.count + 1) <= device_sm_count() &&
         (split.count + 1) * 2 * T::kN <= longest)
    ++split.count;
  if (p.items * split.count > INT32_MAX) return cudaErrorInvalidConfiguration;
  cudaError_t e = allow_shared<kv4_prefill_kernel<D, NQ>>(T::kSmem);
  if (e == cudaSuccess) e = has_registers<kv4_prefill_kernel<D, NQ>>(T::kLaunchRegs);
  if (e != cudaSuccess) return e;
  e = launch_kernel(kv4_prefill_kernel<D, NQ>, p.items * split.count, T::kThreads, T::kSmem, s, a, split, p.blocks_q);
  if (e != cudaSuccess || split.count == 1) return e;
  return launch_kernel(kv4_prefill_join_kernel<D, NQ>, p.items * NQ * (D / kJoinElements), kM, 0, s, a, split,
                       p.blocks_q);
}

}  // namespace

int64_t kv4_prefill_workspace(int64_t batch_kv_heads, int64_t rows, int64_t head_dim) {
  const PrefillShape p = prefill_shape(batch_kv_heads, rows, head_dim);
  const int64_t most = device_sm_count() / (p.items > 0 ? p.items : 1);  // CTAs per item, for any cache length
  return most < 2 ? 0 : p.items * most * prefill_part(p.nq, head_dim) * (int64_t)sizeof(float);
}

cudaError_t launch_kv4_prefill(const AttnArgs& a, int64_t head_dim, int64_t longest, float* parts, cudaStream_t s) {
  const PrefillShape p = prefill_shape(a.batch * a.kv_heads, (int64_t)a.group * a.seq, head_dim);
  switch (head_dim) {
    case 64:
      return p.nq == 1 ? launch_prefill<64, 1>(a, p, longest, parts, s) : launch_prefill<64, 2>(a, p, longest, parts, s);
    case 128:
      return p.nq == 1 ? launch_prefill<128, 1>(a, p, longest, parts, s)
                       : launch_prefill<128, 2>(a, p, longest, parts, s);
    case 192: return launch_prefill<192, 1>(a, p, longest, parts, s);
    default: return launch_prefill<256, 1>(a, p, longest, parts, s);
  }
}

cudaError_t launch_kv4_weights(const AttnArgs& a, int64_t head_dim, int64_t longest, cudaStream_t s) {
  switch (head_dim) {
    case 64: return launch_weights<64>(a, longest, s);
    case 128: return launch_weights<128>(a, longest, s);
    case 192: return launch_weights<192>(a, longest, s);
    default: return launch_weights<256>(a, longest, s);
  }
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
