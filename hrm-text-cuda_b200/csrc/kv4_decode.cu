// Attention of few query rows over the 4-bit cache: decoding, drafted tokens,
// shared kv heads.  All queries of one kv head that fit in 8 rows are one block
// of work, an item (more rows: more items).
//
// What bounds it: the cache is read once, 5 bits per element (D / 2 bytes of
// codes and D / 8 of scales per row for k and again for v), so the floor is HBM
// bandwidth; next to it the instructions that turn 4-bit codes into bf16 operands,
// 1.5 per element.  Hence:
//   * the codes become matrix operands in registers (mma.sync m16n8k16): the
//     tensor cores take the dot products off the fp32 pipe, and the dequantised
//     tile is never stored.  tcgen05 takes operands from shared memory only,
//     which would add a store and a barrier per element for a product whose 8
//     useful rows leave that unit idle either way.
//   * both products are transposed, so that the dequantised operand is A, whose 16
//     rows are all in use, and the 8 query columns are B: scores = k (16 cache rows)
//     x queries, output = v (16 elements x 16 cache rows) x probabilities.  With the
//     queries as A, half the products' rows were zeros, and filling A's register
//     quads with them took more instructions than the products (D = 128, per 16
//     cache rows: 412 instructions against 344).  The contraction order is free,
//     so lane t of a quad owns whole 16-byte pieces of a row of k.
//   * a probability is split into two bf16 numbers, hi + lo, multiplied in turn, so
//     that it carries 16 significant bits; v's operand serves both products.
//   * each warp streams its own 32-row tiles through a private ring of
//     shared-memory stages (cp.async), with no CTA barrier until the end.
//   * the long axis is split over the warps of a CTA and over CTAs.  Short caches:
//     the CTAs of an item are a cluster and join through distributed shared memory,
//     one launch.  Long ones: the items' blocks of 128 rows, laid end to end, are cut
//     into as many equal shares as CTAs fit on the GPU at once, whatever the
//     sequences' lengths; an item that is cut leaves partial results in the
//     workspace, and a second launch joins those.
// The softmax runs online: running maximum and sum in fp32, log2 units.
//
// Measured (D = 128): 1 token, 12 heads over 4096 rows 8.6 us, over 65536 39 us (3.2 TB/s
// of the cache); 32 x 16 heads over up to 8191 rows with gate and weights 96 us (3.8 TB/s).
// A tile of 32 rows takes a warp 690 to 730 instructions; with 16 x 16 heads over 8192 rows
// (78 us) the kernel takes 72 us without the copies and 63 without the arithmetic.
#include <cooperative_groups.h>

#include "kv4_mma.cuh"
#include "launch.h"

namespace hrm {
namespace {

namespace cg = cooperative_groups;

constexpr int kTileRows = 32;
constexpr int kStages = 2;
constexpr int kBlockRows = 8;   // query rows per item
constexpr int kClusterMax = 8;  // CTAs of a cluster
constexpr int kClusterWarps = 8, kShareWarps = 4;  // warps of a CTA, in the two launch forms
constexpr int64_t kSplitRows = 4096;  // cache rows up to which a cluster serves an item, whatever its CTAs
constexpr uint32_t kAll = 0xffffffffu;

template <int D>
struct Shape {
  static constexpr int kCodeBytes = D / 2;       // per row
  static constexpr int kGroups = D / kKv4Group;  // words of scales per row
  static constexpr int kStageBytes = kTileRows * 2 * (kCodeBytes + 4 * kGroups);
  static constexpr int kLaneWords = D / 32;  // 32-bit words of k codes per lane and row
};
// Of a CTA of W warps.
template <int D, int W>
struct Cta {
  // the warps' rings; after the loop, their partial results
  static constexpr int kSmem = W * (kStages * Shape<D>::kStageBytes > kBlockRows * D * 4
                                        ? kStages * Shape<D>::kStageBytes
                                        : kBlockRows * D * 4);
  // CTAs per SM that the registers allow (64 K): 128 per thread up to D = 128, else 255
  static constexpr int kPerSm = (D <= 128 ? 16 : 8) / W;
};

// A partial result in the workspace: rows x D sums, then the rows' maxima, sums and
// masks of groups that are not finite, then a Cut.  In floats, a multiple of 4.
__host__ __device__ inline int64_t part_floats(int rows, int64_t head_dim) { return rows * (head_dim + 4) + 8; }

// What the joining launch has to know of a partial result: the item, the CTA that
// its rows begin in and the slot of its part there, the number of CTAs, and the
// cache rows of this part.
struct Cut {
  int item, c0, slot0, n;  // item < 0: no partial result
  int from, to, unused[2];
};

// Which queries an item holds.  (32-bit indices: a 64-bit division costs a hundred
// instructions, and every thread of every CTA divides here.)
struct Item {
  int bh, b, hk, row0, nrows;
};
__device__ __forceinline__ Item item_of(const AttnArgs& a, unsigned item) {
  const unsigned rows = a.group * a.seq, blocks = (rows + kBlockRows - 1) / kBlockRows;
  const unsigned bh = blocks == 1 ? item : item / blocks, b = bh / (unsigned)a.kv_heads;
  const unsigned row0 = (item - bh * blocks) * kBlockRows;
  return {(int)bh, (int)b, (int)(bh - b * a.kv_heads), (int)row0, (int)min(rows - row0, (unsigned)kBlockRows)};
}
// Head and query position of an item's query row r.
struct Place {
  int h, s;
};
__device__ __forceinline__ Place place_of(const AttnArgs& a, const Item& x, int r) {
  const unsigned row = x.row0 + r, seq = a.seq, g = seq == 1 ? row : row / seq;
  return {(int)(x.hk * a.group + g), (int)(row - g * seq)};
}

// Where tile row r of k goes: the mma's row 2t + e of 8 is cache row t + 4e,
// so that the rows of a lane's probabilities are 4 apart and a warp's
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

// A lane's share of a tile's copies: where it reads in the head's buffers (at
// their first row) and where it writes in a stage.  Piece i of a lane is 512 i bytes
// further in global memory, and its place in the stage is the lane's first one
// plus a constant: a whole tile costs an address per buffer and a copy
// instruction per piece.  (Computing each piece's place took 15% of the kernel's
// instructions.)
template <int D>
struct Loader {
  using T = Shape<D>;
  static constexpr int kPieces = T::kCodeBytes / 16;  // per row
  static constexpr int kScaleUnit = D % 128 == 0 ? 16 : 8;
  static constexpr int kScalePieces = 4 * T::kGroups / kScaleUnit;
  static constexpr int kCodes = kTileRows * T::kCodeBytes, kScales = kTileRows * 4 * T::kGroups;
  static constexpr bool kEven = D != 192;  // 32 lanes' pieces are whole rows
  static constexpr int kRows = 32 / kPieces, kScaleRows = 32 / kScalePieces;  // rows per step of 32 lanes, if so
  const uint8_t *k, *v, *ks, *vs;
  uint32_t dk, dv, dks;
  int lane;

  __device__ __forceinline__ Loader(const Kv4View& c, int64_t head_row, int lane_) : lane(lane_) {
    k = c.k_codes + head_row * T::kCodeBytes;
    v = c.v_codes + head_row * T::kCodeBytes;
    ks = reinterpret_cast<const uint8_t*>(c.k_scales) + head_row * (4 * T::kGroups);
    vs = reinterpret_cast<const uint8_t*>(c.v_scales) + head_row * (4 * T::kGroups);
    dk = place_k(lane);
    dv = place_v(lane);
    dks = place_ks(lane);
  }
  __device__ __forceinline__ static uint32_t place_k(int idx) {
    return k_place(idx / kPieces) * T::kCodeBytes + 16 * (idx % kPieces);
  }
  __device__ __forceinline__ static uint32_t place_v(int idx) {
    return kCodes + (idx / kPieces) * T::kCodeBytes + 16 * v_piece<D>(idx / kPieces, idx % kPieces);
  }
  __device__ __forceinline__ static uint32_t place_ks(int idx) {
    return 2 * kCodes + k_place(idx / kScalePieces) * 4 * T::kGroups + (idx % kScalePieces) * kScaleUnit;
  }
  // k_place(first + r) - k_place(r) for a step's first row and r < its rows (both multiples of the step)
  __host__ __device__ static constexpr int k_shift(int first, int rows) {
    return rows >= 8 ? first : (first & ~7) + ((first >> 2) & 1);
  }

  // Rows [32 * tile, + 32), of which those past `limit` become zeros.
  __device__ __forceinline__ void operator()(uint32_t stage, int tile, int limit) const {
    const int left = limit - tile * kTileRows;
    const uint8_t* gk = k + (int64_t)tile * kCodes;
    const uint8_t* gv = v + (int64_t)tile * kCodes;
    const uint8_t* gks = ks + (int64_t)tile * kScales;
    const uint8_t* gvs = vs + (int64_t)tile * kScales;
    if (kEven && left >= kTileRows) {
      gk += 16 * lane;
      gv += 16 * lane;
      gks += kScaleUnit * lane;
      gvs += kScaleUnit * lane;
      const uint32_t vsd = stage + 2 * kCodes + kScales + kScaleUnit * lane;
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        cp_async16(stage + dk + k_shift(i * kRows, kRows) * T::kCodeBytes, gk + 512 * i);
        cp_async16(stage + dv + i * kRows * T::kCodeBytes, gv + 512 * i);
      }
#pragma unroll
      for (int i = 0; i < kScalePieces; ++i) {
        cp_async_zfill<kScaleUnit>(stage + dks + k_shift(i * kScaleRows, kScaleRows) * 4 * T::kGroups,
                                   gks + 32 * kScaleUnit * i, true);
        cp_async_zfill<kScaleUnit>(vsd + 32 * kScaleUnit * i, gvs + 32 * kScaleUnit * i, true);
      }
    } else {  // what is past the limit is not read; its address is the head's first row
#pragma unroll 1
      for (int i = 0; i < kPieces; ++i) {
        const int idx = i * 32 + lane;
        const bool ok = idx / kPieces < left;
        cp_async_zfill<16>(stage + place_k(idx), ok ? gk + 16 * idx : k, ok);
        cp_async_zfill<16>(stage + place_v(idx), ok ? gv + 16 * idx : v, ok);
      }
#pragma unroll 1
      for (int i = 0; i < kScalePieces; ++i) {
        const int idx = i * 32 + lane;
        const bool ok = idx / kScalePieces < left;
        cp_async_zfill<kScaleUnit>(stage + place_ks(idx), ok ? gks + kScaleUnit * idx : ks, ok);
        cp_async_zfill<kScaleUnit>(stage + 2 * kCodes + kScales + kScaleUnit * idx, ok ? gvs + kScaleUnit * idx : vs,
                                   ok);
      }
    }
  }
};

// The two mma steps of one k word of 16 cache rows: wa, wb of the lane's rows g and g + 8.
__device__ __forceinline__ void k_steps(float (&acc)[4], uint32_t wa, uint32_t wb, const uint32_t (&s2)[2],
                                        const uint32_t (&z2)[2], const uint32_t (&q)[4]) {
  mma_bf16(acc, fma_bf16x2(kv4_pair<0>(wa), s2[0], z2[0]), fma_bf16x2(kv4_pair<0>(wb), s2[1], z2[1]),
           fma_bf16x2(kv4_pair<1>(wa), s2[0], z2[0]), fma_bf16x2(kv4_pair<1>(wb), s2[1], z2[1]), q[0], q[1]);
  mma_bf16(acc, fma_bf16x2(kv4_pair<2>(wa), s2[0], z2[0]), fma_bf16x2(kv4_pair<2>(wb), s2[1], z2[1]),
           fma_bf16x2(kv4_pair<3>(wa), s2[0], z2[0]), fma_bf16x2(kv4_pair<3>(wb), s2[1], z2[1]), q[2], q[3]);
}

// Transposes the 8x8 matrix of 16-bit elements whose row g, columns 2t and 2t + 1 lane (g, t) holds.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
  return r;
}

// One 16-row step of 32 output elements: elements P and P + 1 (words a, in the mma's row g)
// and 4 + P, 5 + P (words b, row g + 8) of each lane's 8; index 0: cache rows t and t + 4 of
// the step, 1: t + 8 and t + 12.  The products of two elements alternate, so that lo does
// not wait for hi's sum.
template <int P>
__device__ __forceinline__ void v_step(float (*o)[4], const uint32_t (&a)[2], const uint32_t (&b)[2],
                                       const uint32_t (&s2)[2], const uint32_t (&z2)[2], const uint32_t (&hi)[2],
                                       const uint32_t (&lo)[2]) {
  uint32_t x[2][4];
  x[0][0] = fma_bf16x2(kv4_pair<P>(a[0]), s2[0], z2[0]);
  x[0][1] = fma_bf16x2(kv4_pair<P>(b[0]), s2[0], z2[0]);
  x[0][2] = fma_bf16x2(kv4_pair<P>(a[1]), s2[1], z2[1]);
  x[0][3] = fma_bf16x2(kv4_pair<P>(b[1]), s2[1], z2[1]);
  x[1][0] = fma_bf16x2(kv4_pair<P + 1>(a[0]), s2[0], z2[0]);
  x[1][1] = fma_bf16x2(kv4_pair<P + 1>(b[0]), s2[0], z2[0]);
  x[1][2] = fma_bf16x2(kv4_pair<P + 1>(a[1]), s2[1], z2[1]);
  x[1][3] = fma_bf16x2(kv4_pair<P + 1>(b[1]), s2[1], z2[1]);
#pragma unroll
  for (int e = 0; e < 2; ++e) mma_bf16(o[P + e], x[e][0], x[e][1], x[e][2], x[e][3], hi[0], hi[1]);
#pragma unroll
  for (int e = 0; e < 2; ++e) mma_bf16(o[P + e], x[e][0], x[e][1], x[e][2], x[e][3], lo[0], lo[1]);
}

// The same with hi and lo in the even and odd columns of one operand.
template <int P>
__device__ __forceinline__ void v_step_one(float (*o)[4], const uint32_t (&a)[2], const uint32_t (&b)[2],
                                           const uint32_t (&s2)[2], const uint32_t (&z2)[2], const uint32_t (&p)[2]) {
  mma_bf16(o[P], fma_bf16x2(kv4_pair<P>(a[0]), s2[0], z2[0]), fma_bf16x2(kv4_pair<P>(b[0]), s2[0], z2[0]),
           fma_bf16x2(kv4_pair<P>(a[1]), s2[1], z2[1]), fma_bf16x2(kv4_pair<P>(b[1]), s2[1], z2[1]), p[0], p[1]);
}

__device__ __forceinline__ float sigmoid_gate(uint16_t g) { return gate_factor(bf16_to_f32(g)); }

// Writes elements d, d + 1 of query row r of the item: gated, rounded once.
__device__ __forceinline__ int64_t out_at(const AttnArgs& a, const Item& x, int64_t head_dim, int r, int d) {
  const Place p = place_of(a, x, r);
  return (((int64_t)x.b * a.seq + p.s) * a.heads + p.h) * head_dim + d;
}
__device__ __forceinline__ uint32_t gate_at(const AttnArgs& a, int64_t at) {
  return *reinterpret_cast<const uint32_t*>(a.gate + at);
}
__device__ __forceinline__ void store_out(const AttnArgs& a, int64_t at, int d, float v0, float v1, uint32_t bad,
                                          uint32_t gate) {
  if (bad >> (d / kKv4Group) & 1u) v0 = v1 = __int_as_float(0x7fc00000);
  if (a.gate != nullptr) {
    v0 *= sigmoid_gate((uint16_t)gate);
    v1 *= sigmoid_gate((uint16_t)(gate >> 16));
  }
  *reinterpret_cast<uint32_t*>(a.out + at) = pack_bf16x2(v0, v1);
}
__device__ __forceinline__ void store_out(const AttnArgs& a, const Item& x, int64_t head_dim, int r, int d, float v0,
                                          float v1, uint32_t bad) {
  const int64_t at = out_at(a, x, head_dim, r, d);
  store_out(a, at, d, v0, v1, bad, a.gate == nullptr ? 0 : gate_at(a, at));
}
__device__ __forceinline__ void store_lse(const AttnArgs& a, const Item& x, int r, float top, float sum) {
  const Place p = place_of(a, x, r);
  a.lse[((int64_t)x.b * a.heads + p.h) * a.seq + p.s] =
      top == -INFINITY ? -INFINITY : top + log2f(sum);
}
// Adds the probabilities of cache rows [from, to) to their weights, over the query rows in order.
__device__ __forceinline__ void add_weights(const AttnArgs& a, const Item& x, int from, int to, const int* limit,
                                            const float* top, const float* inv) {
  const float* sc = a.scores + ((int64_t)x.bh * (a.group * a.seq) + x.row0) * a.c.cache_len;
  float* w = a.c.weights + (int64_t)x.bh * a.c.cache_len;
  int last = 0;
  for (int r = 0; r < x.nrows; ++r) last = max(last, limit[r]);
  to = min(to, last);
  constexpr int kAhead = 4;  // rows whose loads are in flight at once
  for (int at = from + threadIdx.x; at < to; at += kAhead * blockDim.x) {
    float sum[kAhead], was[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      sum[i] = 0.0f;
      was[i] = at + i * (int)blockDim.x < to ? w[at + i * blockDim.x] : 0.0f;
    }
    for (int r = 0; r < x.nrows; ++r) {
      const float* row = sc + (int64_t)r * a.c.cache_len + at;
      const int lim = min(limit[r], to) - at;
      float v[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) v[i] = i * (int)blockDim.x < lim ? row[i * blockDim.x] : -INFINITY;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (i * (int)blockDim.x < lim) sum[i] += exp2_approx(v[i] - top[r]) * inv[r];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (at + i * (int)blockDim.x < to) w[at + i * blockDim.x] = was[i] + sum[i];
  }
}

// What a CTA has of an item after its tiles: row r's sum of 2^(score - m) v in
// the first floats of the dynamic shared memory, [row][D], and these.
template <int W>
struct Shared {
  float m[W][kBlockRows], l[W][kBlockRows];  // each warp's
  uint32_t bad[W][kBlockRows];
  float c_m[kBlockRows], c_l[kBlockRows];  // the CTA's
  uint32_t c_bad[kBlockRows];
  int limit[kBlockRows];
};

// The CTA's tiles [t0, t1) of item x (of which those past its limit are nothing).
// Ends with a barrier: the results are ready for every thread.
//
// ONE: a single query per item (a decode step without shared kv heads).  All 8
// columns of the scores' B operand hold it, so that every lane has scores of 4 rows
// and takes one of them: the softmax costs one exponential per lane and tile, not
// 8, and hi and lo take the even and odd columns of a single product.
template <int D, int W, bool ONE>
__device__ __forceinline__ void attend(const AttnArgs& a, const Item& x, int t0, int t1, uint8_t* smem, Shared<W>& s) {
  using T = Shape<D>;
  constexpr int kWarps = W;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;

  // the query rows' limits; this lane's queries are row0 + 2t and row0 + 2t + 1
  int limit = 0, lowest = INT32_MAX, my_limit[2] = {0, 0};
  for (int r = 0; r < x.nrows; ++r) {
    const int l = visible_rows(a, x.b, place_of(a, x, r).s);
    limit = max(limit, l);
    lowest = min(lowest, l);
    if (r == 2 * t) my_limit[0] = l;
    if (r == 2 * t + 1) my_limit[1] = l;
    if (threadIdx.x == r) s.limit[r] = l;
  }
  t1 = min(t1, (limit + kTileRows - 1) / kTileRows);
  const Loader<D> load(a.c, (int64_t)x.bh * a.c.cache_len, lane);

  const uint32_t ring = smem_addr(smem) + warp * kStages * T::kStageBytes;
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    const int tile = t0 + warp + i * kWarps;
    if (tile < t1) load(ring + i * T::kStageBytes, tile, limit);
    cp_async_commit();
  }

  // queries as B operands: lane (g, t) has query g's words (ONE: the query's); the
  // words' 8 elements in the order in which kv4_pair yields them
  uint32_t q[T::kLaneWords][4];
  {
    // (the query rows of a kv head lie one after another)
    const int64_t row = ((int64_t)x.b * a.heads + x.hk * a.group) * a.seq + x.row0 + (!ONE && g < x.nrows ? g : 0);
    const uint4* src = a.q + row * (D / 8);
#pragma unroll
    for (int i = 0; i < T::kLaneWords; ++i) {
      uint4 v = ld_keep(src + k_word<D>(i, t));
      if (!ONE && g >= x.nrows) v = make_uint4(0, 0, 0, 0);
      q[i][0] = __byte_perm(v.x, v.z, 0x5410);
      q[i][1] = __byte_perm(v.x, v.z, 0x7632);
      q[i][2] = __byte_perm(v.y, v.w, 0x5410);
      q[i][3] = __byte_perm(v.y, v.w, 0x7632);
    }
  }

  float o[D / 16][4];  // [4 * word + P]: element P of the word for queries 2t, 2t + 1, then element 4 + P
#pragma unroll
  for (int j = 0; j < D / 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};  // of queries 2t, 2t + 1; l: this lane's rows
  uint32_t bad[2] = {0, 0};  // groups of v that are not finite in a row that the query sees
  float* scores = a.scores == nullptr
                      ? nullptr
                      : a.scores + ((int64_t)x.bh * (a.group * a.seq) + x.row0 + (ONE ? 0 : 2 * t)) * a.c.cache_len;

  // This lane's places in a stage, so that every read below is one of these plus
  // a constant (left to the compiler, the pieces' swizzle was worked out at each read).
  constexpr int kVCodes = kTileRows * T::kCodeBytes, kKScales = 2 * kVCodes;
  constexpr int kVScales = kKScales + kTileRows * 4 * T::kGroups;
  constexpr int kTail = T::kLaneWords % 4;   // words of k codes past the 16-byte pieces
  constexpr int kWords = D / 64;             // words of v codes per lane and row
  constexpr int kSz = kWords == 3 ? 3 : 1;   // their groups: one, but for D = 192
  const int k_at = g * T::kCodeBytes + 16 * t, ks_at = kKScales + 4 * (g * T::kGroups + t);
  const int k_tail = g * T::kCodeBytes + (T::kLaneWords / 4) * 64 + 8 * t;
  const int ks_tail = kKScales + 4 * (g * T::kGroups + T::kLaneWords / 4 * 4 + t / 2);
  const int v_at = kVCodes + t * T::kCodeBytes +
                   (D == 128 ? 16 * v_piece<D>(t, g >> 1) + 8 * (g & 1)
                             : (D == 256 ? 16 * v_piece<D>(t, g) : 4 * kWords * g));
  int vs_at[kSz];
#pragma unroll
  for (int y = 0; y < kSz; ++y) vs_at[y] = kVScales + 4 * (t * T::kGroups + (kWords * g + y) / 4);

  int stage = 0;
  for (int tile = t0 + warp; tile < t1; tile += kWarps) {
    // the other stages' copies are in flight while this one's tile is worked on
    const int next = tile + (kStages - 1) * kWarps;
    const int into = stage == 0 ? kStages - 1 : stage - 1;
    if (next < t1) load(ring + into * T::kStageBytes, next, limit);
    cp_async_commit();
    cp_async_wait<kStages - 1>();
    __syncwarp();
    uint8_t* st = smem + (warp * kStages + stage) * T::kStageBytes;
    auto word = [&](int at) -> uint32_t { return *reinterpret_cast<const uint32_t*>(st + at); };
    const int first = tile * kTileRows;

    // scores: acc[i][2h + e] is query 2t + e on cache row at[i] + 8h
    // (the two 16-row tiles' sums alternate: neither product waits for the one before it)
    float acc[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
#pragma unroll
    for (int j = 0; j < T::kLaneWords / 4; ++j) {
      uint4 w[4];
      uint32_t s2[2][2], z2[2][2];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // rows g, g + 8, g + 16, g + 24
        w[i] = *reinterpret_cast<const uint4*>(st + k_at + 8 * i * T::kCodeBytes + 64 * j);
        const uint32_t y = word(ks_at + 4 * (8 * i * T::kGroups + 4 * j));
        s2[i >> 1][i & 1] = kv4_scale2(y);
        z2[i >> 1][i & 1] = kv4_base2(y);
      }
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          k_steps(acc[i], vget(w[2 * i], y), vget(w[2 * i + 1], y), s2[i], z2[i], q[4 * j + y]);
    }
    if (kTail) {
      constexpr int j = T::kLaneWords / 4;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint2 wa = *reinterpret_cast<const uint2*>(st + k_tail + 16 * i * T::kCodeBytes);
        const uint2 wb = *reinterpret_cast<const uint2*>(st + k_tail + (16 * i + 8) * T::kCodeBytes);
        const uint32_t ya = word(ks_tail + 64 * i * T::kGroups), yb = word(ks_tail + (64 * i + 32) * T::kGroups);
        const uint32_t s2[2] = {kv4_scale2(ya), kv4_scale2(yb)}, z2[2] = {kv4_base2(ya), kv4_base2(yb)};
        k_steps(acc[i], wa.x, wb.x, s2, z2, q[4 * j]);
        k_steps(acc[i], wa.y, wb.y, s2, z2, q[4 * j + 1]);
      }
    }
    uint32_t pair = 0;  // ONE: hi and lo of this lane's probability
    float shift[2];
    if (ONE) {
      // this lane's row: mma row g of 16-row tile t / 2, half t % 2
      const int mine = first + 8 * t + (g >> 1) + 4 * (g & 1);
      float y = (t & 2 ? (t & 1 ? acc[1][2] : acc[1][0]) : (t & 1 ? acc[0][2] : acc[0][0])) * a.scale_log2;
      if (mine >= limit) y = -INFINITY;
      if (scores != nullptr && mine < limit) scores[mine] = y;
      float top = y;
#pragma unroll
      for (int w = 1; w < 32; w *= 2) top = max_nan(top, __shfl_xor_sync(kAll, top, w));
      top = max_nan(top, m[0]);
      if (top != m[0]) {  // the same in every lane
        const float f = m[0] == -INFINITY ? 0.0f : exp2_approx(m[0] - top);
        l[0] *= f;
        m[0] = top;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[j][0] *= f;
          o[j][1] *= f;
          o[j][2] *= f;
          o[j][3] *= f;
        }
      }
      const float p = exp2_approx(y - (top == -INFINITY ? 0.0f : top));
      l[0] += p;
      const float hi = bf16_lo(pack_bf16x2(p, 0.0f));
      pair = pack_bf16x2(hi, p - hi);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] *= a.scale_log2;
      // the cache rows of mma rows g (k_place's inverse), and 8 and 16 further
      const int at = first + (g >> 1) + 4 * (g & 1);
      const bool border = first + kTileRows > lowest;  // some query does not see some row
      if (border) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (at + 16 * i + 8 * (e >> 1) >= my_limit[e & 1]) acc[i][e] = -INFINITY;
      }
      if (scores != nullptr) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* to = scores + e * a.c.cache_len + at;
          if (2 * t + e < x.nrows) {
            if (!border) {
              to[0] = acc[0][e];
              to[8] = acc[0][2 + e];
              to[16] = acc[1][e];
              to[24] = acc[1][2 + e];
            } else {
#pragma unroll
              for (int h = 0; h < 4; ++h)
                if (at + 8 * h < my_limit[e]) to[8 * h] = acc[h >> 1][2 * (h & 1) + e];
            }
          }
        }
      }
      float top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = max_nan(max_nan(acc[0][e], acc[0][2 + e]), max_nan(acc[1][e], acc[1][2 + e]));
#pragma unroll
        for (int w = 4; w < 32; w *= 2) top[e] = max_nan(top[e], __shfl_xor_sync(kAll, top[e], w));
        top[e] = max_nan(top[e], m[e]);
      }
      if (__any_sync(kAll, top[0] != m[0] || top[1] != m[1])) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          f[e] = m[e] == -INFINITY ? 0.0f : exp2_approx(m[e] - top[e]);
          l[e] *= f[e];
          m[e] = top[e];
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[j][0] *= f[0];
          o[j][1] *= f[1];
          o[j][2] *= f[0];
          o[j][3] *= f[1];
        }
      }
      shift[0] = m[0] == -INFINITY ? 0.0f : m[0];
      shift[1] = m[1] == -INFINITY ? 0.0f : m[1];

      // A row that some of the queries must not see, holding a value that is not
      // finite: 0 * NaN would reach them.  Such groups are read as zeros here and
      // the queries that do see them are marked.
      if (border && lowest < limit) {
        uint32_t* vs = reinterpret_cast<uint32_t*>(st + kVScales);
        bool any = false;  // in this lane's row
#pragma unroll
        for (int x = 0; x < T::kGroups; ++x) any |= kv4_not_finite(vs[lane * T::kGroups + x]);
        if (__any_sync(kAll, any)) {
#pragma unroll 1
          for (int r = 0; r < kTileRows; ++r) {
            const bool mine = lane < T::kGroups && kv4_not_finite(vs[r * T::kGroups + lane]);
            const uint32_t found = __ballot_sync(kAll, mine);
            if (mine) vs[r * T::kGroups + lane] = 0;
            if (first + r < my_limit[0]) bad[0] |= found;
            if (first + r < my_limit[1]) bad[1] |= found;
          }
          __syncwarp();
        }
      }
    }

#pragma unroll
    for (int i = 0; i < 2; ++i) {
      // probabilities as B operands: rows (t, t + 4) of query g, then (t + 8, t + 12)
      uint32_t hi[2], lo[2];
      if (ONE) {  // of lanes (2t, 2i + h) and (2t + 1, 2i + h); column g: hi if g is even, else lo
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t w0 = __shfl_sync(kAll, pair, 8 * t + 2 * i + h);
          const uint32_t w1 = __shfl_sync(kAll, pair, 8 * t + 4 + 2 * i + h);
          hi[h] = __byte_perm(w0, w1, g & 1 ? 0x7632 : 0x5410);
        }
      }
#pragma unroll
      for (int h = 0; h < 2 && !ONE; ++h) {
        const float p0 = exp2_approx(acc[i][2 * h] - shift[0]), p1 = exp2_approx(acc[i][2 * h + 1] - shift[1]);
        l[0] += p0;
        l[1] += p1;
        const uint32_t x2 = pack_bf16x2(p0, p1);
        hi[h] = transpose8(x2);
        lo[h] = transpose8(pack_bf16x2(p0 - bf16_lo(x2), p1 - bf16_hi(x2)));
      }
      uint32_t w[4][kWords], sz[4][kSz];
#pragma unroll
      for (int r = 0; r < 4; ++r) {  // cache rows t + 4r of the 16
        const int step = 16 * i + 4 * r;
        const uint8_t* from = st + v_at + step * T::kCodeBytes;
        if (D == 128) {
          const uint2 y = *reinterpret_cast<const uint2*>(from);
          w[r][0] = y.x;
          w[r][kWords > 1 ? 1 : 0] = y.y;
        } else if (D == 256) {
          const uint4 y = *reinterpret_cast<const uint4*>(from);
#pragma unroll
          for (int z = 0; z < kWords; ++z) w[r][z] = vget(y, z);
        } else {
#pragma unroll
          for (int y = 0; y < kWords; ++y) w[r][y] = *reinterpret_cast<const uint32_t*>(from + 4 * y);
        }
#pragma unroll
        for (int y = 0; y < kSz; ++y) sz[r][y] = word(vs_at[y] + 4 * step * T::kGroups);
      }
#pragma unroll
      for (int y = 0; y < kWords; ++y) {
        constexpr int kOne = kSz - 1;
        const int u = kOne ? y : 0;
        const uint32_t s2[2] = {__byte_perm(sz[0][u], sz[1][u], 0x5410), __byte_perm(sz[2][u], sz[3][u], 0x5410)};
        const uint32_t z2[2] = {__byte_perm(sz[0][u], sz[1][u], 0x7632), __byte_perm(sz[2][u], sz[3][u], 0x7632)};
        // kv4_pair takes a nibble of each half: put two rows' half words together
        const uint32_t va[2] = {__byte_perm(w[0][y], w[1][y], 0x5410), __byte_perm(w[2][y], w[3][y], 0x5410)};
        const uint32_t vb[2] = {__byte_perm(w[0][y], w[1][y], 0x7632), __byte_perm(w[2][y], w[3][y], 0x7632)};
        if (ONE) {
          v_step_one<0>(o + 4 * y, va, vb, s2, z2, hi);
          v_step_one<1>(o + 4 * y, va, vb, s2, z2, hi);
          v_step_one<2>(o + 4 * y, va, vb, s2, z2, hi);
          v_step_one<3>(o + 4 * y, va, vb, s2, z2, hi);
        } else {
          v_step<0>(o + 4 * y, va, vb, s2, z2, hi, lo);
          v_step<2>(o + 4 * y, va, vb, s2, z2, hi, lo);
        }
      }
    }
    __syncwarp();  // every lane is done with this stage's buffers
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  cp_async_wait<0>();

  // ---- join the warps
  __syncthreads();
  float* part = reinterpret_cast<float*>(smem);  // [warp][row][D], then [row][D]
  if (ONE) {
#pragma unroll
    for (int w = 1; w < 32; w *= 2) l[0] += __shfl_xor_sync(kAll, l[0], w);
    if (lane == 0) {
      s.m[warp][0] = m[0];
      s.l[warp][0] = l[0];
      s.bad[warp][0] = 0;
    }
    if (t == 0) {  // columns 0 and 1: hi's and lo's sums
      float4* dst = reinterpret_cast<float4*>(part + warp * kBlockRows * D + (D / 8) * g);
#pragma unroll
      for (int y = 0; y < D / 64; ++y) {
        dst[2 * y] = make_float4(o[4 * y][0] + o[4 * y][1], o[4 * y + 1][0] + o[4 * y + 1][1],
                                 o[4 * y + 2][0] + o[4 * y + 2][1], o[4 * y + 3][0] + o[4 * y + 3][1]);
        dst[2 * y + 1] = make_float4(o[4 * y][2] + o[4 * y][3], o[4 * y + 1][2] + o[4 * y + 1][3],
                                     o[4 * y + 2][2] + o[4 * y + 2][3], o[4 * y + 3][2] + o[4 * y + 3][3]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int w = 4; w < 32; w *= 2) l[e] += __shfl_xor_sync(kAll, l[e], w);
      if (g == 0) {
        s.m[warp][2 * t + e] = m[e];
        s.l[warp][2 * t + e] = l[e];
        s.bad[warp][2 * t + e] = bad[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (2 * t + e < x.nrows) {
        float4* dst = reinterpret_cast<float4*>(part + (warp * kBlockRows + 2 * t + e) * D + (D / 8) * g);
#pragma unroll
        for (int y = 0; y < D / 64; ++y) {
          dst[2 * y] = make_float4(o[4 * y][e], o[4 * y + 1][e], o[4 * y + 2][e], o[4 * y + 3][e]);
          dst[2 * y + 1] = make_float4(o[4 * y][2 + e], o[4 * y + 1][2 + e], o[4 * y + 2][2 + e], o[4 * y + 3][2 + e]);
        }
      }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < x.nrows * D; e += kWarps * 32) {
    const int r = e / D, d = e % D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = max_nan(top, s.m[w][r]);
    float sum = 0.0f, norm = 0.0f;
    uint32_t any = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = s.m[w][r] == -INFINITY ? 0.0f : exp2_approx(s.m[w][r] - top);
      sum += f * part[(w * kBlockRows + r) * D + d];
      norm += f * s.l[w][r];
      any |= s.bad[w][r];
    }
    part[e] = sum;  // warp 0's element of the same thread's own (r, d)
    if (d == 0) {
      s.c_m[r] = top;
      s.c_l[r] = norm;
      s.c_bad[r] = any;
    }
  }
  __syncthreads();
}

// One launch for short caches: `count` CTAs, a cluster, share each item.
template <int D, bool ONE>
__global__ void __launch_bounds__(kClusterWarps * 32, Cta<D, kClusterWarps>::kPerSm)
    kv4_decode_kernel(const AttnArgs a, const int count) {
  constexpr int kWarps = kClusterWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Shared<kWarps> s;
  grid_dependency_begin();
  const unsigned item = count == 1 ? blockIdx.x : blockIdx.x / (unsigned)count;
  const int rank = (int)(blockIdx.x - item * count);
  const Item x = item_of(a, item);
  const int tiles = (visible_rows(a, x.b, a.seq - 1) + kTileRows - 1) / kTileRows;
  // (a cluster's items are short: no overflow)
  const int t0 = (unsigned)(tiles * rank) / (unsigned)count, t1 = (unsigned)(tiles * (rank + 1)) / (unsigned)count;
  // the gate of this thread's first output, read while the tiles are worked on
  const int e0 = rank * kWarps * 32 + threadIdx.x;
  uint32_t gate0 = 0;
  if (a.gate != nullptr && e0 < x.nrows * (D / 2))
    gate0 = gate_at(a, out_at(a, x, D, e0 / (D / 2), 2 * (e0 % (D / 2))));
  attend<D, kWarps, ONE>(a, x, t0, t1, smem, s);

  cg::cluster_group cluster = cg::this_cluster();
  if (count > 1) cluster.sync();
  // join the cluster's CTAs; each writes its share of the output
  float* part = reinterpret_cast<float*>(smem);
  __shared__ float f_inv[kBlockRows], f_m[kBlockRows], f_w[kClusterMax][kBlockRows];
  __shared__ uint32_t f_bad[kBlockRows];
  if (threadIdx.x < x.nrows) {
    const int r = threadIdx.x;
    float top = -INFINITY, sum = 0.0f;
    uint32_t any = 0;
    for (int y = 0; y < count; ++y) top = max_nan(top, *cluster.map_shared_rank(&s.c_m[r], y));
    for (int y = 0; y < count; ++y) {
      const float cm = *cluster.map_shared_rank(&s.c_m[r], y);
      const float f = cm == -INFINITY ? 0.0f : exp2_approx(cm - top);
      f_w[y][r] = f;
      sum += f * *cluster.map_shared_rank(&s.c_l[r], y);
      any |= *cluster.map_shared_rank(&s.c_bad[r], y);
    }
    f_m[r] = top;
    f_inv[r] = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row that sees nothing: 0
    f_bad[r] = any;
    if (a.lse != nullptr && rank == 0) store_lse(a, x, r, top, sum);
  }
  __syncthreads();
  for (int e = e0; e < x.nrows * (D / 2); e += count * kWarps * 32) {
    const int r = e / (D / 2), d = 2 * (e % (D / 2));
    float v0 = 0.0f, v1 = 0.0f;
    for (int y = 0; y < count; ++y) {
      const float2 v = *reinterpret_cast<const float2*>(cluster.map_shared_rank(part, y) + r * D + d);
      v0 += f_w[y][r] * v.x;
      v1 += f_w[y][r] * v.y;
    }
    const int64_t at = out_at(a, x, D, r, d);
    store_out(a, at, d, v0 * f_inv[r], v1 * f_inv[r], f_bad[r],
              e == e0 ? gate0 : (a.gate == nullptr ? 0 : gate_at(a, at)));
  }
  // this CTA's rows, whose scores this CTA wrote
  if (a.scores != nullptr && a.lse == nullptr) add_weights(a, x, t0 * kTileRows, t1 * kTileRows, s.limit, f_m, f_inv);
  if (count > 1) cluster.sync();  // the shares are read: no CTA may leave before
}

// ---- equal shares of all items' rows, for long caches
//
// A sequence has `per` items (kv heads x blocks of query rows) of the same number
// of 128-row blocks, and one more for what a piece of work costs beside its rows
// (32 x 16 heads over up to 8191 rows with weights 96 us; without it, where a share of
// many short sequences was as long as one of a long one's rows, 111; two: 94, but 83
// against 82 without weights).  All blocks of all items in order are the
// positions [0, total); CTA c of G = min(the grid, total) has the positions
// [total * c / G, total * (c + 1) / G), at least one.

constexpr int kShareRows = kTileRows * kShareWarps;  // rows of a position: a tile per warp
constexpr int kStart = 1;  // positions that an item's start counts as

struct Line {
  unsigned per, total, shares;
  unsigned mine;  // blocks of the sequence of this lane's number
};
__device__ __forceinline__ unsigned blocks_of(const AttnArgs& a, int b) {
  return kStart + (visible_rows(a, b, a.seq - 1) + kShareRows - 1) / kShareRows;
}
__device__ __forceinline__ Line line_of(const AttnArgs& a) {  // every lane of the warp
  Line y;
  y.per = a.kv_heads * (unsigned)((a.group * a.seq + kBlockRows - 1) / kBlockRows);
  const int lane = threadIdx.x & 31;
  y.mine = lane < a.batch ? blocks_of(a, lane) : 0;
  unsigned sum = y.mine;
  for (int b = lane + 32; b < a.batch; b += 32) sum += blocks_of(a, b);
  y.total = __reduce_add_sync(kAll, sum) * y.per;
  y.shares = min(gridDim.x, y.total);
  return y;
}
__device__ __forceinline__ unsigned share_begin(const Line& y, unsigned c) {
  return (unsigned)((uint64_t)y.total * c / y.shares);
}
__device__ __forceinline__ unsigned share_at(const Line& y, unsigned pos) {  // the CTA that has pos
  return (unsigned)(((uint64_t)(pos + 1) * y.shares - 1) / y.total);
}
// The item at a position: its first position, its number of positions, its index.
struct Span {
  unsigned first, count, item;
};
__device__ __forceinline__ Span span_at(const AttnArgs& a, const Line& y, unsigned pos) {  // every lane of the warp
  const int lane = threadIdx.x & 31;
  unsigned base = 0;  // first position of sequence b0
  for (int b0 = 0;; b0 += 32) {
    const unsigned n = b0 == 0 ? y.mine : (b0 + lane < a.batch ? blocks_of(a, b0 + lane) : 0);
    unsigned sum = n * y.per;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const unsigned v = __shfl_up_sync(kAll, sum, o);
      if (lane >= o) sum += v;
    }
    const uint32_t past = __ballot_sync(kAll, pos < base + sum);  // sequences that end past pos
    if (past != 0 || b0 + 32 >= a.batch) {
      const int l = past == 0 ? 0 : __ffs(past) - 1;
      const unsigned count = __shfl_sync(kAll, n, l), end = base + __shfl_sync(kAll, sum, l);
      const unsigned start = end - count * y.per, i = (pos - start) / count;
      return {start + i * count, count, (b0 + l) * y.per + i};
    }
    base += __shfl_sync(kAll, sum, 31);
  }
}

// Where CTA c leaves its part of an item: slot 0 if the part is the first of its share, else slot 1.
__device__ __forceinline__ float* part_of(float* parts, unsigned c, int slot, int rows, int64_t head_dim) {
  return parts + (2 * (int64_t)c + slot) * part_floats(rows, head_dim);
}

template <int D, bool ONE>
__global__ void __launch_bounds__(kShareWarps * 32, Cta<D, kShareWarps>::kPerSm)
    kv4_decode_shares_kernel(const AttnArgs a, float* parts, const int rows) {
  constexpr int kWarps = kShareWarps;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Shared<kWarps> s;
  __shared__ float f_inv[kBlockRows];
  grid_dependency_begin();
  const Line y = line_of(a);
  const int64_t cut_at = rows * (D + 4);  // of the Cut in a part
  if (threadIdx.x < 2)
    reinterpret_cast<Cut*>(part_of(parts, blockIdx.x, threadIdx.x, rows, D) + cut_at)->item = -1;
  if (blockIdx.x >= y.shares) return;
  const unsigned begin = share_begin(y, blockIdx.x), end = share_begin(y, blockIdx.x + 1);
  float* part = reinterpret_cast<float*>(smem);
  for (unsigned pos = begin; pos < end;) {
    const Span span = span_at(a, y, pos);
    const Item x = item_of(a, span.item);
    const unsigned stop = min(end, span.first + span.count);
    const int t0 = max((int)(pos - span.first) - kStart, 0) * kWarps;
    const int t1 = max((int)(stop - span.first) - kStart, 0) * kWarps;
    attend<D, kWarps, ONE>(a, x, t0, t1, smem, s);
    if (stop - pos == span.count) {  // the whole item
      if (threadIdx.x < x.nrows) {
        const int r = threadIdx.x;
        f_inv[r] = s.c_l[r] == 0.0f ? 0.0f : 1.0f / s.c_l[r];
        if (a.lse != nullptr) store_lse(a, x, r, s.c_m[r], s.c_l[r]);
      }
      __syncthreads();
      for (int e = threadIdx.x; e < x.nrows * (D / 2); e += kWarps * 32) {
        const int r = e / (D / 2), d = 2 * (e % (D / 2));
        store_out(a, x, D, r, d, part[r * D + d] * f_inv[r], part[r * D + d + 1] * f_inv[r], s.c_bad[r]);
      }
      if (a.scores != nullptr && a.lse == nullptr) add_weights(a, x, 0, t1 * kTileRows, s.limit, s.c_m, f_inv);
    } else {
      float* mine = part_of(parts, blockIdx.x, pos == begin ? 0 : 1, rows, D);
      for (int e = threadIdx.x; e < x.nrows * D; e += kWarps * 32) mine[e] = part[e];
      if (threadIdx.x < x.nrows) {
        float* tail = mine + rows * D + threadIdx.x;
        tail[0] = s.c_m[threadIdx.x];
        tail[rows] = s.c_l[threadIdx.x];
        tail[2 * rows] = __uint_as_float(s.c_bad[threadIdx.x]);
      }
      if (threadIdx.x == 0) {
        const unsigned c0 = share_at(y, span.first), c1 = share_at(y, span.first + span.count - 1);
        Cut* cut = reinterpret_cast<Cut*>(mine + cut_at);
        cut->item = (int)span.item;
        cut->c0 = (int)c0;
        // parts of the CTAs after c0 are the first of their shares; c0's is where the item begins
        cut->slot0 = span.first > share_begin(y, c0) ? 1 : 0;
        cut->n = (int)(c1 - c0) + 1;
        cut->from = t0 * kTileRows;
        cut->to = t1 * kTileRows;
      }
    }
    __syncthreads();  // the results are read: the ring may be filled again
    pos = stop;
  }
}

constexpr int kJoinThreads = 256;

// Joins the items that were cut.  CTA c has the partial results of share c: it writes
// the output of the item that begins there, and adds the probabilities of its own
// rows to the weights.  Its latency is that of three dependent reads (the Cut; the
// maxima and the first sums; the other sums).
__global__ void __launch_bounds__(kJoinThreads, 4) kv4_join_kernel(const AttnArgs a, float* parts, const int rows,
                                                                const int head_dim) {
  extern __shared__ float f_w[];  // [row][shares of the item]
  __shared__ float f_m[kBlockRows], f_inv[kBlockRows];
  __shared__ uint32_t f_bad[kBlockRows];
  __shared__ int s_limit[kBlockRows];
  __shared__ float4 s_sum[kJoinThreads];
  grid_dependency_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t each = part_floats(rows, head_dim);
  int4 cuts[2][2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const float* tail = part_of(parts, blockIdx.x, side, rows, head_dim) + rows * (head_dim + 4);
    const int4* c = reinterpret_cast<const int4*>(tail);
    cuts[side][0] = c[0];
    cuts[side][1] = c[1];
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int item = cuts[side][0].x, c0 = cuts[side][0].y, slot0 = cuts[side][0].z, n = cuts[side][0].w;
    if (item < 0) continue;
    const bool first = c0 == (int)blockIdx.x;  // the item begins here
    const bool adds = a.scores != nullptr && a.lse == nullptr;
    if (!first && !adds) continue;
    const Item x = item_of(a, item);
    const float* base = part_of(parts, c0, 0, rows, head_dim);
    auto at = [&](int i) -> const float* { return base + (2 * (int64_t)i + (i == 0 ? slot0 : 0)) * each; };

    // a thread has 4 elements; the parts are shared out over the threads left
    constexpr int kAhead = 8;  // parts whose sums are read before their factors are known
    const int quads = x.nrows * (head_dim / 4), ways = max(1, kJoinThreads / quads);
    const int way = ways == 1 ? 0 : threadIdx.x / quads;
    float4 ahead[kAhead];
    const int e_first = ways == 1 ? threadIdx.x : threadIdx.x % quads;
    const bool mine = e_first < quads && way < ways && first;
    if (mine) {
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (way + k * ways < n) ahead[k] = *reinterpret_cast<const float4*>(at(way + k * ways) + 4 * e_first);
    }
    for (int r = warp; r < x.nrows; r += kJoinThreads / 32) {
      float top = -INFINITY, sum = 0.0f;
      uint32_t any = 0;
      for (int i = lane; i < n; i += 32) top = max_nan(top, at(i)[rows * head_dim + r]);
#pragma unroll
      for (int o = 16; o > 0; o /= 2) top = max_nan(top, __shfl_xor_sync(kAll, top, o));
      for (int i = lane; i < n; i += 32) {
        const float* tail = at(i) + rows * head_dim + r;
        const float m = tail[0], l = tail[rows];
        any |= __float_as_uint(tail[2 * rows]);
        const float f = m == -INFINITY ? 0.0f : exp2_approx(m - top);
        sum += f * l;
        f_w[r * n + i] = f;
      }
#pragma unroll
      for (int o = 16; o > 0; o /= 2) sum += __shfl_xor_sync(kAll, sum, o);
      any = __reduce_or_sync(kAll, any);
      if (lane == 0) {
        s_limit[r] = visible_rows(a, x.b, place_of(a, x, r).s);
        f_m[r] = top;
        f_inv[r] = sum == 0.0f ? 0.0f : 1.0f / sum;
        f_bad[r] = any;
        if (a.lse != nullptr && first) store_lse(a, x, r, top, sum);
      }
    }
    __syncthreads();
    if (first) {
      for (int e0 = 0; e0 < quads; e0 += kJoinThreads) {
        const int e = e0 + e_first;
        const bool ok = e < quads && way < ways;
        const int r = e / (head_dim / 4), d = 4 * (e % (head_dim / 4));
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto add = [&](const float4& v, float f) {
          sum.x += f * v.x;
          sum.y += f * v.y;
          sum.z += f * v.z;
          sum.w += f * v.w;
        };
        if (ok) {
#pragma unroll
          for (int k = 0; k < kAhead; ++k) {
            const int i = way + k * ways;
            if (i < n) add(e0 == 0 ? ahead[k] : *reinterpret_cast<const float4*>(at(i) + 4 * e), f_w[r * n + i]);
          }
#pragma unroll 4
          for (int i = way + kAhead * ways; i < n; i += ways)
            add(*reinterpret_cast<const float4*>(at(i) + 4 * e), f_w[r * n + i]);
        }
        s_sum[threadIdx.x] = sum;
        __syncthreads();
        if (ok && way == 0) {
          for (int w = 1; w < ways; ++w) add(s_sum[w * quads + e], 1.0f);  // in order: the same sum from call to call
          store_out(a, x, head_dim, r, d, sum.x * f_inv[r], sum.y * f_inv[r], f_bad[r]);
          store_out(a, x, head_dim, r, d + 2, sum.z * f_inv[r], sum.w * f_inv[r], f_bad[r]);
        }
        __syncthreads();
      }
    }
    if (adds) add_weights(a, x, cuts[side][1].x, cuts[side][1].y, s_limit, f_m, f_inv);
    __syncthreads();
  }
}

// The probabilities of kDecodeRows to kScoreRows query rows, from the kept scores: a CTA has
// kAddRows cache rows of a kv head.  Bandwidth: 4 bytes per row and cache row, written and
// read (16 x 16 heads, 16 query rows over 8192, attention and weights: 214 us; with the
// scores computed again 528).
constexpr int kAddRows = 1024, kAddThreads = 256;
__global__ void __launch_bounds__(kAddThreads) kv4_add_weights_kernel(const AttnArgs a) {
  __shared__ float s_lse[kScoreRows], s_one[kScoreRows];
  __shared__ int s_limit[kScoreRows];
  grid_dependency_begin();
  const unsigned heads_all = (unsigned)(a.batch * a.kv_heads), chunk = blockIdx.x / heads_all;
  const int bh = (int)(blockIdx.x - chunk * heads_all), b = bh / a.kv_heads, rows = a.group * a.seq;
  const Item x{bh, b, bh - b * a.kv_heads, 0, rows};
  if ((int)threadIdx.x < rows) {
    s_limit[threadIdx.x] = visible_rows(a, b, (int)(threadIdx.x % (unsigned)a.seq));
    s_lse[threadIdx.x] = a.lse[((int64_t)b * a.heads + x.hk * a.group) * a.seq + threadIdx.x];
    s_one[threadIdx.x] = 1.0f;
  }
  __syncthreads();
  add_weights(a, x, (int)chunk * kAddRows, (int)chunk * kAddRows + kAddRows, s_limit, s_lse, s_one);
}

int64_t items_of(const AttnArgs& a) {
  return a.batch * a.kv_heads * (((int64_t)a.group * a.seq + kBlockRows - 1) / kBlockRows);
}
int part_rows(int64_t rows) { return (int)(rows < kBlockRows ? rows : kBlockRows); }
// CTAs of kv4_decode_shares_kernel that the GPU holds at once.
int64_t shares_for(int64_t head_dim) {
  return (int64_t)device_sm_count() * (head_dim <= 128 ? Cta<128, kShareWarps>::kPerSm : Cta<256, kShareWarps>::kPerSm);
}

template <int D, bool ONE>
cudaError_t launch_decode(const AttnArgs& a, int64_t longest, float* parts, cudaStream_t s) {
  {
    // CTAs per item: while each has an SM for itself and its warps a tile each.  Two on
    // an SM pay from some 2000 rows on (128 items of 6 query rows, D = 64, one CTA against
    // two of them each: 600 rows 8.4 against 10.2 us, 1250 10.8 against 11.8, ragged
    // up to 2500 15.1 against 14.2).
    constexpr int kWarps = kClusterWarps;
    using T = Cta<D, kWarps>;
    const int64_t items = items_of(a), slots = (int64_t)device_sm_count() * (longest > 2048 ? T::kPerSm : 1);
    int count = 1;
    while (count < kClusterMax && items * (count + 1) <= slots && (int64_t)kTileRows * kWarps * count < longest) ++count;
    // A cluster saves the joining launch (5 us) but leaves SMs idle, or waits for the longest
    // item: 12 items over 4096 rows 8.6 against 11.7 us, over 12000 13.9 against 16.5; 96 items over
    // 4096 27.8 against 26.1, over 8192 43.9 against 38.5.
    if (longest <= kSplitRows || longest <= kSplitRows * 3 / 8 * count) {
      const cudaError_t e = allow_shared<kv4_decode_kernel<D, ONE>>(T::kSmem);
      if (e != cudaSuccess) return e;
      return launch_cluster(kv4_decode_kernel<D, ONE>, items * count, kWarps * 32, T::kSmem, count, s, a, count);
    }
  }
  using T = Cta<D, kShareWarps>;
  const int rows = part_rows((int64_t)a.group * a.seq);
  const int64_t shares = shares_for(D);
  cudaError_t e = allow_shared<kv4_decode_shares_kernel<D, ONE>>(T::kSmem);
  if (e != cudaSuccess) return e;
  e = launch_kernel(kv4_decode_shares_kernel<D, ONE>, shares, kShareWarps * 32, T::kSmem, s, a, parts, rows);
  if (e != cudaSuccess) return e;
  return launch_kernel(kv4_join_kernel, shares, kJoinThreads, rows * shares * sizeof(float), s, a, parts, rows, D);
}

template <int D>
cudaError_t launch_decode(const AttnArgs& a, int64_t longest, float* parts, cudaStream_t s) {
  return a.group * a.seq == 1 ? launch_decode<D, true>(a, longest, parts, s)
                              : launch_decode<D, false>(a, longest, parts, s);
}

}  // namespace

int64_t kv4_decode_workspace(int64_t rows, int64_t head_dim, int64_t longest) {
  if (longest <= kSplitRows) return 0;
  return 2 * shares_for(head_dim) * part_floats(part_rows(rows), head_dim) * (int64_t)sizeof(float);
}

cudaError_t launch_kv4_add_weights(const AttnArgs& a, int64_t longest, cudaStream_t s) {
  const int64_t grid = a.batch * a.kv_heads * ((longest + kAddRows - 1) / kAddRows);
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_kernel(kv4_add_weights_kernel, grid, kAddThreads, 0, s, a);
}

cudaError_t launch_kv4_decode(const AttnArgs& a, int64_t head_dim, int64_t longest, float* parts, cudaStream_t s) {
  switch (head_dim) {
    case 64: return launch_decode<64>(a, longest, parts, s);
    case 128: return launch_decode<128>(a, longest, parts, s);
    case 192: return launch_decode<192>(a, longest, parts, s);
    default: return launch_decode<256>(a, longest, parts, s);
  }
}

}  // namespace hrm
