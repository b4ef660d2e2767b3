// Eviction from the 4-bit KV cache by accumulated attention weight.
//
// Per (batch, kv head), of n rows the `budget` with the largest key stay: the key
// is the row's weight, or +inf for a row at or past the protected position; a NaN
// weight ranks last; of equal keys the lowest rows stay.  Kept rows below `budget` keep
// their places; the i-th kept row past it moves to the i-th freed place.  So an
// in-place eviction moves the fewest rows -- one per decode step -- and attention
// over the cache, which is indifferent to the order of its rows, reads it as is.
//
// What bounds it: 8 bytes per row read (weight, position) and the rows moved;
// small cases are bound by the latency of the selection.  The selection keeps
// the keys in registers, as integers that order like them, and bisects on the
// key's value with one CTA-wide count per step -- no sort, no atomics, and it
// ends as soon as a threshold leaves exactly `budget` keys.  When a single row
// must go (a decode step) it is a CTA-wide minimum instead.
// The CTAs of a cluster select redundantly (the keys come from L2) and share the
// rows to move; a cluster barrier separates reading the keys from moving rows.
#include <cooperative_groups.h>

#include "kv4.cuh"
#include "launch.h"

namespace hrm {
namespace {

namespace cg = cooperative_groups;

struct EvictArgs {
  Kv4View from, to;  // the same buffers: in place
  int64_t kv_heads;
  int64_t length;
  const int* lengths;  // per sequence, or null
  int64_t protect_from;
  const int* protect_froms;
  int budget;
  int* new_lengths;
  int code_pieces;  // 16-byte pieces of a row's codes, and 32-bit words of its scales: head_dim / 32
  bool in_place;
};

constexpr uint32_t kInfKey = 0xff800000u;

// An integer that orders like the weight; 0 for NaN, kInfKey for +inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 and +0 alike
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum over the CTA, given to every thread; `buf` holds one word per warp.  Two
// alternating buffers make one barrier per call enough.
template <int W>
__device__ __forceinline__ int cta_sum(int x, int* buf) {
  x = __reduce_add_sync(0xffffffffu, x);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = x;
  __syncthreads();
  int s = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) s += buf[w];
  return s;
}

// Words of shared memory: the moving rows in order, then a bit per place that
// keeps its row and, per 32 places, how many are freed before them.
inline int64_t evict_moves(int64_t n, int64_t budget) { return n <= budget ? 0 : (n - budget < budget ? n - budget : budget); }
constexpr size_t kSharedMost = 200 * 1024;
inline size_t evict_shared(int64_t n, int64_t budget) {
  return 4 * (size_t)(evict_moves(n, budget) + 2 * ((budget + 31) / 32));
}

// W warps; K keys per lane held in registers, or K = 0: read again at each use.
// Warp w owns the rows [w * steps * 32, (w + 1) * steps * 32), 32 at a time, so
// that ranks in row order need one CTA-wide step.
template <int W, int K>
__global__ void __launch_bounds__(W * 32) kv4_evict_kernel(const EvictArgs a, const int shares, const int moves_at_most) {
  extern __shared__ int movers[];
  uint32_t* keeps = reinterpret_cast<uint32_t*>(movers + moves_at_most);
  int* freed = reinterpret_cast<int*>(keeps + (a.budget + 31) / 32);
  __shared__ int buf[2][32];
  __shared__ int s_total[3][32];
  __shared__ unsigned long long s_low[32];
  grid_dependency_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int share = blockIdx.x % shares;
  const int64_t bh = blockIdx.x / shares, b = bh / a.kv_heads;
  int64_t len = a.lengths ? a.lengths[b] : a.length;
  len = len < 0 ? 0 : (len > a.from.cache_len ? a.from.cache_len : len);
  const int n = (int)len, budget = a.budget, kept = n < budget ? n : budget;
  const int64_t protect = a.protect_froms ? a.protect_froms[b] : a.protect_from;
  if (share == 0 && bh == b * a.kv_heads && threadIdx.x == 0) a.new_lengths[b] = kept;
  const float* weights = a.from.weights + bh * a.from.cache_len;
  const int* positions = a.from.positions + bh * a.from.cache_len;

  const int steps = K > 0 ? K : (n + W * 32 - 1) / (W * 32);
  const int base = warp * steps * 32 + lane;
  auto read_key = [&](int row) -> uint32_t {
    return row >= n ? 0 : (positions[row] >= protect ? kInfKey : weight_key(weights[row]));
  };
  uint32_t reg[K > 0 ? K : 1];
  if (n > budget) {
#pragma unroll
    for (int i = 0; i < K; ++i) reg[i] = read_key(base + 32 * i);
  }
  auto key = [&](int i) -> uint32_t { return K > 0 ? reg[K > 0 ? i : 0] : read_key(base + 32 * i); };

  const bool single = n - budget == 1;
  int out = -1;  // single: the row that goes
  if (single) {
    // the smallest key, of equal ones the last row
    unsigned long long low = ~0ull;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int row = base + 32 * i;
      const unsigned long long x = (unsigned long long)key(i) << 32 | (uint32_t)(n - 1 - row);
      if (row < n && x < low) low = x;
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
      const unsigned long long x = __shfl_xor_sync(0xffffffffu, low, o);
      low = x < low ? x : low;
    }
    if (lane == 0) s_low[warp] = low;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) low = s_low[w] < low ? s_low[w] : low;
    out = n - 1 - (int)(uint32_t)low;
  } else if (n > budget) {
    // bisect: count(key >= lo) >= budget > count(key >= hi); mid >= 1, so the keys
    // 0 past the last row never count
    uint64_t lo = 0, hi = 1ull << 32;
    int above = 0, at_lo = n, turn = 0;
    while (hi - lo > 1 && at_lo != budget) {
      const uint32_t mid = (uint32_t)((lo + hi) / 2);
      int c = 0;
#pragma unroll
      for (int i = 0; i < steps; ++i) c += key(i) >= mid;
      c = cta_sum<W>(c, buf[turn]);
      turn ^= 1;
      if (c >= budget) {
        lo = mid;
        at_lo = c;
      } else {
        hi = mid;
        above = c;
      }
    }
    // all keys >= lo stay; or those above it and, in row order, as many equal to it as there is room for
    const bool exact = at_lo == budget;
    const uint32_t threshold = (uint32_t)lo;
    const int room = budget - above;
    int eq = 0;  // keys equal to the threshold in earlier rows
    if (!exact) {
      int c = 0;
#pragma unroll
      for (int i = 0; i < steps; ++i)
        c += __popc(__ballot_sync(0xffffffffu, base + 32 * i < n && key(i) == threshold));
      if (lane == 0) s_total[0][warp] = c;
      __syncthreads();
      for (int w = 0; w < warp; ++w) eq += s_total[0][w];
    }
    // Per 32 rows the mask of those that stay.  It goes to shared memory for places;
    // for rows past them the counts give the moving rows' ranks.
    int holes = 0, moves = 0;
    uint32_t mine = 0;  // lane i keeps the mask of step i (K > 0 has at most 32 steps)
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int row = base + 32 * i, first = row - lane;
      const uint32_t k = key(i);
      uint32_t mask;
      if (exact) {
        mask = __ballot_sync(0xffffffffu, row < n && k >= threshold);
      } else {
        const uint32_t same = __ballot_sync(0xffffffffu, row < n && k == threshold);
        const bool stays = row < n && (k > threshold || (k == threshold && eq + __popc(same & ((1u << lane) - 1)) < room));
        eq += __popc(same);
        mask = __ballot_sync(0xffffffffu, stays);
      }
      const int places = budget - first;  // of these 32 rows, the first ones that are places
      const uint32_t low = places >= 32 ? 0xffffffffu : (places <= 0 ? 0u : (1u << places) - 1);
      if (K > 0) mine = lane == i ? mask : mine;
      if (lane == 0 && low != 0) {
        keeps[first / 32] = mask;
        freed[first / 32] = holes;  // within this warp's rows: completed below
      }
      holes += __popc(~mask & low);
      moves += __popc(mask & ~low);
    }
    if (lane == 0) {
      s_total[1][warp] = holes;
      s_total[2][warp] = moves;
    }
    __syncthreads();
    int hole = 0, move = 0;
    for (int w = 0; w < warp; ++w) {
      hole += s_total[1][w];
      move += s_total[2][w];
    }
    if (!exact) {  // the equal keys' ranks again
      eq = 0;
      for (int w = 0; w < warp; ++w) eq += s_total[0][w];
    }
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int row = base + 32 * i, first = row - lane;
      uint32_t mask;
      if (K > 0) {
        mask = __shfl_sync(0xffffffffu, mine, i);
      } else {
        const uint32_t k = key(i);
        const uint32_t same = __ballot_sync(0xffffffffu, row < n && k == threshold);
        mask = __ballot_sync(0xffffffffu, row < n && (k > threshold || (k == threshold &&
                                              (exact || eq + __popc(same & ((1u << lane) - 1)) < room))));
        eq += __popc(same);
      }
      const int places = budget - first;
      const uint32_t low = places >= 32 ? 0xffffffffu : (places <= 0 ? 0u : (1u << places) - 1);
      const uint32_t moving = mask & ~low;
      if (moving >> lane & 1u) movers[move + __popc(moving & ((1u << lane) - 1))] = row;
      move += __popc(moving);
      if (lane == 0 && low != 0) freed[first / 32] += hole;
    }
  }
  __syncthreads();
  // In place, no CTA of this head may move a row while another still reads keys.
  if (shares > 1 && a.in_place) cg::this_cluster().sync();
  if (a.in_place && n <= budget) return;

  // Copies: a lane moves one 16-byte piece of codes (k, then v) and one word of
  // scales of a row; 2 * code_pieces lanes (rounded up to `lanes`) make a row.
  const int p = a.code_pieces, lanes = 2 * p <= 4 ? 4 : (2 * p <= 8 ? 8 : 16);
  const int per_warp = 32 / lanes, sub = lane % lanes;
  const int first = (share * W + warp) * per_warp + lane / lanes;
  auto source = [&](int d) -> int {
    if (n <= budget) return d;
    if (single) return d == out ? n - 1 : d;
    const uint32_t m = keeps[d / 32];
    if (m >> (d & 31) & 1u) return d;
    return movers[freed[d / 32] + __popc(~m & ((1u << (d & 31)) - 1))];
  };
  auto copy = [&](int d, int src) {
    const int64_t x = bh * a.from.cache_len + src, y = bh * a.to.cache_len + d;
    if (sub < 2 * p) {
      const bool v = sub >= p;
      const int c = v ? sub - p : sub;
      const uint4* from = reinterpret_cast<const uint4*>(v ? a.from.v_codes : a.from.k_codes) + x * p + c;
      uint4* to = reinterpret_cast<uint4*>(v ? a.to.v_codes : a.to.k_codes) + y * p + c;
      const uint32_t* sf = (v ? a.from.v_scales : a.from.k_scales) + x * p + c;
      uint32_t* st = (v ? a.to.v_scales : a.to.k_scales) + y * p + c;
      const uint4 code = *from;
      const uint32_t scale = *sf;
      *to = code;
      *st = scale;
    }
    if (sub == 0) a.to.weights[y] = a.from.weights[x];
    if (sub == 1) a.to.positions[y] = a.from.positions[x];
  };
  if (single && a.in_place) {
    if (out < budget && share == 0 && warp == 0 && lane < lanes) copy(out, n - 1);
    return;
  }
#pragma unroll 4
  for (int d = first; d < kept; d += shares * W * per_warp) {
    const int src = source(d);
    if (!a.in_place || src != d) copy(d, src);
  }
}

template <int W, int K>
cudaError_t launch(const EvictArgs& a, int64_t batch, int64_t n, int shares, cudaStream_t s) {
  const size_t smem = evict_shared(n, a.budget);
  // the size varies from call to call: allow the largest that kv4_evict_fits lets through
  const cudaError_t e = smem <= 48 * 1024 ? cudaSuccess : allow_shared<kv4_evict_kernel<W, K>>(kSharedMost);
  if (e != cudaSuccess) return e;
  const int64_t grid = batch * a.kv_heads * shares;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_cluster(kv4_evict_kernel<W, K>, grid, W * 32, smem, shares, s, a, shares, (int)evict_moves(n, a.budget));
}

}  // namespace

bool kv4_evict_fits(int64_t n, int64_t budget) { return evict_shared(n, budget) <= kSharedMost; }

cudaError_t launch_kv4_evict(const Kv4View& from, const Kv4View& to, bool in_place, int64_t batch, int64_t kv_heads,
                             int64_t head_dim, int64_t length, const int* lengths, int64_t budget,
                             int64_t protect_from, const int* protect_froms, int* new_lengths, cudaStream_t s) {
  EvictArgs a{};
  a.from = from;
  a.to = to;
  a.kv_heads = kv_heads;
  a.length = length;
  a.lengths = lengths;
  a.protect_from = protect_from;
  a.protect_froms = protect_froms;
  a.budget = (int)budget;
  a.new_lengths = new_lengths;
  a.code_pieces = (int)(head_dim / 32);
  a.in_place = in_place;
  const int64_t n = lengths ? from.cache_len : (length < from.cache_len ? length : from.cache_len);
  // CTAs per head that share the moves: at least 256 places each, while the heads leave SMs idle
  int shares = 1;
  while (shares < 8 && batch * kv_heads * shares * 2 <= 2 * device_sm_count() && budget >= 256 * shares * 2) shares *= 2;
  if (n <= 8 * 256) return launch<8, 8>(a, batch, n, shares, s);
  if (n <= 8 * 1024) return launch<32, 8>(a, batch, n, shares, s);
  if (n <= 32 * 1024) return launch<32, 32>(a, batch, n, shares, s);
  return launch<32, 0>(a, batch, n, shares, s);
}

}  // namespace hrm
