// Eviction from the 4-bit KV cache by accumulated attention weight.
//
// Per (batch, kv head), of n rows the `budget` with the largest key stay: the key
// is the row's weight, or +inf for a row at or past the protected position; a NaN
// weight ranks last; of equal keys the lowest rows stay.  Kept rows below `budget` keep
// their places; the i-th kept row past it moves to the i-th freed place.  So an
// in-place eviction moves the fewest rows -- one per decode step -- and attention
// over the cache, which is indifferent to the order of its rows, reads it as is.
//
// What bounds it: 8 bytes per row read (weight, position) and the rows moved, by
// bandwidth only in large batches; else by the latency of the selection's steps.
// The CTAs of a cluster share a head's rows.  Keys stay in registers, as integers
// that order like the weights; the budget-th largest is found digit by digit (11, 11
// and 10 bits), each by counting in shared memory and adding up the cluster's counts
// over distributed shared memory -- counts only, so their order changes nothing --
// and ends early when a digit's border leaves exactly `budget` rows.  Rows whose key
// is the threshold are then taken in row order.  When a single row must go (a
// decode step) it is one CTA-wide minimum instead.
//
// Measured: 64 x 16 heads, one of 1025 rows each, 10 us with the write of the new row;
// 12 heads, 32768 rows to 4096 of D = 128, 25 us (a third of it the three digits, a third the
// copies); 16 x 16 heads, up to 5000 rows to 1111 of D = 64, 28 us.
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
constexpr uint32_t kAll = 0xffffffffu;
constexpr int kBins = 2048;
constexpr int kListed = 128;  // rows that a warp lists before it copies them

// An integer that orders like the weight; 0 for NaN, kInfKey for +inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 and +0 alike
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum of x over the CTA's threads in order, and the total.  Two alternating
// buffers of a word per warp make one barrier per call enough.
template <int W>
__device__ __forceinline__ int cta_scan(int x, int* buf, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = x;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int y = __shfl_up_sync(kAll, sum, o);
    if (lane >= o) sum += y;
  }
  if (lane == 31) buf[warp] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int y = buf[w];
    all += y;
    if (w < warp) before += y;
  }
  *total = all;
  return before + sum - x;
}

// Rows that can move at most, and the dynamic shared memory: counts of the three
// digits, the cluster's sums of one, per 32 rows of the CTA a mask and two ranks,
// and the freed places in order (in the cluster's first CTA).
inline int64_t evict_moves(int64_t n, int64_t budget) {
  return n <= budget ? 0 : (n - budget < budget ? n - budget : budget);
}
constexpr size_t kSharedMost = 200 * 1024;
inline size_t evict_shared(int64_t groups, int64_t moves) { return 4 * (size_t)(4 * kBins + 3 * groups + moves); }

// W warps per CTA; K steps of 32 rows per warp, their keys in registers (K = 0: any
// number, the keys read again at each use).  CTA c of the cluster's `count` has the
// rows [c, c + 1) * W * steps * 32; groups of 32 rows go to the warps in turn, so that the
// copies are even over the warps wherever the rows that stay lie.
template <int W, int K>
__global__ void __launch_bounds__(W * 32, W == 8 ? 4 : 2)
    kv4_evict_kernel(const EvictArgs a, const int count, const int steps_at_most) {
  extern __shared__ __align__(16) int shared[];
  int* hist = shared;                                                 // [3][kBins]
  int* sums = shared + 3 * kBins;                                     // [kBins]: the cluster's
  uint32_t* masks = reinterpret_cast<uint32_t*>(shared + 4 * kBins);  // per group: rows that stay
  int* hole_at = shared + 4 * kBins + W * steps_at_most;              // freed places in the groups before
  int* move_at = hole_at + W * steps_at_most;                         // moving rows in the groups before
  int* freed = move_at + W * steps_at_most;                           // in the cluster's first CTA
  __shared__ int buf[2][32];
  __shared__ int s_totals[2];  // this CTA's sums of the counts being ranked
  __shared__ int s_bin, s_above, s_in;
  __shared__ unsigned long long s_low[32];
  __shared__ int2 s_copy[W][kListed];  // (source row, place)
  grid_dependency_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned head = count == 1 ? blockIdx.x : blockIdx.x / (unsigned)count;
  const int rank = (int)(blockIdx.x - head * count);
  const int64_t bh = head, b = bh / a.kv_heads;
  int64_t len = a.lengths ? a.lengths[b] : a.length;
  len = len < 0 ? 0 : (len > a.from.cache_len ? a.from.cache_len : len);
  const int n = (int)len, budget = a.budget, kept = n < budget ? n : budget;
  const int64_t protect = a.protect_froms ? a.protect_froms[b] : a.protect_from;
  if (rank == 0 && bh == b * a.kv_heads && threadIdx.x == 0) a.new_lengths[b] = kept;
  const float* weights = a.from.weights + bh * a.from.cache_len;
  const int* positions = a.from.positions + bh * a.from.cache_len;
  cg::cluster_group cluster = cg::this_cluster();
  auto join = [&]() {  // a barrier over the CTAs that share the head
    if (count > 1)
      cluster.sync();
    else
      __syncthreads();
  };

  const int steps = K > 0 ? K : (n + count * W * 32 - 1) / (count * W * 32);
  const int cta_row = rank * W * steps * 32;           // the CTA's first row
  auto row_of = [&](int i) -> int { return cta_row + (i * W + warp) * 32 + lane; };
  auto make_key = [&](int row, int position, float weight) -> uint32_t {
    return row >= n ? 0 : (position >= protect ? kInfKey : weight_key(weight));
  };
  auto read_key = [&](int row) -> uint32_t {
    const int at = row < n ? row : 0;
    return make_key(row, positions[at], weights[at]);
  };
  uint32_t reg[K > 0 ? K : 1];
  if (n > budget) {
    int position[K > 0 ? K : 1];
    float weight[K > 0 ? K : 1];
#pragma unroll
    for (int i = 0; i < K; ++i) {  // all reads in flight at once
      const int at = row_of(i) < n ? row_of(i) : 0;
      position[i] = positions[at];
      weight[i] = weights[at];
    }
#pragma unroll
    for (int i = 0; i < K; ++i) reg[i] = make_key(row_of(i), position[i], weight[i]);
  }
  auto key = [&](int i) -> uint32_t { return K > 0 ? reg[K > 0 ? i : 0] : read_key(row_of(i)); };

  // A lane copies one 16-byte piece of codes (k, then v) and one word of scales of a
  // row; `lanes` lanes (2 * code_pieces of them at work) make a row.
  const int p = a.code_pieces, lanes = 2 * p <= 4 ? 4 : (2 * p <= 8 ? 8 : 16), sub = lane % lanes;
  const bool works = sub < 2 * p, is_v = sub >= p;
  const int64_t from0 = bh * a.from.cache_len, to0 = bh * a.to.cache_len;
  const int piece = is_v ? sub - p : sub;
  const uint4* code_from = reinterpret_cast<const uint4*>(is_v ? a.from.v_codes : a.from.k_codes) + from0 * p + piece;
  const uint32_t* scale_from = (is_v ? a.from.v_scales : a.from.k_scales) + from0 * p + piece;
  uint4* code_to = reinterpret_cast<uint4*>(is_v ? a.to.v_codes : a.to.k_codes) + to0 * p + piece;
  uint32_t* scale_to = (is_v ? a.to.v_scales : a.to.k_scales) + to0 * p + piece;

  if (n <= budget && a.in_place) return;  // the whole cluster
  if (count == 1 && a.in_place && n - budget == 1) {
    // One row goes: the smallest key, of equal ones the last row; the last row takes its place.
    unsigned long long low = ~0ull;
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const int row = row_of(i);
      const unsigned long long x = (unsigned long long)key(i) << 32 | (uint32_t)(n - 1 - row);
      if (row < n && x < low) low = x;
    }
#pragma unroll
    for (int o = 16; o > 0; o /= 2) {
      const unsigned long long x = __shfl_xor_sync(kAll, low, o);
      low = x < low ? x : low;
    }
    if (lane == 0) s_low[warp] = low;
    __syncthreads();
    if (warp > 0) return;
#pragma unroll
    for (int w = 0; w < W; ++w) low = s_low[w] < low ? s_low[w] : low;
    const int out = n - 1 - (int)(uint32_t)low;
    if (out < budget) {
      if (lane < lanes && works) {
        code_to[(int64_t)out * p] = code_from[(int64_t)(n - 1) * p];
        scale_to[(int64_t)out * p] = scale_from[(int64_t)(n - 1) * p];
      }
      if (lane == 0) {
        a.to.weights[to0 + out] = weights[n - 1];
        a.to.positions[to0 + out] = positions[n - 1];
      }
    }
    return;
  }

  uint32_t threshold = 0;
  bool exact = true;  // all keys >= threshold stay (n <= budget: all rows)
  int room = 0;       // else: keys above it, and as many equal ones, in row order
  if (n > budget) {
    for (int i = threadIdx.x; i < 3 * kBins; i += W * 32) hist[i] = 0;
    __syncthreads();
    room = budget;
    uint32_t prefix = 0, known = 0;  // the threshold's digits so far
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      const int shift = d == 0 ? 21 : (d == 1 ? 10 : 0), bins = d == 2 ? 1024 : kBins;
      int* h = hist + d * kBins;
#pragma unroll
      for (int i = 0; i < steps; ++i) {
        const uint32_t k = key(i);
        if (row_of(i) < n && (k & known) == prefix) atomicAdd(&h[k >> shift & (bins - 1)], 1);
      }
      join();
      // The cluster's sums: each CTA adds up its slice of the bins and gives it to the
      // others (all CTAs adding up all bins moved four times as much).
      const int* total = h;
      if (count > 1) {
        const int slice = bins / count;
        for (int x = threadIdx.x; x < slice; x += W * 32) {
          const int bin = rank * slice + x;
          int y = 0;
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (c < count) y += *cluster.map_shared_rank(&h[bin], c);
#pragma unroll
          for (int c = 0; c < 8; ++c)
            if (c < count) *cluster.map_shared_rank(&sums[bin], c) = y;
        }
        join();
        total = sums;
      }
      // each thread: its consecutive bins, highest first
      constexpr int kMost = kBins / (W * 32);
      const int each = d == 2 ? kMost / 2 : kMost;
      const int* own = total + bins - ((int)threadIdx.x + 1) * each;  // the lowest of them
      int mine[kMost], sum = 0;
#pragma unroll
      for (int x = 0; x < kMost; ++x) {
        mine[x] = x < each ? own[x] : 0;
        sum += mine[x];
      }
      int all, above = cta_scan<W>(sum, buf[d & 1], &all);
      if (above < room && above + sum >= room) {  // one thread
#pragma unroll
        for (int x = kMost - 1; x >= 0; --x) {
          if (x < each && above < room && above + mine[x] >= room) {
            s_bin = bins - ((int)threadIdx.x + 1) * each + x;
            s_above = above;
            s_in = mine[x];
            above = room;  // found
          } else {
            above += mine[x];
          }
        }
      }
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      known |= (uint32_t)(bins - 1) << shift;
      room -= s_above;
      exact = s_in == room;
      if (exact) break;  // the same in every CTA
      join();            // s_bin, its neighbours and the sums are read
    }
    threshold = prefix;
  }

  // Ranks in row order: per group a count, then its sum over the groups before, over
  // the CTA (each thread has some consecutive groups) and the cluster's CTAs before.
  // N kinds of counts at once: their barriers are shared.
  const int groups = W * steps, per_thread = (groups + W * 32 - 1) / (W * 32);
  auto ranks = [&](auto const& at, auto count_of) {
    constexpr int N = sizeof(at) / sizeof(at[0]);
    const int g0 = threadIdx.x * per_thread;
    int before[N];
#pragma unroll
    for (int x = 0; x < N; ++x) {
      int mine = 0, all;
      for (int g = g0; g < g0 + per_thread && g < groups; ++g) mine += count_of(g, x);
      before[x] = cta_scan<W>(mine, buf[x], &all);
      if (threadIdx.x == 0) s_totals[x] = all;
    }
    join();
#pragma unroll
    for (int x = 0; x < N; ++x) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < rank) before[x] += *cluster.map_shared_rank(&s_totals[x], c);
      for (int g = g0; g < g0 + per_thread && g < groups; ++g) {
        const int n_g = count_of(g, x);  // (the counts may lie where the ranks go)
        at[x][g] = before[x];
        before[x] += n_g;
      }
    }
  };
  if (!exact) {  // all digits known: keys equal to the threshold, in row order
#pragma unroll
    for (int i = 0; i < steps; ++i) {
      const uint32_t same = __ballot_sync(kAll, row_of(i) < n && key(i) == threshold);
      if (lane == 0) hole_at[i * W + warp] = __popc(same);
    }
    __syncthreads();
    int* const at[1] = {hole_at};
    ranks(at, [&](int g, int) { return hole_at[g]; });
    join();  // the totals are read
  }

  // the bits of group g that are places
  auto places = [&](int g) -> uint32_t {
    const int x = kept - (cta_row + 32 * g);
    return x >= 32 ? kAll : (x <= 0 ? 0u : (1u << x) - 1);
  };
  // per 32 rows the mask of those that stay
#pragma unroll
  for (int i = 0; i < steps; ++i) {
    const int row = row_of(i);
    const uint32_t k = n > budget ? key(i) : 0;
    uint32_t mask;
    if (exact) {
      mask = __ballot_sync(kAll, row < n && k >= threshold);
    } else {
      const uint32_t same = __ballot_sync(kAll, row < n && k == threshold);
      const int before = hole_at[i * W + warp] + __popc(same & ((1u << lane) - 1));
      mask = __ballot_sync(kAll, row < n && (k > threshold || (k == threshold && before < room)));
    }
    if (lane == 0) masks[i * W + warp] = mask;
  }
  __syncthreads();
  if (n > budget) {
    int* const at[2] = {hole_at, move_at};
    ranks(at, [&](int g, int x) { return __popc(x == 0 ? ~masks[g] & places(g) : masks[g] & ~places(g)); });
    __syncthreads();
    int* list = count == 1 ? freed : cluster.map_shared_rank(freed, 0);
    for (int g = warp; g < groups && places(g) != 0; g += W) {
      const uint32_t out = ~masks[g] & places(g);
      if (out >> lane & 1u) list[hole_at[g] + __popc(out & ((1u << lane) - 1))] = cta_row + 32 * g + lane;
    }
    // The list is complete; and, in place, every CTA has read its keys.
    join();
  }

  // Copies: each warp its rows that stay (in place: that move).  They are listed until
  // the list could overflow, so that many rows' reads are in flight at once.
  const int per_pass = 32 / lanes, part = lane / lanes;
  // Weight and position go with the row's codes, by its first two lanes, in clusters of CTAs of
  // 2048 to 4096 rows, else before them, a lane per row (12 heads to a quarter, with
  // against before: CTAs of 2100 rows, 2, 4 and 8 of them, 20.3 against 20.5 us, 22.4 and 22.7,
  // 25.6 and 28.2; of 3000 21.5 and 21.7, 23.0 and 24.0, 27.0 and 30.9; of 4000, 2 of
  // them, 22.2 and 23.0; 32768 rows on 8 to an eighth 24.2 and 26.8.  Smaller CTAs: 8192
  // on 4 18.4 and 17.7; 16 x 16 heads of 5000 on one CTA, whose keys leave no
  // registers for it, 29.9 and 28.0).
  const bool with_codes = W == 16 && K == 8 && count > 1;
  const uint32_t* word_from = reinterpret_cast<const uint32_t*>(sub == 0 ? (const void*)weights : positions);
  uint32_t* word_to = reinterpret_cast<uint32_t*>(sub == 0 ? (void*)(a.to.weights + to0) : a.to.positions + to0);
  constexpr int kAhead = 4;
  int listed = 0;
  for (int i = 0; i < steps; ++i) {
    const int g = i * W + warp, first = cta_row + 32 * g;
    const uint32_t low = places(g), mask = masks[g], moving = mask & ~low, todo = a.in_place ? moving : mask;
    if (todo >> lane & 1u) {
      const int at = move_at[g] + __popc(moving & ((1u << lane) - 1));
      const int to = low >> lane & 1u
                         ? first + lane
                         : (count == 1 ? freed[at] : *cluster.map_shared_rank(freed + at, 0));
      s_copy[warp][listed + __popc(todo & ((1u << lane) - 1))] = make_int2(first + lane, to);
    }
    listed += __popc(todo);
    if (listed <= kListed - 32 && i + 1 < steps) continue;
    __syncwarp();
    for (int r = lane; !with_codes && r < listed; r += 32) {
      const int2 c = s_copy[warp][r];
      const float w = weights[c.x];
      const int at = positions[c.x];
      a.to.weights[to0 + c.y] = w;
      a.to.positions[to0 + c.y] = at;
    }
    for (int r0 = part; r0 < listed; r0 += kAhead * per_pass) {
      uint4 code[kAhead];
      uint32_t scale[kAhead], word[kAhead];
      int to[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int r = r0 + x * per_pass;
        const int2 c = s_copy[warp][r < listed ? r : 0];
        to[x] = r < listed && works ? c.y : -1;
        if (works) {  // past the last row: the first once more
          code[x] = code_from[(int64_t)c.x * p];
          scale[x] = scale_from[(int64_t)c.x * p];
          if (with_codes && sub < 2) word[x] = word_from[c.x];
        }
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x)
        if (to[x] >= 0) {
          code_to[(int64_t)to[x] * p] = code[x];
          scale_to[(int64_t)to[x] * p] = scale[x];
          if (with_codes && sub < 2) word_to[to[x]] = word[x];
        }
    }
    __syncwarp();
    listed = 0;
  }
  if (count > 1) cluster.sync();  // the list is read: its CTA may leave
}

template <int W, int K>
cudaError_t launch(const EvictArgs& a, int64_t batch, int64_t n, int count, cudaStream_t s) {
  const int64_t steps = K > 0 ? K : (n + (int64_t)count * W * 32 - 1) / ((int64_t)count * W * 32);
  const size_t smem = evict_shared(W * steps, evict_moves(n, a.budget));
  // the size varies from call to call: allow the largest that kv4_evict_fits lets through
  const cudaError_t e = allow_shared<kv4_evict_kernel<W, K>>(kSharedMost);
  if (e != cudaSuccess) return e;
  const int64_t grid = batch * a.kv_heads * count;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_cluster(kv4_evict_kernel<W, K>, grid, W * 32, smem, count, s, a, count, (int)steps);
}

}  // namespace

bool kv4_evict_fits(int64_t n, int64_t budget) {
  return evict_shared(n / 32 + 1024, evict_moves(n, budget)) <= kSharedMost;  // groups: of one CTA at most
}

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
  // CTAs per head: while they leave room on the GPU (2 of 512 threads per SM) and have 2048 rows
  // each (12 heads: 2048 rows on one CTA 11.4 us, on two 15.8; 4096 17.3 and 18.0; 8192 25.6
  // and, on four, 18.0; 32768 198 and, on eight, 27.7); also without that room, where a
  // CTA's keys would not fit its registers (256 heads of 12000 rows, D = 64: on one 166 us,
  // on two 128; 128 of 20000: on two 137, on four 126).
  constexpr int64_t kKeys = 16 * 512;  // keys that a CTA holds at most
  int count = 1;
  while (count < 8 && n >= 2048 * count * 2 &&
         (batch * kv_heads * count * 2 <= 2 * device_sm_count() || n > kKeys * count))
    count *= 2;
  const int64_t mine = (n + count - 1) / count;
  if (mine <= 8 * 256) return launch<8, 8>(a, batch, n, count, s);
  if (mine <= 8 * 512) return launch<16, 8>(a, batch, n, count, s);
  if (mine <= kKeys) return launch<16, 16>(a, batch, n, count, s);
  return launch<16, 0>(a, batch, n, count, s);
}

}  // namespace hrm
