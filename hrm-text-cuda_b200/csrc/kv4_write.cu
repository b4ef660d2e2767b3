// Writes into the 4-bit KV cache (format: kv4.cuh): the attention prologue
// (split + RoPE + cache write in one read of the projection's output) and the
// plain append of keys and values.
//
// Both are HBM streams.  A thread owns 8 consecutive pairs of a head -- the
// 16-byte chunk j of the low half and the matching chunk of the high half, as
// in the bf16 prologue (rope.cu) -- so the 4 lanes of an aligned quad hold one
// whole quantisation group of each half, and two shuffles give its range.
// Per head a thread has 8 x 16 B of loads in flight before any use, and its
// cos/sin (loaded once) serve every head that it visits.  The gate, q and the
// rotated k (before quantisation) have the bits of the bf16 prologue.
//
// Measured (D = 128, k and v kept): 8 x 4096 tokens of 16 heads 187 us, 0.95 of the
// copy bandwidth; 1001 tokens of 12 heads 8.1 us (4.2 at that bandwidth: one wave of
// threads that load, shuffle and store once); 64 x 1 tokens 3.4 us, of which an empty
// launch is 2.
#include "kv4.cuh"
#include "launch.h"
#include "rope_math.cuh"

namespace hrm {
namespace {

struct WriteArgs {
  const uint4* gqkv;
  uint4* gate;
  uint4* q;
  uint4* k;  // may be null, with v
  uint4* v;
  Kv4View c;
  int64_t seq;
  int64_t tiles_per_batch;
  int heads;
  int ht;  // head slices per tile, a power of two; the other slots are positions
  int64_t position_offset, cache_offset;
  const int* position_offsets;  // per sequence, or null
  const int* cache_offsets;
  const float4* table;
  int64_t table_positions;
  float theta;
};

// Threads of a write tile: head_dim / 16 per head, times a power of two of
// slots (head, position) that makes whole warps.
template <int D>
struct Tile {
  static constexpr int G = D / 16;
  static constexpr int kSlots = G == 12 ? 8 : 128 / G;
  static constexpr int kThreads = G * kSlots;
};

// Stores a lane's 8 codes of one half (chunk `c` of the row) and the group's word.
__device__ __forceinline__ void store_chunk(uint8_t* codes, uint32_t* scales, int c, uint32_t code, uint32_t sz) {
  reinterpret_cast<uint32_t*>(codes)[c] = code;
  if ((c & 3) == 0) scales[c >> 2] = sz;
}

template <int D>
__global__ void __launch_bounds__(Tile<D>::kThreads) split_rope_kv4_kernel(const WriteArgs a) {
  constexpr int G = Tile<D>::G, C = D / 8;
  grid_dependency_begin();
  const int j = threadIdx.x % G, slot = threadIdx.x / G;
  const int64_t b = blockIdx.x / a.tiles_per_batch;
  const int64_t s = (blockIdx.x - b * a.tiles_per_batch) * (Tile<D>::kSlots / a.ht) + slot / a.ht;
  if (s >= a.seq) return;  // whole quads: a slot is G threads
  const uint32_t quad = 0xfu << (threadIdx.x & 28);
  const int64_t pos = (a.position_offsets ? a.position_offsets[b] : a.position_offset) + s;
  const int64_t row = (a.cache_offsets ? a.cache_offsets[b] : a.cache_offset) + s;
  const bool stored = row >= 0 && row < a.c.cache_len;

  float cs[8], sn[8];
  if (a.table != nullptr && pos >= 0 && pos < a.table_positions) {
    table_cos_sin(a.table, (int)pos, j, D, cs, sn);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) sincosf(rope_angle((int)pos, 8 * j + i, D, a.theta), &sn[i], &cs[i]);
  }

  const int64_t token = b * a.seq + s, seg = (int64_t)a.heads * C;
  for (int h = slot % a.ht; h < a.heads; h += a.ht) {
    const uint4* in = a.gqkv + token * 4 * seg + (int64_t)h * C + j;
    const uint4 g0 = ld_l2(in), g1 = ld_l2(in + G);
    uint4 q0 = ld_l2(in + seg), q1 = ld_l2(in + seg + G);
    uint4 k0 = ld_l2(in + 2 * seg), k1 = ld_l2(in + 2 * seg + G);
    const uint4 v0 = ld_l2(in + 3 * seg), v1 = ld_l2(in + 3 * seg + G);

    uint4* gate = a.gate + token * seg + (int64_t)h * C + j;
    st_l2(gate, g0);
    st_l2(gate + G, g1);
    const int64_t out = ((b * a.heads + h) * a.seq + s) * C + j;
    rotate8<false>(q0, q1, cs, sn);
    st_l2(a.q + out, q0);
    st_l2(a.q + out + G, q1);
    rotate8<true>(k0, k1, cs, sn);

    uint32_t zk0, zk1, zv0, zv1;
    const uint32_t ck0 = kv4_quantise(k0, quad, zk0), ck1 = kv4_quantise(k1, quad, zk1);
    const uint32_t cv0 = kv4_quantise(v0, quad, zv0), cv1 = kv4_quantise(v1, quad, zv1);
    if (stored) {
      const int64_t at = (b * a.heads + h) * a.c.cache_len + row;
      uint8_t* kc = a.c.k_codes + at * (D / 2);
      uint8_t* vc = a.c.v_codes + at * (D / 2);
      uint32_t* ks = a.c.k_scales + at * (D / kKv4Group);
      uint32_t* vs = a.c.v_scales + at * (D / kKv4Group);
      store_chunk(kc, ks, j, ck0, zk0);
      store_chunk(kc, ks, j + G, ck1, zk1);
      store_chunk(vc, vs, j, cv0, zv0);
      store_chunk(vc, vs, j + G, cv1, zv1);
      if (j == 0) {
        if (a.c.weights) a.c.weights[at] = 0.0f;
        if (a.c.positions) a.c.positions[at] = (int)pos;
      }
    }
    if (a.k != nullptr) {
      st_l2(a.k + out, kv4_values(ck0, zk0));
      st_l2(a.k + out + G, kv4_values(ck1, zk1));
      st_l2(a.v + out, kv4_values(cv0, zv0));
      st_l2(a.v + out + G, kv4_values(cv1, zv1));
    }
  }
}

struct UpdateArgs {
  const uint4* k;
  const uint4* v;
  Kv4View c;
  int64_t rows;  // batch * heads * seq
  int64_t heads, seq;
  int64_t position_offset, cache_offset;
  const int* position_offsets;
  const int* cache_offsets;
};

// One thread per 16-byte chunk of a row of k and of v.
template <int D>
__global__ void __launch_bounds__(128) kv4_update_kernel(const UpdateArgs a) {
  constexpr int C = D / 8;
  grid_dependency_begin();
  const int64_t t = (int64_t)blockIdx.x * 128 + threadIdx.x;
  const int64_t r = t / C;
  const int j = (int)(t - r * C);
  if (r >= a.rows) return;  // whole quads: a row is C = 4 * k threads
  const uint32_t quad = 0xfu << (threadIdx.x & 28);
  const uint4 k = ld_l2(a.k + t), v = ld_l2(a.v + t);
  const int64_t bh = r / a.seq, s = r - bh * a.seq, b = bh / a.heads;
  const int64_t pos = (a.position_offsets ? a.position_offsets[b] : a.position_offset) + s;
  const int64_t row = (a.cache_offsets ? a.cache_offsets[b] : a.cache_offset) + s;
  if (row < 0 || row >= a.c.cache_len) return;
  uint32_t zk, zv;
  const uint32_t ck = kv4_quantise(k, quad, zk), cv = kv4_quantise(v, quad, zv);
  const int64_t at = bh * a.c.cache_len + row;
  store_chunk(a.c.k_codes + at * (D / 2), a.c.k_scales + at * (D / kKv4Group), j, ck, zk);
  store_chunk(a.c.v_codes + at * (D / 2), a.c.v_scales + at * (D / kKv4Group), j, cv, zv);
  if (j == 0) {
    if (a.c.weights) a.c.weights[at] = 0.0f;
    if (a.c.positions) a.c.positions[at] = (int)pos;
  }
}

template <int D>
cudaError_t launch_split(WriteArgs a, int64_t batch, cudaStream_t s) {
  constexpr int kSlots = Tile<D>::kSlots;
  // Head slices per tile: all slots for one position, as far as there are heads; where the
  // tiles are many, a quarter of them, so that a thread's cos/sin serve several heads
  // (16 heads, D = 128, whole against quarter: 64 x 1 tokens 3.4 and 7.6 us, 4 x 512 15.6 and 18.3,
  // 8 x 4096 with inputs that change from call to call 202 and 190).
  int ht = 1;
  while (ht < kSlots && ht < a.heads) ht *= 2;
  if (batch * a.seq > 64 * device_sm_count()) ht = ht < 4 ? 1 : ht / 4;
  a.ht = ht;
  const int64_t pt = kSlots / ht;
  a.tiles_per_batch = (a.seq + pt - 1) / pt;
  const int64_t grid = batch * a.tiles_per_batch;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_kernel(split_rope_kv4_kernel<D>, grid, Tile<D>::kThreads, 0, s, a);
}

template <int D>
cudaError_t launch_update(const UpdateArgs& a, cudaStream_t s) {
  const int64_t grid = (a.rows * (D / 8) + 127) / 128;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_kernel(kv4_update_kernel<D>, grid, 128, 0, s, a);
}

}  // namespace

cudaError_t launch_split_rope_kv4(const void* gqkv, void* gate, void* q, void* k, void* v, const Kv4View& c,
                                  int64_t batch, int64_t heads, int64_t seq, int64_t head_dim,
                                  int64_t position_offset, const int* position_offsets, float theta,
                                  const float* table, int64_t table_positions, int64_t cache_offset,
                                  const int* cache_offsets, cudaStream_t s) {
  WriteArgs a{};
  a.gqkv = static_cast<const uint4*>(gqkv);
  a.gate = static_cast<uint4*>(gate);
  a.q = static_cast<uint4*>(q);
  a.k = static_cast<uint4*>(k);
  a.v = static_cast<uint4*>(v);
  a.c = c;
  a.seq = seq;
  a.heads = (int)heads;
  a.position_offset = position_offset;
  a.cache_offset = cache_offset;
  a.position_offsets = position_offsets;
  a.cache_offsets = cache_offsets;
  a.table = reinterpret_cast<const float4*>(table);
  a.table_positions = table_positions;
  a.theta = theta;
  switch (head_dim) {
    case 64: return launch_split<64>(a, batch, s);
    case 128: return launch_split<128>(a, batch, s);
    case 192: return launch_split<192>(a, batch, s);
    default: return launch_split<256>(a, batch, s);
  }
}

cudaError_t launch_kv4_update(const void* k, const void* v, const Kv4View& c, int64_t batch, int64_t heads,
                              int64_t seq, int64_t head_dim, int64_t position_offset, const int* position_offsets,
                              int64_t cache_offset, const int* cache_offsets, cudaStream_t s) {
  UpdateArgs a{static_cast<const uint4*>(k), static_cast<const uint4*>(v), c, batch * heads * seq, heads, seq,
               position_offset, cache_offset, position_offsets, cache_offsets};
  switch (head_dim) {
    case 64: return launch_update<64>(a, s);
    case 128: return launch_update<128>(a, s);
    case 192: return launch_update<192>(a, s);
    default: return launch_update<256>(a, s);
  }
}

}  // namespace hrm
