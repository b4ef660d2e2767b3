// Attention of many query rows over the 4-bit cache (prompts, further turns of
// a chat), and the pass that adds the probabilities of many rows to the cache
// rows' weights.
//
// A CTA owns 64 query rows of one kv head (16 per warp) and walks the cache in
// tiles of 64 rows.  Each tile is dequantised once into shared memory as bf16 (1.5
// instructions per element, shared by the 64 query rows) and multiplied with
// mma.sync; the softmax runs online on the accumulators, which have the layout
// of the next product's operand.  Within each 8 elements the tile keeps
// kv4_pair's order (0, 4, 1, 5, 2, 6, 3, 7): the queries are stored the same way,
// and the output is put back in order when it is written.
#include "kv4_mma.cuh"
#include "launch.h"

namespace hrm {
namespace {

constexpr int kM = 64;  // query rows per CTA
constexpr int kN = 64;  // cache rows per tile
constexpr int kThreads = 128;

template <int D>
struct Chunk {
  static constexpr int kStride = D + 8;  // elements per shared row: 16 bytes of padding spread the banks
  static constexpr int kGroups = D / kKv4Group;
  static constexpr int kQ = 0, kK = kM * kStride * 2, kV = kK + kN * kStride * 2;
  static constexpr int kSmem = kV + kN * kStride * 2;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// Dequantises kN rows from `first` (zeros from `limit` on) into dst.  With
// `flags`, groups that are not finite are stored as zeros and marked there, per
// row; returns whether this thread met one.
template <int D>
__device__ __forceinline__ bool fill_tile(uint8_t* dst, const uint8_t* codes, const uint32_t* scales, int first,
                                          int limit, uint32_t* flags) {
  using T = Chunk<D>;
  constexpr int kPieces = D / 32;  // 16-byte pieces of codes per row: one group each
  bool met = false;
#pragma unroll
  for (int i = 0; i < kN * kPieces / kThreads; ++i) {
    const int idx = i * kThreads + threadIdx.x, r = idx / kPieces, p = idx % kPieces;
    uint4 c = make_uint4(0, 0, 0, 0);
    uint32_t sz = 0;
    if (first + r < limit) {
      c = ld_keep(reinterpret_cast<const uint4*>(codes + (int64_t)(first + r) * (D / 2)) + p);
      sz = __ldg(scales + (int64_t)(first + r) * T::kGroups + p);
    }
    if (flags != nullptr && kv4_not_finite(sz)) {
      atomicOr(&flags[r], 1u << p);
      sz = 0;
      met = true;
    }
    const uint32_t s2 = kv4_scale2(sz), z2 = kv4_base2(sz);
    uint4* row = reinterpret_cast<uint4*>(dst + r * T::kStride * 2) + p * 4;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t x = vget(c, w);
      row[w] = make_uint4(fma_bf16x2(kv4_pair<0>(x), s2, z2), fma_bf16x2(kv4_pair<1>(x), s2, z2),
                          fma_bf16x2(kv4_pair<2>(x), s2, z2), fma_bf16x2(kv4_pair<3>(x), s2, z2));
    }
  }
  return met;
}

// The block's kM query rows into shared memory, elements in kv4_pair's order; zeros past the last row.
template <int D>
__device__ __forceinline__ void fill_queries(uint8_t* dst, const AttnArgs& a, int64_t b, int64_t hk, int64_t row0,
                                             int64_t rows) {
  for (int idx = threadIdx.x; idx < kM * (D / 8); idx += kThreads) {
    const int r = idx / (D / 8), p = idx % (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row0 + r < rows) {
      const int64_t x = row0 + r;
      v = ld_keep(a.q + ((b * a.heads + hk * a.group + x / a.seq) * a.seq + x % a.seq) * (D / 8) + p);
    }
    reinterpret_cast<uint4*>(dst + r * Chunk<D>::kStride * 2)[p] =
        make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                   __byte_perm(v.y, v.w, 0x7632));
  }
}

// acc = the warp's 16 query rows x the tile's kN cache rows.
template <int D>
__device__ __forceinline__ void tile_scores(float (&acc)[kN / 8][4], uint32_t q, uint32_t k, int lane) {
  constexpr int kRow = Chunk<D>::kStride * 2;
#pragma unroll
  for (int n = 0; n < kN / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
  const uint32_t qa = q + (lane & 15) * kRow + (lane >> 4) * 16;
  const uint32_t ka = k + ((lane & 7) + ((lane >> 4) << 3)) * kRow + ((lane >> 3) & 1) * 16;
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    uint32_t qf[4];
    ldmatrix4(qf, qa + 32 * c);
#pragma unroll
    for (int n = 0; n < kN / 16; ++n) {
      uint32_t kf[4];
      ldmatrix4(kf, ka + n * 16 * kRow + 32 * c);
      mma_bf16(acc[2 * n], qf[0], qf[1], qf[2], qf[3], kf[0], kf[1]);
      mma_bf16(acc[2 * n + 1], qf[0], qf[1], qf[2], qf[3], kf[2], kf[3]);
    }
  }
}

template <int D>
__global__ void __launch_bounds__(kThreads) kv4_chunk_kernel(const AttnArgs a, const int64_t tiles_q) {
  using T = Chunk<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_limit[kM];
  __shared__ uint32_t flags[kN];
  grid_dependency_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int64_t rows = a.group * a.seq;
  const int64_t bh = blockIdx.x / tiles_q, b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
  // last tiles first: under a causal mask they are the longest
  const int64_t row0 = (tiles_q - 1 - (blockIdx.x - bh * tiles_q)) * kM;

  if (threadIdx.x < kM) {
    const int64_t r = row0 + threadIdx.x;
    s_limit[threadIdx.x] = r < rows ? visible_rows(a, b, r % a.seq) : -1;
    flags[threadIdx.x] = 0;
  }
  fill_queries<D>(smem + T::kQ, a, b, hk, row0, rows);
  __syncthreads();
  int limit = 0, lowest = INT32_MAX;
  for (int r = 0; r < kM; ++r) {
    limit = max(limit, s_limit[r]);
    if (s_limit[r] >= 0) lowest = min(lowest, s_limit[r]);
  }
  const int lim[2] = {s_limit[16 * warp + g], s_limit[16 * warp + g + 8]};
  const int64_t head_row = bh * a.c.cache_len;
  const uint8_t* kc = a.c.k_codes + head_row * (D / 2);
  const uint8_t* vc = a.c.v_codes + head_row * (D / 2);
  const uint32_t* ks = a.c.k_scales + head_row * T::kGroups;
  const uint32_t* vs = a.c.v_scales + head_row * T::kGroups;
  const uint32_t sq = smem_addr(smem + T::kQ) + 16 * warp * T::kStride * 2;
  const uint32_t sk = smem_addr(smem + T::kK), sv = smem_addr(smem + T::kV);

  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
  uint32_t bad[2] = {0, 0};

  for (int first = 0; first < limit; first += kN) {
    // A value that is not finite in a row that some of the queries must not see:
    // see fill_tile; the queries that do see it are marked below.
    const bool border = first + kN > lowest;
    fill_tile<D>(smem + T::kK, kc, ks, first, limit, nullptr);
    const bool met = fill_tile<D>(smem + T::kV, vc, vs, first, limit, border ? flags : nullptr);
    const bool any_bad = __syncthreads_or(met);

    float acc[kN / 8][4];
    tile_scores<D>(acc, sq, sk, lane);
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int n = 0; n < kN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = first + 8 * n + 2 * t + (e & 1);
        acc[n][e] = at < lim[e >> 1] ? acc[n][e] * a.scale_log2 : -INFINITY;
        top[e >> 1] = max_nan(top[e >> 1], acc[n][e]);
      }
    float f[2], shift[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = max_nan(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = max_nan(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      f[h] = m[h] == -INFINITY ? 0.0f : exp2_approx(m[h] - top[h]);
      l[h] *= f[h];
      m[h] = top[h];
      shift[h] = m[h] == -INFINITY ? 0.0f : m[h];
    }
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      o[j][0] *= f[0];
      o[j][1] *= f[0];
      o[j][2] *= f[1];
      o[j][3] *= f[1];
    }
    uint32_t p[kN / 8][2];
#pragma unroll
    for (int n = 0; n < kN / 8; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float p0 = exp2_approx(acc[n][2 * h] - shift[h]), p1 = exp2_approx(acc[n][2 * h + 1] - shift[h]);
        l[h] += p0 + p1;
        p[n][h] = pack_bf16x2(p0, p1);
      }
    if (any_bad) {
      for (int r = 0; r < kN; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (first + r < lim[h]) bad[h] |= flags[r];
    }
    const uint32_t va = sv + ((lane & 7) + ((lane >> 3) & 1) * 8) * (T::kStride * 2) + (lane >> 4) * 16;
#pragma unroll
    for (int n = 0; n < kN / 16; ++n)
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t vf[4];
        ldmatrix4_trans(vf, va + n * 16 * T::kStride * 2 + 32 * j);
        mma_bf16(o[2 * j], p[2 * n][0], p[2 * n][1], p[2 * n + 1][0], p[2 * n + 1][1], vf[0], vf[1]);
        mma_bf16(o[2 * j + 1], p[2 * n][0], p[2 * n][1], p[2 * n + 1][0], p[2 * n + 1][1], vf[2], vf[3]);
      }
    __syncthreads();
    if (any_bad) {  // uniform over the CTA
      if (threadIdx.x < kN) flags[threadIdx.x] = 0;
      __syncthreads();
    }
  }

#pragma unroll
  for (int h = 0; h < 2; ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    const int64_t r = row0 + 16 * warp + g + 8 * h;
    if (r >= rows) continue;
    const int64_t head = hk * a.group + r / a.seq, s = r % a.seq;
    const float inv = l[h] == 0.0f ? 0.0f : 1.0f / l[h];
    if (a.lse != nullptr && t == 0)
      a.lse[(b * a.heads + head) * a.seq + s] = m[h] == -INFINITY ? -INFINITY : m[h] + log2f(l[h]);
    const int64_t at = ((b * a.seq + s) * a.heads + head) * D;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      // columns 2t and 2t + 1 of 8 are elements t and t + 4
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int d = 8 * j + t + 4 * e;
        float x = o[j][2 * h + e] * inv;
        if (bad[h] >> (d / kKv4Group) & 1u) x = __int_as_float(0x7fc00000);
        if (a.gate != nullptr) x *= 1.0f / (1.0f + __expf(-bf16_to_f32(a.gate[at + d])));
        a.out[at + d] = f32_to_bf16(x);
      }
    }
  }
}

// weights[j] += the probabilities of cache row j, summed over the query rows in
// their order: a CTA owns kN cache rows, keeps their keys in shared memory and
// recomputes the scores of all queries, 64 rows at a time.  No atomics: the
// sums have one order whatever the launch.
template <int D>
__global__ void __launch_bounds__(kThreads) kv4_weights_kernel(const AttnArgs a, const int64_t tiles_k) {
  using T = Chunk<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_limit[kM];
  __shared__ float s_lse[kM];
  __shared__ float s_sum[4][kN];
  grid_dependency_begin();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int64_t rows = a.group * a.seq;
  const int64_t bh = blockIdx.x / tiles_k, b = bh / a.kv_heads, hk = bh - b * a.kv_heads;
  const int first = (int)(blockIdx.x - bh * tiles_k) * kN;
  const int limit = visible_rows(a, b, a.seq - 1);  // of the last query: the highest
  if (first >= limit) return;
  const int64_t head_row = bh * a.c.cache_len;
  fill_tile<D>(smem + T::kK, a.c.k_codes + head_row * (D / 2), a.c.k_scales + head_row * T::kGroups, first, limit,
               nullptr);
  const uint32_t sq = smem_addr(smem + T::kQ) + 16 * warp * T::kStride * 2, sk = smem_addr(smem + T::kK);
  float sum[kN / 8][2];
#pragma unroll
  for (int n = 0; n < kN / 8; ++n) sum[n][0] = sum[n][1] = 0.0f;

  for (int64_t row0 = 0; row0 < rows; row0 += kM) {
    __syncthreads();
    if (threadIdx.x < kM) {
      const int64_t r = row0 + threadIdx.x;
      s_limit[threadIdx.x] = r < rows ? visible_rows(a, b, r % a.seq) : -1;
      s_lse[threadIdx.x] = r < rows ? a.lse[(b * a.heads + hk * a.group + r / a.seq) * a.seq + r % a.seq] : 0.0f;
    }
    if (!__syncthreads_or(threadIdx.x < kM && s_limit[threadIdx.x] > first)) continue;  // no query here sees the tile
    fill_queries<D>(smem + T::kQ, a, b, hk, row0, rows);
    __syncthreads();
    float acc[kN / 8][4];
    tile_scores<D>(acc, sq, sk, lane);
    const int lim[2] = {s_limit[16 * warp + g], s_limit[16 * warp + g + 8]};
    const float lse[2] = {s_lse[16 * warp + g], s_lse[16 * warp + g + 8]};
#pragma unroll
    for (int n = 0; n < kN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int at = first + 8 * n + 2 * t + (e & 1), h = e >> 1;
        if (at < lim[h]) sum[n][e & 1] += exp2_approx(acc[n][e] * a.scale_log2 - lse[h]);
      }
  }
#pragma unroll
  for (int n = 0; n < kN / 8; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = sum[n][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) s_sum[warp][8 * n + 2 * t + e] = x;
    }
  __syncthreads();
  const int at = first + threadIdx.x;
  if (threadIdx.x < kN && at < limit)
    a.c.weights[head_row + at] += (s_sum[0][threadIdx.x] + s_sum[1][threadIdx.x]) +
                                  (s_sum[2][threadIdx.x] + s_sum[3][threadIdx.x]);
}

template <int D>
cudaError_t launch_chunk(const AttnArgs& a, cudaStream_t s) {
  const int64_t tiles = ((int64_t)a.group * a.seq + kM - 1) / kM, grid = a.batch * a.kv_heads * tiles;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  const cudaError_t e = allow_shared<kv4_chunk_kernel<D>>(Chunk<D>::kSmem);
  if (e != cudaSuccess) return e;
  return launch_kernel(kv4_chunk_kernel<D>, grid, kThreads, Chunk<D>::kSmem, s, a, tiles);
}

template <int D>
cudaError_t launch_weights(const AttnArgs& a, int64_t longest, cudaStream_t s) {
  const int64_t tiles = (longest + kN - 1) / kN, grid = a.batch * a.kv_heads * tiles;
  if (grid > INT32_MAX) return cudaErrorInvalidConfiguration;
  const cudaError_t e = allow_shared<kv4_weights_kernel<D>>(Chunk<D>::kV);
  if (e != cudaSuccess) return e;
  return launch_kernel(kv4_weights_kernel<D>, grid, kThreads, Chunk<D>::kV, s, a, tiles);
}

}  // namespace

cudaError_t launch_kv4_chunk(const AttnArgs& a, int64_t head_dim, cudaStream_t s) {
  return head_dim == 192 ? launch_chunk<192>(a, s) : launch_chunk<256>(a, s);
}

cudaError_t launch_kv4_weights(const AttnArgs& a, int64_t head_dim, int64_t longest, cudaStream_t s) {
  switch (head_dim) {
    case 64: return launch_weights<64>(a, longest, s);
    case 128: return launch_weights<128>(a, longest, s);
    case 192: return launch_weights<192>(a, longest, s);
    default: return launch_weights<256>(a, longest, s);
  }
}

}  // namespace hrm
