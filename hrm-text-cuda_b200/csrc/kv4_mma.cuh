// Warp-level helpers of the attention kernels over the 4-bit cache.
#pragma once

#include "kv4.cuh"

namespace hrm {

__device__ __forceinline__ float exp2_approx(float x) {  // 2^x, within 2 ulp; 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// sigmoid(g), what the gate of an output multiplies it by.  __expf(x) is good to 2 + 1.173 |x|
// ulp, the reciprocal to 1: within 5 + 1.2 |g| ulp of fp32, 2^-16 of itself where the
// factor is smallest (g near -87), well below the rounding of the bf16 product, 2^-8.
// (The exact division is a call of some 40 instructions; in a prompt's 128 x 256
// outputs per CTA it took as long as 4 tiles.)
__device__ __forceinline__ float gate_factor(float g) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + __expf(-g)));
  return y;
}
// D = A (16x16, row) * B (16x8, col) + D, bf16 operands, fp32 accumulators.
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
// cp.async of BYTES (8 or 16) global -> shared; zeros where !valid (src is not read then).
template <int BYTES>
__device__ __forceinline__ void cp_async_zfill(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? BYTES : 0;
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;\n" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n)
                 : "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

// Query rows of one kv head up to which the probabilities are added to the
// weights by the decode kernel itself (one block of rows holds them all).  It keeps the
// scores for that; the kernel that computes them again takes longer (16 x 16 heads
// over 8192 rows, 1 query row: 87 us against 433; 8 rows: 156 against 452).
constexpr int64_t kDecodeRows = 8;
// And up to which it keeps the scores, for a kernel that adds several blocks' up:
// 4 bytes per row and cache row, against the 160 that the cache has of head_dim 128.
constexpr int64_t kScoreRows = 16;
// Query rows of one kv head up to which the decode kernel serves them, in blocks of 8, with
// 16 bits of a probability where the prompts' kernel has 8.  12 heads of 128, decode
// kernel against the prompts': 17 to 24 rows over 1024 11.3 and 12.1 us, a batch of 8 18.9
// and 21.7, over 8192 29 to 32 and 25, a batch of 8 101 to 103 and 128; 32 rows 13.0 and
// 12.1, 28 and 21, 37 and 24, 130 and 120.  So a fourth block makes it the slower one, by
// up to 1.6 times; those rows are served by it for its bits.
constexpr int64_t kChunkRows = 32;

// What every attention kernel is given.
struct AttnArgs {
  const uint4* q;        // [batch, heads, seq, D] bf16
  const uint16_t* gate;  // [batch, seq, heads, D] bf16, or null
  uint16_t* out;         // [batch, seq, heads, D] bf16
  Kv4View c;
  int64_t batch;
  int heads, kv_heads, group, seq;  // group * seq * batch * kv_heads fits in 31 bits
  int64_t cache_offset;
  const int* cache_offsets;  // per sequence, or null
  int64_t prefix_len;
  float scale_log2;  // softmax scale * log2(e)
  // Weights wanted: up to kScoreRows rows [batch * kv_heads, rows, cache_len] scores (log2
  // units); past kDecodeRows [batch, heads, seq], log2 of each row's sum of 2^score.
  float* scores;
  float* lse;
};

// Cache rows that the queries of a sequence see: query s rows [0, rows(s)).
struct Visible {
  int64_t off, prefix, top;
  __device__ __forceinline__ Visible(const AttnArgs& a, int b)
      : off(a.cache_offsets ? a.cache_offsets[b] : a.cache_offset), prefix(a.prefix_len) {
    top = off + a.seq < a.c.cache_len ? off + a.seq : a.c.cache_len;
  }
  __device__ __forceinline__ int rows(int s) const {
    int64_t lim = off + s + 1;
    if (lim < prefix) lim = prefix;
    if (lim > top) lim = top;
    return lim < 0 ? 0 : (int)lim;
  }
};
__device__ __forceinline__ int visible_rows(const AttnArgs& a, int b, int s) { return Visible(a, b).rows(s); }

}  // namespace hrm
