// The 4-bit KV cache's number format, shared by the kernels that write, read
// and move it.
//
// A row of head_dim elements is cut into groups of 32 consecutive elements.
// A group holds a 4-bit code n per element and two bf16 numbers (S, Z):
//   value = bf16_rn(S * (1 + n / 16) + Z)
// with, for the group's smallest and largest element lo and hi,
//   S = bf16_rn((hi - lo) * 16/15)   (0 where hi - lo < 2^-100)
//   Z = bf16_rn(lo - S)
//   n = clamp(rint((x - Z) * (16 / S) - 16), 0, 15)   (0 where S == 0)
// in fp32, each operation rounded to nearest even.  One step is S / 16 =
// (hi - lo) / 15; the roundings of S and Z to 8 significant bits move the grid by
// at most 2^-8 of (hi - lo) and 2^-8 of |lo - S| (a tenth of a step for values
// around zero), and n is taken against the rounded grid.  A group that holds a NaN or an infinity, or whose
// S, Z or largest value S * 31/16 + Z is out of bf16's range, gets S = NaN and reads back as NaN.
//
// Why 1 + n/16 and not n: the bf16 pattern 0x3f80 | n << 3 IS 1 + n/16, so a
// code becomes a bf16 operand with one shift and one and-or (two elements at
// a time), and one packed fma with a single rounding gives the value.
#pragma once

#include "common.cuh"

namespace hrm {

constexpr int kKv4Group = 32;  // elements per (S, Z) pair

// The cache's buffers: per (batch, kv head, row) head_dim / 2 bytes of codes
// (element 2i in the low nibble of byte i) and head_dim / 32 words (S in the low
// half, Z in the high half); optionally an fp32 weight and an int32 position.
struct Kv4View {
  uint8_t* k_codes;
  uint32_t* k_scales;
  uint8_t* v_codes;
  uint32_t* v_scales;
  float* weights;
  int* positions;
  int64_t cache_len;
};

__device__ __forceinline__ float min_nan(float a, float b) {  // NaN where either is
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
// Both halves of a (S, Z) word, each duplicated into a packed pair.
__device__ __forceinline__ uint32_t kv4_scale2(uint32_t sz) { return __byte_perm(sz, sz, 0x1010); }
__device__ __forceinline__ uint32_t kv4_base2(uint32_t sz) { return __byte_perm(sz, sz, 0x3232); }

// A word (S, Z) some of whose 16 values are not finite: those lie between S + Z and
// S * 31/16 + Z, which is a NaN or an infinity where S or Z is.
__device__ __forceinline__ bool kv4_not_finite(uint32_t sz) {
  const uint32_t x = fma_bf16x2(0x3ff83f80u, kv4_scale2(sz), kv4_base2(sz));
  return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}

// 1 + n/16 of nibbles P and P + 4 of w, as a packed bf16 pair: one shift and one
// three-input and-or (written out: the compiler made two instructions of it).
// Extracting nibbles 0 and 1 without a shift, by packed fmas that scale the masked
// bits, measured slower: the fma's pipe is no less busy, and denormal operands
// (bits 4-7 alone) cost it several times a normal one.
template <int P>
__device__ __forceinline__ uint32_t kv4_pair(uint32_t w) {
  const uint32_t x = P == 0 ? w << 3 : w >> (P == 0 ? 0 : 4 * P - 3);
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(x), "r"(0x00780078u), "r"(0x3f803f80u));
  return r;
}

// Quantises 8 elements per lane; the 4 lanes of an aligned quad hold one group
// (`quad` is their lane mask).  Returns the 8 codes (element i in nibble i);
// sz receives the group's (S, Z) word.
__device__ __forceinline__ uint32_t kv4_quantise(const uint4& x, uint32_t quad, uint32_t& sz) {
  float f[8];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[2 * w] = bf16_lo(vget(x, w));
    f[2 * w + 1] = bf16_hi(vget(x, w));
  }
  float lo = f[0], hi = f[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = min_nan(lo, f[i]);
    hi = max_nan(hi, f[i]);
  }
#pragma unroll
  for (int m = 1; m <= 2; m *= 2) {
    lo = min_nan(lo, __shfl_xor_sync(quad, lo, m));
    hi = max_nan(hi, __shfl_xor_sync(quad, hi, m));
  }
  const float range = __fsub_rn(hi, lo);
  const uint32_t s = range < 0x1p-100f ? 0u : f32_to_bf16(__fmul_rn(range, 16.0f / 15.0f));
  const float scale = bf16_to_f32((uint16_t)s);
  const uint32_t z = f32_to_bf16(__fsub_rn(lo, scale));
  const float base = bf16_to_f32((uint16_t)z);
  sz = s | z << 16;
  if (kv4_not_finite(sz)) {
    sz = 0x00007fc0u;  // S = NaN, Z = 0
    return 0;
  }
  if (s == 0) return 0;
  const float inv = __fdiv_rn(16.0f, scale);
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float t = __fsub_rn(__fmul_rn(__fsub_rn(f[i], base), inv), 16.0f);
    // rint by adding 1.5 * 2^23: the integer lands in the low mantissa bits
    const float r = __fadd_rn(fminf(fmaxf(t, 0.0f), 15.0f), 12582912.0f);
    codes |= (__float_as_uint(r) & 15u) << (4 * i);
  }
  return codes;
}

// The 8 values that a lane's codes stand for, in element order.
__device__ __forceinline__ uint4 kv4_values(uint32_t codes, uint32_t sz) {
  const uint32_t s2 = kv4_scale2(sz), z2 = kv4_base2(sz);
  uint4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t c = codes >> (8 * w);
    vset(v, w, fma_bf16x2(((c & 15u) << 3) | ((c & 0xf0u) << 15) | 0x3f803f80u, s2, z2));
  }
  return v;
}

}  // namespace hrm
