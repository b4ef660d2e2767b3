// The rotation's arithmetic, shared by the RoPE kernels and the 4-bit cache
// write, so that both round every element alike.
#pragma once

#include "common.cuh"

namespace hrm {

__device__ __forceinline__ float rope_angle(int pos, int i, int head_dim, float theta) {
  return (float)pos * expf(-2.0f * i * logf(theta) / (float)head_dim);
}

// x0' and x1' of one pair, rounded as the reference kernel rounds them.
__device__ __forceinline__ float rot_lo(float x0, float x1, float c, float s) {
  return __fmaf_rn(x0, c, -__fmul_rn(x1, s));
}
__device__ __forceinline__ float rot_hi_q(float x0, float x1, float c, float s) {
  return __fmaf_rn(x1, c, __fmul_rn(x0, s));
}
__device__ __forceinline__ float rot_hi_k(float x0, float x1, float c, float s) {
  return __fmaf_rn(x0, s, __fmul_rn(x1, c));
}

template <bool IS_K>
__device__ __forceinline__ void rotate8(uint4& lo, uint4& hi, const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t wl = vget(lo, w), wh = vget(hi, w);
    const float x0a = bf16_lo(wl), x0b = bf16_hi(wl);
    const float x1a = bf16_lo(wh), x1b = bf16_hi(wh);
    const float ca = c[2 * w], sa = s[2 * w], cb = c[2 * w + 1], sb = s[2 * w + 1];
    vset(lo, w, pack_bf16x2(rot_lo(x0a, x1a, ca, sa), rot_lo(x0b, x1b, cb, sb)));
    if (IS_K)
      vset(hi, w, pack_bf16x2(rot_hi_k(x0a, x1a, ca, sa), rot_hi_k(x0b, x1b, cb, sb)));
    else
      vset(hi, w, pack_bf16x2(rot_hi_q(x0a, x1a, ca, sa), rot_hi_q(x0b, x1b, cb, sb)));
  }
}

// cos/sin of pairs 8j..8j+7 at position pos from the table.
__device__ __forceinline__ void table_cos_sin(const float4* table, int pos, int j, int head_dim, float (&c)[8],
                                              float (&sn)[8]) {
  const float4* row = table + (int64_t)pos * (head_dim / 4);
  const float4 c0 = ld_keep(row + 2 * j), c1 = ld_keep(row + 2 * j + 1);
  const float4 s0 = ld_keep(row + head_dim / 8 + 2 * j), s1 = ld_keep(row + head_dim / 8 + 2 * j + 1);
  c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
  sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
}

}  // namespace hrm
