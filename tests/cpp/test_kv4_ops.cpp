// Tests of the C++ host layer's 4-bit KV cache: a prompt, an eviction and decoding
// steps through HrmLayerOps, against plain double-precision attention over the values
// that the cache stands for; and the refusals.  Needs a GPU; prints one line per
// test and exits non-zero on the first failure.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <string>
#include <vector>

#include "hrm_layer_ops.hpp"

using hrm::bf16;
using hrm::CudaSlice;
using hrm::HrmError;
using hrm::HrmLayerOps;

namespace {

struct Failure {
  std::string what;
};
void expect(bool ok, const std::string& what) {
  if (!ok) throw Failure{what};
}

template <class T>
std::vector<T> to_host(const HrmLayerOps& m, const CudaSlice<T>& s) {
  std::vector<T> v(s.len());
  expect(cudaStreamSynchronize(m.cu_stream()) == cudaSuccess, "synchronize");
  expect(cudaMemcpy(v.data(), s.device_ptr(), s.len() * sizeof(T), cudaMemcpyDeviceToHost) == cudaSuccess, "copy");
  return v;
}

std::vector<float> noise(size_t n, uint32_t seed) {
  std::vector<float> v(n);
  uint32_t x = seed * 2654435761u + 1;
  for (float& f : v) {
    x = x * 1664525u + 1013904223u;
    f = (float)(int32_t)x * (1.0f / 2147483648.0f);
  }
  return v;
}
std::vector<bf16> to_bf16(const std::vector<float>& v) {
  std::vector<bf16> o;
  for (float x : v) o.push_back(bf16::from_f32(x));
  return o;
}

// The values of row `row` (of all batch * kv_heads * cache_len).
std::vector<double> row_values(const std::vector<uint8_t>& codes, const std::vector<uint32_t>& scales, size_t row,
                               size_t dim) {
  std::vector<double> v(dim);
  for (size_t e = 0; e < dim; ++e) {
    const uint32_t sz = scales[row * (dim / 32) + e / 32];
    bf16 s, z;
    s.bits = (uint16_t)(sz & 0xffff);
    z.bits = (uint16_t)(sz >> 16);
    const uint32_t code = codes[row * (dim / 2) + e / 2] >> (4 * (e & 1)) & 15;
    v[e] = bf16::from_f32(s.to_f32() * (1.0f + code / 16.0f) + z.to_f32()).to_f32();
  }
  return v;
}

// out of query (head, s) of sequence 0 over rows [0, limit), times sigmoid(gate).
std::vector<double> attend(const std::vector<std::vector<double>>& k, const std::vector<std::vector<double>>& v,
                           const float* q, const float* gate, size_t dim, size_t limit, double scale) {
  std::vector<double> p(limit), out(dim, 0.0);
  double top = -INFINITY, sum = 0;
  for (size_t j = 0; j < limit; ++j) {
    double x = 0;
    for (size_t e = 0; e < dim; ++e) x += q[e] * k[j][e];
    top = std::max(top, p[j] = x * scale);
  }
  for (double& x : p) sum += x = std::exp(x - top);
  for (size_t j = 0; j < limit; ++j)
    for (size_t e = 0; e < dim; ++e) out[e] += p[j] / sum * v[j][e];
  for (size_t e = 0; e < dim; ++e) out[e] /= 1.0 + std::exp(-(double)gate[e]);
  return out;
}

constexpr size_t kHeads = 2, kDim = 64, kCache = 96;

// A prompt of `seq` tokens into an empty cache (split, attention with gate and
// accumulated weights), checked against the cache's own values.  The output's
// rounding is 2^-8 of itself, the probabilities' 2^-8 of the values (|v| <= 1.1).
void step(HrmLayerOps& m, HrmLayerOps::Kv4Cache& cache, size_t seq, size_t at, size_t position, uint32_t seed) {
  const size_t n = seq * kHeads * kDim;
  auto gqkv = m.htod_copy_bf16(to_bf16(noise(4 * n, seed)));
  auto gate = m.alloc_zero_bf16(n), q = m.alloc_zero_bf16(n), out = m.alloc_zero_bf16(n);
  m.split_gqkv_rope_kv4(gqkv, gate, q, nullptr, nullptr, cache, seq, position, at);
  const float scale = 1.0f / std::sqrt((float)kDim);
  m.kv4_attention(q, cache, &gate, out, kHeads, seq, at, 0, scale, true);
  const auto kc = to_host(m, cache.k_codes), vc = to_host(m, cache.v_codes);
  const auto ks = to_host(m, cache.k_scales), vs = to_host(m, cache.v_scales);
  const auto hq = to_host(m, q), hg = to_host(m, gate), ho = to_host(m, out);
  for (size_t h = 0; h < kHeads; ++h) {
    std::vector<std::vector<double>> k, v;
    for (size_t j = 0; j < at + seq; ++j) {
      k.push_back(row_values(kc, ks, h * kCache + j, kDim));
      v.push_back(row_values(vc, vs, h * kCache + j, kDim));
    }
    for (size_t s = 0; s < seq; ++s) {
      std::vector<float> fq(kDim), fg(kDim);
      for (size_t e = 0; e < kDim; ++e) {
        fq[e] = hq[(h * seq + s) * kDim + e].to_f32();
        fg[e] = hg[(s * kHeads + h) * kDim + e].to_f32();
      }
      const auto want = attend(k, v, fq.data(), fg.data(), kDim, at + s + 1, scale);
      for (size_t e = 0; e < kDim; ++e) {
        const double got = ho[(s * kHeads + h) * kDim + e].to_f32();
        expect(std::fabs(got - want[e]) <= std::ldexp(std::fabs(want[e]), -8) + std::ldexp(1.1, -8),
               "head " + std::to_string(h) + " query " + std::to_string(s) + " element " + std::to_string(e));
      }
    }
  }
}

void test_serving_loop(HrmLayerOps& m) {
  auto cache = m.alloc_kv4_cache(1, kHeads, kCache, kDim, true);
  auto lengths = m.htod_copy_i32({-1});
  step(m, cache, 70, 0, 0, 1);
  size_t length = 70, position = 70;
  for (uint32_t t = 0; t < 4; ++t) {
    // 40 rows stay, the last 8 tokens among them
    m.kv4_evict(cache, length, 40, (int64_t)position - 8, lengths);
    expect(to_host(m, lengths)[0] == 40, "new length");
    length = 40;
    const auto pos = to_host(m, cache.positions);
    for (size_t h = 0; h < kHeads; ++h)
      for (size_t p = position - 8; p < position; ++p)
        expect(std::count(pos.begin() + h * kCache, pos.begin() + h * kCache + 40, (int32_t)p) == 1,
               "a protected token stays");
    step(m, cache, 1, length, position, 2 + t);
    ++length;
    ++position;
  }
  // every query's probabilities sum to 1, so what is left weighs less than all of them
  const auto w = to_host(m, cache.weights);
  for (size_t h = 0; h < kHeads; ++h) {
    double sum = 0;
    for (size_t j = 0; j < length; ++j) sum += w[h * kCache + j];
    expect(sum > 1.0 && sum < 74.0 * 1.001, "accumulated weights");
  }
}

// update's rows read back as the formula says, and only those rows are written.
void test_update_in_place(HrmLayerOps& m) {
  auto cache = m.alloc_kv4_cache(2, kHeads, kCache, kDim);
  const size_t seq = 3;
  auto off = m.htod_copy_i32({5, 90});
  const auto hk = to_bf16(noise(2 * kHeads * seq * kDim, 9)), hv = to_bf16(noise(2 * kHeads * seq * kDim, 10));
  auto k = m.htod_copy_bf16(hk), v = m.htod_copy_bf16(hv);
  m.kv4_update(cache, k, v, seq, 0, 0, nullptr, &off);
  const auto kc = to_host(m, cache.k_codes);
  const auto ks = to_host(m, cache.k_scales);
  const size_t at[2] = {5, 90};
  for (size_t b = 0; b < 2; ++b)
    for (size_t h = 0; h < kHeads; ++h)
      for (size_t j = 0; j < kCache; ++j) {
        const size_t row = (b * kHeads + h) * kCache + j;
        if (j < at[b] || j >= at[b] + seq) {
          expect(ks[row * 2] == 0 && ks[row * 2 + 1] == 0 && kc[row * 32] == 0, "a row outside is left alone");
          continue;
        }
        const auto got = row_values(kc, ks, row, kDim);
        for (size_t e = 0; e < kDim; ++e) {
          const double want = hk[((b * kHeads + h) * seq + j - at[b]) * kDim + e].to_f32();
          // half a step of range (<= 2) / 15, S and Z rounded to bf16 (|Z| <= 3.2, S <= 2.14), the value too
          expect(std::fabs(got[e] - want) <= 1.0 / 15 + 3.2 / 256 + 4.3 / 256 + 1.1 / 256, "value");
        }
      }
}

void test_refusals(HrmLayerOps& m) {
  auto refused = [&](const std::function<void()>& f, const char* what) {
    try {
      f();
    } catch (const HrmError& e) {
      expect(e.kind() == HrmError::Kind::InvalidInput, std::string(what) + ": kind");
      return;
    }
    throw Failure{std::string(what) + " was accepted"};
  };
  auto cache = m.alloc_kv4_cache(1, kHeads, kCache, kDim);
  auto x = m.alloc_zero_bf16(kHeads * kDim), small = m.alloc_zero_bf16(kDim), out = m.alloc_zero_bf16(kHeads * kDim);
  auto lengths = m.htod_copy_i32({0});
  refused([&] { m.alloc_kv4_cache(1, 1, 8, 96); }, "head_dim 96");
  refused([&] { m.kv4_update(cache, x, small, 1, 0, 0); }, "a short v");
  refused([&] { m.kv4_update(cache, x, x, 1, 0, kCache); }, "a row past the cache");
  refused([&] { m.kv4_attention(x, cache, nullptr, out, kHeads, 1, kCache, 0, 1.0f); }, "an offset past the cache");
  refused([&] { m.kv4_attention(x, cache, nullptr, small, kHeads, 1, 0, 0, 1.0f); }, "a short output");
  refused([&] { m.kv4_attention(x, cache, nullptr, out, kHeads, 1, 0, 0, 1.0f, true); }, "accumulate without weights");
  refused([&] { m.kv4_evict(cache, 8, 4, 0, lengths); }, "eviction without weights");
  cache.cache_len *= 2;
  refused([&] { m.kv4_update(cache, x, x, 1, 0, 0); }, "a cache longer than its buffers");
}

}  // namespace

int main() {
  const std::vector<std::pair<const char*, std::function<void(HrmLayerOps&)>>> tests = {
      {"test_update_in_place", test_update_in_place},
      {"test_serving_loop", test_serving_loop},
      {"test_refusals", test_refusals},
  };
  try {
    HrmLayerOps m(0);
    for (const auto& t : tests) {
      try {
        t.second(m);
      } catch (const Failure& f) {
        std::printf("FAIL %s: %s\n", t.first, f.what.c_str());
        return 1;
      }
      std::printf("ok   %s\n", t.first);
    }
  } catch (const HrmError& e) {
    std::printf("FAIL HrmError: %s\n", e.what());
    return 1;
  }
  std::printf("all kv4 tests passed\n");
  return 0;
}
