// What the prompts' attention kernels leave where a bounded wait ran out.  Needs a GPU;
// exits non-zero on a failure.  No wait of a running kernel is made to run out: the
// wait is tested alone, on a barrier that nothing completes, with a deadline of 50 ms;
// and what a kernel leaves then is set from the host between two kernels.
//   1. mbar_wait_bounded returns true for a barrier that completes, false after the
//      deadline for one that does not, and counts itself;
//   2. the rows of a partial result that is marked are not written by the joining
//      kernel, whichever part has the mark, and their log-sum is +inf; the others
//      are written bit for bit as without marks;
//   3. rows whose log-sum is +inf add nothing to the weights.
#include <chrono>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#define HRM_WAIT_LIMIT_NS 50000000ull
#include "kv4_prefill.cu"

namespace hrm {
int device_sm_count() { return 148; }
}  // namespace hrm

// (not unnamed: the included file has one of those with kernels in it)
namespace timeout_test {
using namespace hrm;

int g_failures = 0;
void expect(bool ok, const char* what) {
  if (!ok) {
    std::printf("FAIL %s\n", what);
    ++g_failures;
  }
}
bool cuda_ok(cudaError_t e, const char* what) {
  if (e != cudaSuccess) std::printf("FAIL %s: %s\n", what, cudaGetErrorString(e));
  return e == cudaSuccess;
}

__global__ void wait_kernel(bool arrive, int* result) {
  __shared__ uint64_t bar;
  const uint32_t b = smem_addr(&bar);
  mbar_init(b, 1);
  mbar_init_fence();
  if (arrive) mbar_arrive(b);
  *result = mbar_wait_bounded(b, 0) ? 1 : 0;
}

bool test_wait() {
  int *d = nullptr, r = -1;
  if (!cuda_ok(cudaMalloc(&d, sizeof(int)), "cudaMalloc")) return false;
  for (int arrive = 1; arrive >= 0; --arrive) {
    const auto t0 = std::chrono::steady_clock::now();
    wait_kernel<<<1, 1>>>(arrive != 0, d);
    if (!cuda_ok(cudaDeviceSynchronize(), "wait_kernel")) return false;
    const double ms = std::chrono::duration<double, std::milli>(std::chrono::steady_clock::now() - t0).count();
    cudaMemcpy(&r, d, sizeof(int), cudaMemcpyDeviceToHost);
    expect(r == arrive, "what the wait returns");
    if (!arrive) expect(ms >= 45.0 && ms <= 5000.0, "the deadline");
  }
  unsigned int n = 0;
  expect(kv4_prefill_wait_timeouts(&n, true) == cudaSuccess && n == 1, "the count");
  expect(kv4_prefill_wait_timeouts(&n, false) == cudaSuccess && n == 0, "the count, reset");
  cudaFree(d);
  return true;
}

// A case of the split attention: heads of kSeq queries over kCache rows of 128.
constexpr int kD = 128, kNq = 2, kHeads = 2, kSeq = 300, kCache = 1500, kOffset = kCache - kSeq, kCount = 3;
constexpr int kBlocks = (kSeq + kNq * kM - 1) / (kNq * kM), kItems = kHeads * kBlocks;

struct Case {
  AttnArgs a{};
  PrefillSplit split{kCount, nullptr};
  std::vector<void*> buffers;
  template <class T>
  T* put(const std::vector<T>& v) {
    void* p = nullptr;
    if (!cuda_ok(cudaMalloc(&p, v.size() * sizeof(T)), "cudaMalloc")) return nullptr;
    cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice);
    buffers.push_back(p);
    return static_cast<T*>(p);
  }
  ~Case() {
    for (void* p : buffers) cudaFree(p);
  }
  bool make() {
    uint32_t x = 7;
    auto next = [&]() { return (x = x * 1664525u + 1013904223u) >> 8; };
    const size_t rows = (size_t)kHeads * kCache, queries = (size_t)kHeads * kSeq;
    std::vector<uint8_t> codes(rows * kD / 2);
    for (auto& c : codes) c = (uint8_t)next();
    std::vector<uint32_t> scales(rows * (kD / 32), 0x3f00u | 0xbf38u << 16);  // S = 0.5, Z = -0.71875
    std::vector<uint16_t> q(queries * kD);
    for (auto& e : q) e = (uint16_t)(0x3f00u | (next() & 0x7fu) | (next() & 1u) << 15);  // +-0.5 .. 1
    a.c.k_codes = put(codes);
    a.c.k_scales = put(scales);
    for (auto& c : codes) c = (uint8_t)next();
    a.c.v_codes = put(codes);
    a.c.v_scales = put(scales);
    a.c.weights = put(std::vector<float>(rows, 0.0f));
    a.c.cache_len = kCache;
    a.q = reinterpret_cast<const uint4*>(put(q));
    a.out = put(std::vector<uint16_t>(queries * kD, 0xabcd));
    a.lse = put(std::vector<float>(queries, -7.0f));
    split.parts = put(std::vector<float>((size_t)kItems * kCount * prefill_part(kNq, kD), 0.0f));
    a.batch = 1;
    a.heads = a.kv_heads = kHeads;
    a.group = 1;
    a.seq = kSeq;
    a.cache_offset = kOffset;
    a.scale_log2 = 0.125f;
    return split.parts != nullptr;
  }
};

bool join(Case& c) {
  return cuda_ok(launch_kernel(kv4_prefill_join_kernel<kD, kNq>, kItems * kNq * (kD / kJoinElements), kM, 0, nullptr, c.a,
                               c.split, kBlocks),
                 "kv4_prefill_join_kernel") &&
         cuda_ok(cudaDeviceSynchronize(), "synchronize");
}

bool test_marks() {
  Case c;
  if (!c.make()) return false;
  using T = Pre<kD, kNq>;
  if (!cuda_ok(allow_shared<kv4_prefill_kernel<kD, kNq>>(T::kSmem), "shared memory")) return false;
  if (!cuda_ok(has_registers<kv4_prefill_kernel<kD, kNq>>(T::kLaunchRegs), "registers")) return false;
  if (!cuda_ok(launch_kernel(kv4_prefill_kernel<kD, kNq>, kItems * kCount, T::kThreads, T::kSmem, nullptr, c.a, c.split,
                             kBlocks),
               "kv4_prefill_kernel") ||
      !join(c))
    return false;
  const size_t queries = (size_t)kHeads * kSeq, n = queries * kD;
  std::vector<uint16_t> want(n), got(n);
  std::vector<float> lse(queries), lse2(queries);
  cudaMemcpy(want.data(), c.a.out, n * 2, cudaMemcpyDeviceToHost);
  cudaMemcpy(lse.data(), c.a.lse, queries * 4, cudaMemcpyDeviceToHost);
  for (uint16_t e : want) expect((e & 0x7f80) != 0x7f80, "the output is finite");

  // marks in part (item % kCount) of every item, for the rows of one warp and some single ones
  auto marked = [](int r) { return (r >= 64 && r < 96) || r % 97 == 5; };
  const int64_t each = prefill_part(kNq, kD);
  std::vector<float> parts((size_t)kItems * kCount * each);
  cudaMemcpy(parts.data(), c.split.parts, parts.size() * 4, cudaMemcpyDeviceToHost);
  const uint32_t mark = 1u << 31;
  for (int item = 0; item < kItems; ++item)
    for (int r = 0; r < kNq * kM; ++r)
      if (marked(r))
        std::memcpy(&parts[(item * kCount + item % kCount) * each + kNq * kM * (kD + 2) + r], &mark, 4);
  cudaMemcpy(c.split.parts, parts.data(), parts.size() * 4, cudaMemcpyHostToDevice);
  cudaMemset(c.a.out, 0x5c, n * 2);
  if (!join(c)) return false;
  cudaMemcpy(got.data(), c.a.out, n * 2, cudaMemcpyDeviceToHost);
  cudaMemcpy(lse2.data(), c.a.lse, queries * 4, cudaMemcpyDeviceToHost);
  int skipped = 0;
  bool as_they_were = true, others = true, sums = true;
  for (int h = 0; h < kHeads; ++h)
    for (int s = 0; s < kSeq; ++s) {
      const bool m = marked(s % (kNq * kM));
      skipped += m;
      const uint16_t* row = &got[((size_t)s * kHeads + h) * kD];
      const uint16_t* before = &want[((size_t)s * kHeads + h) * kD];
      for (int d = 0; d < kD; ++d) (m ? as_they_were : others) &= row[d] == (m ? 0x5c5c : before[d]);
      const float l = lse2[(size_t)h * kSeq + s];
      sums &= m ? std::isinf(l) && l > 0 : l == lse[(size_t)h * kSeq + s];
    }
  expect(skipped > 64, "marked rows");
  expect(as_they_were, "a marked row is not written");
  expect(others, "the other rows are written as without marks");
  expect(sums, "log-sums: +inf where marked");

  // the weights without the marked rows: each of them would have added 1 in all
  double total[2];
  for (int pass = 0; pass < 2; ++pass) {
    const std::vector<float>& l = pass == 0 ? lse : lse2;
    cudaMemcpy(c.a.lse, l.data(), queries * 4, cudaMemcpyHostToDevice);
    cudaMemset(c.a.c.weights, 0, (size_t)kHeads * kCache * 4);
    if (!cuda_ok(launch_weights<kD>(c.a, kCache, nullptr), "kv4_weights_kernel") ||
        !cuda_ok(cudaDeviceSynchronize(), "synchronize"))
      return false;
    std::vector<float> w((size_t)kHeads * kCache);
    cudaMemcpy(w.data(), c.a.c.weights, w.size() * 4, cudaMemcpyDeviceToHost);
    total[pass] = 0;
    for (float x : w) total[pass] += x;
  }
  // fp32: scores of at most 128 * 0.25 * 0.125 = 4 in log2 units, off by (128 + 8) 2^-23 of that; sums of 300 terms
  expect(std::fabs(total[0] - queries) < 1e-3 * queries, "all weights");
  expect(std::fabs(total[1] - (queries - skipped)) < 1e-3 * queries, "weights without the marked rows");
  unsigned int waits = 1;
  expect(kv4_prefill_wait_timeouts(&waits, false) == cudaSuccess && waits == 0, "no wait ran out");
  return true;
}

}  // namespace timeout_test

int main() {
  if (!timeout_test::test_wait() || !timeout_test::test_marks() || timeout_test::g_failures > 0) return 1;
  std::printf("all timeout tests passed\n");
  return 0;
}
