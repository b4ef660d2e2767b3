// The C++ layer's workspace of kv4_attention: a captured call replays after later calls
// have outgrown the workspace of its capture, and leaves what was allocated since
// alone.  Needs a GPU; exits non-zero on a failure.
#include <cmath>
#include <cstdio>
#include <cstring>
#include <thread>
#include <vector>

#include "hrm_layer_ops.hpp"

using hrm::bf16;
using hrm::CudaSlice;
using hrm::HrmError;
using hrm::HrmLayerOps;

namespace {

constexpr size_t kHeads = 4, kDim = 64, kCache = 6000, kAt = 5000;

bool ok(cudaError_t e, const char* what) {
  if (e != cudaSuccess) std::printf("FAIL %s: %s\n", what, cudaGetErrorString(e));
  return e == cudaSuccess;
}

std::vector<bf16> noise(size_t n, uint32_t x) {
  std::vector<bf16> v(n);
  for (bf16& e : v) {
    x = x * 1664525u + 1013904223u;
    e = bf16::from_f32((float)(int32_t)x * (1.0f / 2147483648.0f));
  }
  return v;
}

template <class T>
std::vector<T> host(const HrmLayerOps& m, const CudaSlice<T>& s) {
  std::vector<T> v(s.len());
  cudaStreamSynchronize(m.cu_stream());
  cudaMemcpy(v.data(), s.device_ptr(), s.len() * sizeof(T), cudaMemcpyDeviceToHost);
  return v;
}

bool same(const std::vector<bf16>& a, const std::vector<bf16>& b) {
  return a.size() == b.size() && std::memcmp(a.data(), b.data(), a.size() * sizeof(bf16)) == 0;
}

bool run() {
  HrmLayerOps m(0);
  auto cache = m.alloc_kv4_cache(1, kHeads, kCache, kDim, true);
  const size_t rows = kHeads * kCache * kDim;
  m.kv4_update(cache, m.htod_copy_bf16(noise(rows, 1)), m.htod_copy_bf16(noise(rows, 2)), kCache, 0, 0);
  auto q = m.htod_copy_bf16(noise(kHeads * kDim, 3));
  auto out = m.alloc_zero_bf16(kHeads * kDim), want = m.alloc_zero_bf16(kHeads * kDim);
  // scores of one query and the partial results of a split cache
  m.kv4_attention(q, cache, nullptr, want, kHeads, 1, kAt, 0, 0.125f, true);
  const std::vector<bf16> expected = host(m, want);

  cudaGraph_t graph = nullptr;
  cudaGraphExec_t exec = nullptr;
  if (!ok(cudaStreamBeginCapture(m.cu_stream(), cudaStreamCaptureModeThreadLocal), "begin capture")) return false;
  m.kv4_attention(q, cache, nullptr, out, kHeads, 1, kAt, 0, 0.125f, true);
  if (!ok(cudaStreamEndCapture(m.cu_stream(), &graph), "end capture") ||
      !ok(cudaGraphInstantiate(&exec, graph, 0), "instantiate"))
    return false;

  // calls that need more, twice, and buffers of the first workspace's size made after them
  for (size_t s : {6, 16}) {
    auto big_q = m.htod_copy_bf16(noise(kHeads * s * kDim, 4));
    auto big_out = m.alloc_zero_bf16(kHeads * s * kDim);
    m.kv4_attention(big_q, cache, nullptr, big_out, kHeads, s, kAt, 0, 0.125f, true);
    host(m, big_out);
  }
  int64_t bytes = 0;
  hrm_kv4_cache sizes{};
  sizes.batch = 1;
  sizes.kv_heads = kHeads;
  sizes.cache_len = kCache;
  sizes.head_dim = kDim;
  if (hrm_kv4_attention_workspace(&sizes, kHeads, 1, 1, &bytes) != HRM_OK || bytes == 0) return false;
  std::vector<CudaSlice<bf16>> since;
  const std::vector<bf16> pattern = noise((size_t)bytes / 2, 9);
  for (int i = 0; i < 4; ++i) since.push_back(m.htod_copy_bf16(pattern));

  for (int i = 0; i < 3; ++i)
    if (!ok(cudaGraphLaunch(exec, m.cu_stream()), "replay") || !ok(cudaStreamSynchronize(m.cu_stream()), "replay"))
      return false;
  if (!same(host(m, out), expected)) {
    std::printf("FAIL the replayed output\n");
    return false;
  }
  for (const auto& s : since)
    if (!same(host(m, s), pattern)) {
      std::printf("FAIL a buffer made since the capture was written\n");
      return false;
    }
  // two host threads that make the workspace grow: one layer, one stream
  auto more = [&](size_t s, CudaSlice<bf16>* o, const CudaSlice<bf16>* x) {
    cudaSetDevice(0);
    for (int i = 0; i < 20; ++i) m.kv4_attention(*x, cache, nullptr, *o, kHeads, s + 1 + i % 4, kAt, 0, 0.125f);
  };
  auto x = m.htod_copy_bf16(noise(kHeads * 40 * kDim, 5));
  auto o1 = m.alloc_zero_bf16(kHeads * 40 * kDim), o2 = m.alloc_zero_bf16(kHeads * 40 * kDim);
  std::thread a(more, 8, &o1, &x), b(more, 30, &o2, &x);
  a.join();
  b.join();
  const bool fine = ok(cudaStreamSynchronize(m.cu_stream()), "two threads");
  cudaGraphExecDestroy(exec);
  cudaGraphDestroy(graph);
  return fine;
}

}  // namespace

int main() {
  try {
    if (!run()) return 1;
  } catch (const HrmError& e) {
    std::printf("FAIL HrmError: %s\n", e.what());
    return 1;
  }
  std::printf("all workspace tests passed\n");
  return 0;
}
