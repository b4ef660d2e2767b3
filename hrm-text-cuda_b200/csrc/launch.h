// Host-side launchers of the sm_100a layer-op kernels (called by abi.cu after
// argument validation; they assume valid, non-empty arguments).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace hrm {

// SM count of the current device, queried once per device and cached.
int device_sm_count();

// True when p is 16-byte aligned (a uint4 access is legal).
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Warps per CTA of a one-warp-per-row launch over `rows` rows: max_warps, or
// fewer when there are fewer than max_warps rows per SM, so that a small
// (decode-size) launch spreads over as many SMs as it has rows instead of
// rows / max_warps of them.
inline int warps_per_cta(int64_t rows, int max_warps) {
  const int64_t per_sm = rows / device_sm_count();
  if (per_sm >= max_warps) return max_warps;
  return per_sm < 1 ? 1 : (int)per_sm;
}

// Programmatic dependent launches (1) or plain stream-ordered ones (0).
#ifndef HRM_PDL
#define HRM_PDL 1
#endif

// Launches kernel k as grid x block threads with smem dynamic shared bytes on
// stream s.  The launch is programmatic (cudaLaunchAttributeProgrammatic-
// StreamSerialization): it may start before the previous kernel in s has
// finished, which is safe because every kernel of this library waits for that
// kernel at its entry (grid_dependency_begin).  Returns the launch's own
// status, so an error left pending by an earlier, unrelated call is neither
// reported as this launch's nor cleared.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_kernel(void (*k)(KArgs...), int64_t grid, int block, size_t smem, cudaStream_t s,
                                 Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = HRM_PDL ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, k, static_cast<Args&&>(args)...);
}

// The same for thread-block clusters of `cluster` CTAs (grid a multiple of it).
template <typename... KArgs, typename... Args>
inline cudaError_t launch_cluster(void (*k)(KArgs...), int64_t grid, int block, size_t smem, int cluster,
                                  cudaStream_t s, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)cluster, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = HRM_PDL ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k, static_cast<Args&&>(args)...);
}

// Lets kernel K be launched with `bytes` of dynamic shared memory on the current
// device (needed above 48 KB).  The driver call is made once per kernel and device:
// a call costs the host about as much as a launch's own bookkeeping.
template <auto K>
inline cudaError_t allow_shared(size_t bytes) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// For a kernel whose warpgroups share its registers out again: whether it was built
// with `regs` per thread.  With fewer the taking would wait for good.
template <auto K>
inline cudaError_t has_registers(int regs) {
  static std::atomic<int> built{0};
  int n = built.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaFuncAttributes attr;
    const cudaError_t e = cudaFuncGetAttributes(&attr, K);
    if (e != cudaSuccess) return e;
    built.store(n = attr.numRegs, std::memory_order_relaxed);
  }
  return n >= regs ? cudaSuccess : cudaErrorInvalidConfiguration;
}

cudaError_t launch_additive_inject(const void* a, const void* b, void* out, int64_t n, cudaStream_t s);
cudaError_t launch_attn_gate(const void* gate, const void* attn, void* out, int64_t n, cudaStream_t s);
cudaError_t launch_broadcast(void* dst, const void* src, int64_t n_copies, int64_t vec_len, cudaStream_t s);
cudaError_t launch_swiglu(const void* gate, const void* up, void* out, int64_t n, cudaStream_t s);

cudaError_t launch_rms_norm_bf16(const void* x, void* y, const void* w, int64_t rows, int64_t hidden,
                                 float eps, cudaStream_t s);
cudaError_t launch_rms_norm_f32(const float* x, float* y, const float* w, int64_t rows, int64_t hidden,
                                float eps, cudaStream_t s);
cudaError_t launch_add_rms_norm(const void* x, const void* b, void* r, void* y, const void* w, int64_t rows,
                                int64_t hidden, float eps, cudaStream_t s);
cudaError_t launch_embed_rms_norm(const uint32_t* ids, const void* table, void* h, void* y, const void* w,
                                  int64_t rows, int64_t hidden, int64_t vocab, float scale, float eps,
                                  cudaStream_t s);
cudaError_t launch_embedding(const uint32_t* ids, const void* table, void* out, int64_t tokens, int64_t hidden,
                             int64_t vocab, float scale, cudaStream_t s);

cudaError_t launch_rope(void* q, void* k, int64_t batch, int64_t heads, int64_t seq, int64_t head_dim,
                        int64_t offset, float theta, const float* table, bool token_major, cudaStream_t s);
cudaError_t launch_split_rope(const void* gqkv, void* gate, void* q, void* k, void* v, void* kc, void* vc,
                              int64_t batch, int64_t heads, int64_t seq, int64_t head_dim, int64_t offset,
                              float theta, const float* table, int64_t cache_len, int64_t cache_offset,
                              cudaStream_t s);
cudaError_t launch_rope_table(float* table, int64_t max_pos, int64_t head_dim, float theta, cudaStream_t s);

cudaError_t launch_convert_to_bf16(const void* src, int dtype, void* dst, int64_t n, cudaStream_t s);

struct Kv4View;
struct AttnArgs;
cudaError_t launch_split_rope_kv4(const void* gqkv, void* gate, void* q, void* k, void* v, const Kv4View& c,
                                  int64_t batch, int64_t heads, int64_t seq, int64_t head_dim,
                                  int64_t position_offset, const int* position_offsets, float theta,
                                  const float* table, int64_t table_positions, int64_t cache_offset,
                                  const int* cache_offsets, cudaStream_t s);
cudaError_t launch_kv4_update(const void* k, const void* v, const Kv4View& c, int64_t batch, int64_t heads,
                              int64_t seq, int64_t head_dim, int64_t position_offset, const int* position_offsets,
                              int64_t cache_offset, const int* cache_offsets, cudaStream_t s);
// `longest`: no sequence has more cache rows than this; `parts`: kv4_decode_workspace
// bytes for the same sizes.
int64_t kv4_decode_workspace(int64_t rows, int64_t head_dim, int64_t longest);
cudaError_t launch_kv4_decode(const AttnArgs& a, int64_t head_dim, int64_t longest, float* parts, cudaStream_t s);
int64_t kv4_prefill_workspace(int64_t batch_kv_heads, int64_t rows, int64_t head_dim);
cudaError_t launch_kv4_prefill(const AttnArgs& a, int64_t head_dim, int64_t longest, float* parts, cudaStream_t s);
cudaError_t kv4_prefill_wait_timeouts(unsigned int* count, bool reset);
cudaError_t launch_kv4_add_weights(const AttnArgs& a, int64_t longest, cudaStream_t s);
cudaError_t launch_kv4_weights(const AttnArgs& a, int64_t head_dim, int64_t longest, cudaStream_t s);
// Whether the selection of `budget` out of at most n rows fits its shared memory.
bool kv4_evict_fits(int64_t n, int64_t budget);
cudaError_t launch_kv4_evict(const Kv4View& from, const Kv4View& to, bool in_place, int64_t batch, int64_t kv_heads,
                             int64_t head_dim, int64_t length, const int* lengths, int64_t budget,
                             int64_t protect_from, const int* protect_froms, int* new_lengths, cudaStream_t s);

// Bounded waits that ran out in the row kernels (device counter); reset sets it to 0.
cudaError_t rownorm_wait_timeouts(unsigned int* count, bool reset);

}  // namespace hrm
