// extern "C" entry points of the 4-bit KV cache: argument checks, then the
// launchers.  Every check runs before anything is queued.
#include <climits>
#include <cmath>

#include "../../include/hrm_ops.h"
#include "abi_checks.h"
#include "kv4_mma.cuh"
#include "launch.h"

namespace {

struct Buffer {
  const void* p;
  int64_t bytes;
  bool written;
};

// HRM_ERR_ALIASING when a written buffer shares a byte with another.
template <int N>
int check_overlaps(const Buffer (&b)[N]) {
  for (int x = 0; x < N; ++x)
    for (int y = x + 1; y < N; ++y)
      if ((b[x].written || b[y].written) && overlap(b[x].p, b[x].bytes, b[y].p, b[y].bytes)) return HRM_ERR_ALIASING;
  return HRM_OK;
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The cache's sizes, checked; `rows` = batch * kv_heads * cache_len.
struct CacheBytes {
  int64_t rows, codes, scales, words;
};

int check_cache_shape(const hrm_kv4_cache* c, CacheBytes* n) {
  if (!c) return HRM_ERR_NULL_POINTER;
  if (c->batch < 0 || c->kv_heads <= 0 || c->cache_len < 0 || c->kv_heads > INT32_MAX) return HRM_ERR_INVALID_SHAPE;
  if (c->head_dim <= 0 || c->head_dim > 256 || c->head_dim % 64 != 0) return HRM_ERR_INVALID_SHAPE;
  if (c->cache_len > INT32_MAX - 4096) return HRM_ERR_SIZE_OVERFLOW;
  n->rows = mul_checked(mul_checked(c->batch, c->kv_heads), c->cache_len);
  if (n->rows < 0 || mul_checked(n->rows, c->head_dim) < 0) return HRM_ERR_SIZE_OVERFLOW;
  n->codes = n->rows * (c->head_dim / 2);
  n->scales = n->rows * (c->head_dim / hrm::kKv4Group * 4);
  n->words = n->rows * 4;
  return HRM_OK;
}

int check_cache_pointers(const hrm_kv4_cache* c) {
  if (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales) return HRM_ERR_NULL_POINTER;
  if (!aligned(c->k_codes, 16) || !aligned(c->k_scales, 16) || !aligned(c->v_codes, 16) || !aligned(c->v_scales, 16) ||
      !aligned(c->weights, 4) || !aligned(c->positions, 4))
    return HRM_ERR_ALIGNMENT;
  return HRM_OK;
}

hrm::Kv4View view(const hrm_kv4_cache* c) {
  return {static_cast<uint8_t*>(c->k_codes), static_cast<uint32_t*>(c->k_scales), static_cast<uint8_t*>(c->v_codes),
          static_cast<uint32_t*>(c->v_scales), c->weights, c->positions, c->cache_len};
}

// seq_len new rows at position_offset / cache_offset (ignored where per-sequence arrays are given).
int check_places(const hrm_kv4_cache* c, int64_t seq_len, int64_t position_offset, const int32_t* position_offsets,
                 int64_t cache_offset, const int32_t* cache_offsets) {
  if (seq_len < 0) return HRM_ERR_INVALID_SHAPE;
  if (seq_len > INT32_MAX) return HRM_ERR_SIZE_OVERFLOW;
  if (!position_offsets) {
    if (position_offset < 0) return HRM_ERR_INVALID_SHAPE;
    if (position_offset > INT32_MAX - seq_len) return HRM_ERR_SIZE_OVERFLOW;
  }
  if (!cache_offsets && (cache_offset < 0 || seq_len > c->cache_len || cache_offset > c->cache_len - seq_len))
    return HRM_ERR_INVALID_SHAPE;
  if (!aligned(position_offsets, 4) || !aligned(cache_offsets, 4)) return HRM_ERR_ALIGNMENT;
  return HRM_OK;
}

// Query rows of one kv head; which attention kernel serves them.
int64_t attn_rows(const hrm_kv4_cache* c, int64_t num_heads, int64_t seq_len) {
  return num_heads / c->kv_heads * seq_len;
}

// Bytes of workspace: the scores and the rows' sums that accumulate needs, then
// the partial results of a split decode.
struct AttnBytes {
  int64_t scores, sums, parts;
};

int check_attention_shape(const hrm_kv4_cache* c, int64_t num_heads, int64_t seq_len, int accumulate, AttnBytes* n) {
  if (num_heads <= 0 || seq_len < 0 || num_heads > INT32_MAX || num_heads % c->kv_heads != 0)
    return HRM_ERR_INVALID_SHAPE;
  if (seq_len > INT32_MAX) return HRM_ERR_SIZE_OVERFLOW;
  const int64_t rows = attn_rows(c, num_heads, seq_len), heads = c->batch * c->kv_heads;
  const int64_t all = mul_checked(heads, rows);
  if (all < 0 || all + 7 * heads > INT32_MAX || mul_checked(all, c->head_dim * 2) < 0) return HRM_ERR_SIZE_OVERFLOW;
  const int64_t tiles = c->cache_len / 64 + 1;  // of a head; (rows + 7) / 8 blocks of queries walk them
  const int64_t walks = mul_checked(mul_checked(heads, (rows + 7) / 8), tiles);
  if (walks < 0 || walks > INT32_MAX) return HRM_ERR_SIZE_OVERFLOW;
  const int64_t scores = mul_checked(mul_checked(all, c->cache_len), 4);
  const bool keeps = accumulate && rows <= hrm::kScoreRows;
  if (keeps && (scores < 0 || scores > INT64_MAX / 2)) return HRM_ERR_SIZE_OVERFLOW;
  n->scores = keeps ? (scores + 15) / 16 * 16 : 0;
  n->sums = accumulate && rows > hrm::kDecodeRows ? (all * 4 + 15) / 16 * 16 : 0;
  n->parts = rows <= hrm::kChunkRows ? hrm::kv4_decode_workspace(rows, c->head_dim, c->cache_len)
                                       : hrm::kv4_prefill_workspace(heads, rows, c->head_dim);
  return HRM_OK;
}

}  // namespace

extern "C" {

int hrm_kv4_update(const hrm_kv4_cache* cache, const void* k, const void* v, int64_t seq_len, int64_t position_offset,
                   const int32_t* position_offsets, int64_t cache_offset, const int32_t* cache_offsets,
                   hrm_stream_t stream) {
  CacheBytes n;
  int e = check_cache_shape(cache, &n);
  if (e != HRM_OK) return e;
  e = check_places(cache, seq_len, position_offset, position_offsets, cache_offset, cache_offsets);
  if (e != HRM_OK) return e;
  if (cache->batch == 0 || seq_len == 0 || cache->cache_len == 0) return HRM_OK;
  if (!k || !v) return HRM_ERR_NULL_POINTER;
  e = check_cache_pointers(cache);
  if (e != HRM_OK) return e;
  if (!aligned(k, 16) || !aligned(v, 16)) return HRM_ERR_ALIGNMENT;
  const int64_t elements = mul_checked(mul_checked(cache->batch * cache->kv_heads, seq_len), cache->head_dim);
  if (elements < 0 || elements / 8 / 128 >= INT32_MAX) return HRM_ERR_SIZE_OVERFLOW;
  const Buffer b[] = {{cache->k_codes, n.codes, true}, {cache->k_scales, n.scales, true},
                      {cache->v_codes, n.codes, true}, {cache->v_scales, n.scales, true},
                      {cache->weights, n.words, true}, {cache->positions, n.words, true},
                      {k, elements * 2, false},        {v, elements * 2, false},
                      {position_offsets, cache->batch * 4, false}, {cache_offsets, cache->batch * 4, false}};
  e = check_overlaps(b);
  if (e != HRM_OK) return e;
  return cuda_status(hrm::launch_kv4_update(k, v, view(cache), cache->batch, cache->kv_heads, seq_len, cache->head_dim,
                                            position_offset, position_offsets, cache_offset, cache_offsets,
                                            as_cuda(stream)));
}

int hrm_split_gqkv_rope_kv4(const void* gqkv, void* gate_out, void* q_out, void* k_out, void* v_out,
                            const hrm_kv4_cache* cache, int64_t seq_len, int64_t position_offset,
                            const int32_t* position_offsets, float theta, const float* rope_table,
                            int64_t table_positions, int64_t cache_offset, const int32_t* cache_offsets,
                            hrm_stream_t stream) {
  CacheBytes n;
  int e = check_cache_shape(cache, &n);
  if (e != HRM_OK) return e;
  e = check_places(cache, seq_len, position_offset, position_offsets, cache_offset, cache_offsets);
  if (e != HRM_OK) return e;
  if ((k_out == nullptr) != (v_out == nullptr)) return HRM_ERR_NULL_POINTER;
  if (cache->batch == 0 || seq_len == 0) return HRM_OK;
  if (!gqkv || !gate_out || !q_out) return HRM_ERR_NULL_POINTER;
  if (cache->cache_len > 0) {
    e = check_cache_pointers(cache);
    if (e != HRM_OK) return e;
  }
  if (!aligned(gqkv, 16) || !aligned(gate_out, 16) || !aligned(q_out, 16) || !aligned(k_out, 16) ||
      !aligned(v_out, 16) || !aligned(rope_table, 16))
    return HRM_ERR_ALIGNMENT;
  const int64_t tokens = mul_checked(cache->batch, seq_len);
  const int64_t bytes = mul_checked(mul_checked(tokens, cache->kv_heads), cache->head_dim * 2);
  if (bytes < 0 || mul_checked(bytes, 4) < 0 || tokens > INT32_MAX) return HRM_ERR_SIZE_OVERFLOW;
  int64_t tbytes = 0;
  if (rope_table != nullptr) {
    if (!position_offsets && table_positions < position_offset + seq_len) return HRM_ERR_TABLE_RANGE;
    tbytes = mul_checked(mul_checked(table_positions, cache->head_dim), 4);
    if (tbytes < 0) return HRM_ERR_SIZE_OVERFLOW;
  }
  const Buffer b[] = {{cache->k_codes, n.codes, true}, {cache->k_scales, n.scales, true},
                      {cache->v_codes, n.codes, true}, {cache->v_scales, n.scales, true},
                      {cache->weights, n.words, true}, {cache->positions, n.words, true},
                      {gate_out, bytes, true},         {q_out, bytes, true},
                      {k_out, bytes, true},            {v_out, bytes, true},
                      {gqkv, bytes * 4, false},        {rope_table, tbytes, false},
                      {position_offsets, cache->batch * 4, false}, {cache_offsets, cache->batch * 4, false}};
  e = check_overlaps(b);
  if (e != HRM_OK) return e;
  return cuda_status(hrm::launch_split_rope_kv4(gqkv, gate_out, q_out, k_out, v_out, view(cache), cache->batch,
                                                cache->kv_heads, seq_len, cache->head_dim, position_offset,
                                                position_offsets, theta, rope_table, table_positions, cache_offset,
                                                cache_offsets, as_cuda(stream)));
}

int hrm_kv4_attention_workspace(const hrm_kv4_cache* cache, int64_t num_heads, int64_t seq_len, int accumulate,
                                int64_t* bytes) {
  if (!bytes) return HRM_ERR_NULL_POINTER;
  CacheBytes n;
  AttnBytes w{};
  int e = check_cache_shape(cache, &n);
  if (e == HRM_OK) e = check_attention_shape(cache, num_heads, seq_len, accumulate, &w);
  if (e == HRM_OK) *bytes = w.scores + w.sums + w.parts;
  return e;
}

int hrm_kv4_attention(const void* q, const hrm_kv4_cache* cache, const void* gate, void* out, int64_t num_heads,
                      int64_t seq_len, int64_t cache_offset, const int32_t* cache_offsets, int64_t prefix_len,
                      float softmax_scale, int accumulate, void* workspace, int64_t workspace_bytes,
                      hrm_stream_t stream) {
  CacheBytes n;
  int e = check_cache_shape(cache, &n);
  if (e != HRM_OK) return e;
  AttnBytes w{};
  e = check_attention_shape(cache, num_heads, seq_len, accumulate, &w);
  if (e != HRM_OK) return e;
  e = check_places(cache, seq_len, 0, nullptr, cache_offset, cache_offsets);
  if (e != HRM_OK) return e;
  if (prefix_len < 0 || !std::isfinite(softmax_scale) || workspace_bytes < 0) return HRM_ERR_INVALID_SHAPE;
  if (cache->batch == 0 || seq_len == 0) return HRM_OK;
  if (!q || !out) return HRM_ERR_NULL_POINTER;
  if (cache->cache_len > 0) {
    e = check_cache_pointers(cache);
    if (e != HRM_OK) return e;
    if (accumulate && !cache->weights) return HRM_ERR_NULL_POINTER;
  } else {
    accumulate = 0;  // no row to add to
    w.scores = w.sums = 0;
  }
  const int64_t need = w.scores + w.sums + w.parts;
  if (need > 0 && !workspace) return HRM_ERR_NULL_POINTER;
  if (need > 0 && workspace_bytes < need) return HRM_ERR_SCRATCH_LIMIT;
  if (!aligned(q, 16) || !aligned(out, 16) || !aligned(gate, 16) || (need > 0 && !aligned(workspace, 16)))
    return HRM_ERR_ALIGNMENT;
  const int64_t bytes = cache->batch * num_heads * seq_len * cache->head_dim * 2;
  const Buffer b[] = {{out, bytes, true},
                      {need > 0 ? workspace : nullptr, need, true},
                      {accumulate ? cache->weights : nullptr, n.words, true},
                      {q, bytes, false},
                      {gate, bytes, false},
                      {cache->k_codes, n.codes, false},
                      {cache->k_scales, n.scales, false},
                      {cache->v_codes, n.codes, false},
                      {cache->v_scales, n.scales, false},
                      {cache_offsets, cache->batch * 4, false}};
  e = check_overlaps(b);
  if (e != HRM_OK) return e;

  hrm::AttnArgs a{};
  a.q = static_cast<const uint4*>(q);
  a.gate = static_cast<const uint16_t*>(gate);
  a.out = static_cast<uint16_t*>(out);
  a.c = view(cache);
  a.batch = cache->batch;
  a.heads = (int)num_heads;
  a.kv_heads = (int)cache->kv_heads;
  a.group = (int)(num_heads / cache->kv_heads);
  a.seq = (int)seq_len;
  a.cache_offset = cache_offset;
  a.cache_offsets = cache_offsets;
  a.prefix_len = prefix_len;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  const int64_t rows = (int64_t)a.group * seq_len;
  char* const space = static_cast<char*>(workspace);
  if (w.scores > 0) a.scores = reinterpret_cast<float*>(space);
  if (w.sums > 0) a.lse = reinterpret_cast<float*>(space + w.scores);
  const int64_t longest = cache_offsets ? cache->cache_len : cache_offset + seq_len;
  float* parts = reinterpret_cast<float*>(space + w.scores + w.sums);
  const cudaStream_t s = as_cuda(stream);
  cudaError_t ce = rows <= hrm::kChunkRows ? hrm::launch_kv4_decode(a, cache->head_dim, longest, parts, s)
                                           : hrm::launch_kv4_prefill(a, cache->head_dim, longest, parts, s);
  if (ce == cudaSuccess && a.lse != nullptr)
    ce = a.scores != nullptr ? hrm::launch_kv4_add_weights(a, longest, s)
                             : hrm::launch_kv4_weights(a, cache->head_dim, longest, s);
  return cuda_status(ce);
}

int hrm_kv4_evict(const hrm_kv4_cache* cache, const hrm_kv4_cache* out, int64_t length, const int32_t* lengths,
                  int64_t budget, int64_t protect_from, const int32_t* protect_froms, int32_t* new_lengths,
                  hrm_stream_t stream) {
  CacheBytes n, m;
  int e = check_cache_shape(cache, &n);
  if (e != HRM_OK) return e;
  e = check_cache_shape(out, &m);
  if (e != HRM_OK) return e;
  const bool in_place = out->k_codes == cache->k_codes && out->v_codes == cache->v_codes &&
                        out->k_scales == cache->k_scales && out->v_scales == cache->v_scales &&
                        out->weights == cache->weights && out->positions == cache->positions;
  if (out->batch != cache->batch || out->kv_heads != cache->kv_heads || out->head_dim != cache->head_dim)
    return HRM_ERR_INVALID_SHAPE;
  if (in_place && out->cache_len != cache->cache_len) return HRM_ERR_INVALID_SHAPE;
  if (budget < 1 || (!lengths && (length < 0 || length > cache->cache_len))) return HRM_ERR_INVALID_SHAPE;
  const int64_t longest = lengths ? cache->cache_len : length;
  if ((budget < longest ? budget : longest) > out->cache_len) return HRM_ERR_INVALID_SHAPE;
  if (!aligned(lengths, 4) || !aligned(protect_froms, 4) || !aligned(new_lengths, 4)) return HRM_ERR_ALIGNMENT;
  if (cache->batch == 0) return HRM_OK;
  if (!new_lengths) return HRM_ERR_NULL_POINTER;
  if (longest > 0) {
    e = check_cache_pointers(cache);
    if (e != HRM_OK) return e;
    e = check_cache_pointers(out);
    if (e != HRM_OK) return e;
    if (!cache->weights || !cache->positions || !out->weights || !out->positions) return HRM_ERR_NULL_POINTER;
  }
  if (budget > longest) budget = longest > 0 ? longest : 1;  // nothing goes
  if (!hrm::kv4_evict_fits(longest, budget)) return HRM_ERR_SCRATCH_LIMIT;
  if (mul_checked(cache->batch * cache->kv_heads, 8) > INT32_MAX) return HRM_ERR_SIZE_OVERFLOW;
  const Buffer b[] = {{out->k_codes, m.codes, true},
                      {out->k_scales, m.scales, true},
                      {out->v_codes, m.codes, true},
                      {out->v_scales, m.scales, true},
                      {out->weights, m.words, true},
                      {out->positions, m.words, true},
                      {new_lengths, cache->batch * 4, true},
                      {lengths, cache->batch * 4, false},
                      {protect_froms, cache->batch * 4, false},
                      {in_place ? nullptr : cache->k_codes, n.codes, false},
                      {in_place ? nullptr : cache->k_scales, n.scales, false},
                      {in_place ? nullptr : cache->v_codes, n.codes, false},
                      {in_place ? nullptr : cache->v_scales, n.scales, false},
                      {in_place ? nullptr : cache->weights, n.words, false},
                      {in_place ? nullptr : cache->positions, n.words, false}};
  e = check_overlaps(b);
  if (e != HRM_OK) return e;
  return cuda_status(hrm::launch_kv4_evict(view(cache), view(out), in_place, cache->batch, cache->kv_heads,
                                           cache->head_dim, length, lengths, budget, protect_from, protect_froms,
                                           new_lengths, as_cuda(stream)));
}

}  // extern "C"
