// C entry points of the attentions with several queries per sequence: argument
// checks, workspace size and the choice of kernel.
#include <algorithm>

#include "multi_query.cuh"

using namespace i4kv;

namespace i4kv {
double multi_query_f32_units(const MultiQueryArgs& a, int dim);
double multi_query_tc_units(const MultiQueryArgs& a, int dim);
size_t multi_query_f32_workspace(int dim, int sms);
cudaError_t multi_query_f32(const MultiQueryArgs& a, int dim, int vk, int sms, void* ws, size_t ws_bytes,
                            cudaStream_t stream);
size_t multi_query_tc_workspace(int dim, long long rows, int sms);
cudaError_t multi_query_tc(const MultiQueryArgs& a, int dim, int sms, void* ws, size_t ws_bytes, cudaStream_t stream);
}  // namespace i4kv

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool is_kind(int k) { return k == INT4KV_VALUES_F32 || k == INT4KV_VALUES_F16 || k == INT4KV_VALUES_BF16; }

cudaError_t sm_count(int* sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  return cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev);
}

// The sizes shared by both entry points.
bool sizes_ok(int batch, int hq, int hkv, int dim, int page, int group, int max_pages, int num_pages,
              int max_drafts) {
  if (batch <= 0 || batch > 65535 || hkv <= 0 || hq < hkv || hq % hkv != 0) return false;
  if (dim != 64 && dim != 128 && dim != 256) return false;
  if (page != kMqPage || group <= 0 || group % kMqPage != 0) return false;
  if (max_pages <= 0 || num_pages <= 0 || (long long)max_pages * kMqPage > 0x7fffffffll - 1024) return false;
  return max_drafts >= 0 && max_drafts <= INT4KV_MAX_DRAFTS && (long long)hq * dim <= (1 << 24);
}

cudaError_t run(const MultiQueryArgs& a, int dim, int vk, void* workspace, size_t bytes, cudaStream_t stream) {
  if (!aligned16(workspace) || !workspace) return cudaErrorInvalidValue;
  int sms = 0;
  if ((long long)a.total_rows * a.kv_heads * a.group_q > 0x7fffffffll) return cudaErrorInvalidValue;
  if ((a.qk != INT4KV_VALUES_F32 ? multi_query_tc_units(a, dim) : multi_query_f32_units(a, dim)) > kMqMostUnits)
    return cudaErrorInvalidValue;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  if (a.qk != INT4KV_VALUES_F32) return multi_query_tc(a, dim, sms, workspace, bytes, stream);
  return multi_query_f32(a, dim, vk, sms, workspace, bytes, stream);
}

}  // namespace

extern "C" {

cudaError_t int4kv_paged_attention_workspace_size(int batch, int num_q_heads, int num_kv_heads,
                                                  int head_dim, int max_drafts, size_t* bytes) {
  if (!bytes || !sizes_ok(batch, num_q_heads, num_kv_heads, head_dim, kMqPage, kMqPage, 1, 1, max_drafts))
    return cudaErrorInvalidValue;
  int sms = 0;
  const cudaError_t e = sm_count(&sms);
  if (e != cudaSuccess) return e;
  const long long rows = (long long)std::max(1, max_drafts) * (num_q_heads / num_kv_heads);
  *bytes = std::max(multi_query_f32_workspace(head_dim, sms), multi_query_tc_workspace(head_dim, rows, sms));
  return cudaSuccess;
}

cudaError_t int4kv_paged_tree_decode(const void* query, const void* k_draft, const void* v_draft,
                                     int qkv_dtype, const int64_t* tree_mask,
                                     const int32_t* draft_offsets, int num_rows, int max_drafts,
                                     const uint8_t* k_pool, const void* v_pool, int value_dtype,
                                     const float* sz_pool, const int32_t* block_table,
                                     const int32_t* seq_lens, int batch, int num_q_heads,
                                     int num_kv_heads, int head_dim, int page_tokens,
                                     int group_tokens, int max_pages, int num_pages, int window,
                                     int sinks, void* out, void* workspace, size_t workspace_bytes,
                                     uint32_t* status, cudaStream_t stream) {
  if (!sizes_ok(batch, num_q_heads, num_kv_heads, head_dim, page_tokens, group_tokens, max_pages,
                num_pages, max_drafts) || num_rows < 0 || window < 0 || sinks < 0)
    return cudaErrorInvalidValue;
  if (!is_kind(qkv_dtype) || !is_kind(value_dtype)) return cudaErrorInvalidValue;
  if (qkv_dtype != INT4KV_VALUES_F32 && value_dtype != qkv_dtype) return cudaErrorInvalidValue;
  if (!draft_offsets || !k_pool || !v_pool || !sz_pool || !block_table || !seq_lens)
    return cudaErrorInvalidValue;
  if (num_rows == 0 || max_drafts == 0) return cudaSuccess;
  if (!query || !k_draft || !v_draft || !tree_mask || !out) return cudaErrorInvalidValue;
  for (const void* p : {query, k_draft, v_draft, (const void*)k_pool, v_pool, (const void*)sz_pool, (const void*)out})
    if (!aligned16(p)) return cudaErrorInvalidValue;
  MultiQueryArgs a{query, k_draft, v_draft, tree_mask, draft_offsets, k_pool, v_pool, sz_pool,
                   block_table, seq_lens, out, nullptr, nullptr, status, qkv_dtype, batch, num_kv_heads,
                   num_q_heads / num_kv_heads, num_rows, max_drafts, max_pages, num_pages,
                   group_tokens / kMqPage, window, sinks};
  return run(a, head_dim, value_dtype, workspace, workspace_bytes, stream);
}

cudaError_t int4kv_paged_window_decode(const void* query, int query_dtype, const uint8_t* k_pool,
                                       const void* v_pool, int value_dtype, const float* sz_pool,
                                       const int32_t* block_table, const int32_t* seq_lens,
                                       int batch, int num_q_heads, int num_kv_heads, int head_dim,
                                       int page_tokens, int group_tokens, int max_pages,
                                       int num_pages, int window, int sinks, void* out,
                                       void* workspace, size_t workspace_bytes, uint32_t* status,
                                       cudaStream_t stream) {
  if (!sizes_ok(batch, num_q_heads, num_kv_heads, head_dim, page_tokens, group_tokens, max_pages,
                num_pages, 1) || window <= 0 || sinks < 0)
    return cudaErrorInvalidValue;
  if (!is_kind(query_dtype) || !is_kind(value_dtype)) return cudaErrorInvalidValue;
  if (query_dtype != INT4KV_VALUES_F32 && value_dtype != query_dtype) return cudaErrorInvalidValue;
  if (!query || !k_pool || !v_pool || !sz_pool || !block_table || !seq_lens || !out)
    return cudaErrorInvalidValue;
  for (const void* p : {query, (const void*)k_pool, v_pool, (const void*)sz_pool, (const void*)out})
    if (!aligned16(p)) return cudaErrorInvalidValue;
  MultiQueryArgs a{query, nullptr, nullptr, nullptr, nullptr, k_pool, v_pool, sz_pool,
                   block_table, seq_lens, out, nullptr, nullptr, status, query_dtype, batch, num_kv_heads,
                   num_q_heads / num_kv_heads, batch, 1, max_pages, num_pages,
                   group_tokens / kMqPage, window, sinks};
  return run(a, head_dim, value_dtype, workspace, workspace_bytes, stream);
}

}  // extern "C"
