// Launch interface of the paged cache's kernels (paged_tables.hip,
// paged_attn.hip).  Not installed; the public surface is include/heatkv.h.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hkv {

constexpr int32_t kMaxRequests = 4096;  // the tables kernel keeps three prefix sums of them in LDS

struct PagedTablesArgs {
  int32_t* block_tables;  // [requests, table_width], row stride table_stride
  int64_t table_stride;
  const int32_t* lengths;     // [requests], rows held
  const int32_t* new_counts;  // [requests], tokens of this step; < 0: the request has ended
  int32_t* free_blocks;       // ring of ring_size
  const int32_t* free_range;  // first, count
  int32_t requests;
  int32_t table_width;
  int32_t ring_size;
  int32_t num_tokens;
  int32_t block_shift;
  int32_t window;  // 0: none
  int32_t sinks;
  int64_t* slot_map;      // [num_tokens]
  int32_t* query_starts;  // [requests + 1]
  int32_t* lengths_out;
  int32_t* range_out;
  int32_t* status;  // [3]: status, blocks popped, blocks pushed
};
hipError_t launch_paged_tables(const PagedTablesArgs& a, hipStream_t stream);

// Strides in elements; a cache row is head_dim contiguous elements of 2 bytes.
struct PagedCacheStrides {
  int64_t block;
  int64_t head;
  int64_t row;
};

struct PagedAppendArgs {
  const void* k;  // [tokens, kv_heads, head_dim]
  const void* v;
  int64_t k_token, k_head, v_token, v_head;  // strides in elements
  void* k_cache;
  void* v_cache;
  PagedCacheStrides ks, vs;
  const int64_t* slot_map;
  int64_t num_slots;  // blocks * block_size
  int32_t num_tokens;
  int32_t kv_heads;
  int32_t head_dim;
  int32_t block_shift;
};
hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t stream);

struct PagedAttnArgs {
  const void* q;  // [tokens, heads, head_dim]
  int64_t q_token, q_head;
  const void* k_cache;
  const void* v_cache;
  PagedCacheStrides ks, vs;
  const int32_t* block_tables;
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* query_starts;
  const int32_t* prefix_blocks;  // the shared prefix, or null
  int32_t prefix_len;            // its rows (0: none)
  void* out;                     // [tokens, heads * head_dim]
  float* lse;                    // [heads, tokens] or null
  int32_t num_tokens;
  int32_t requests;
  int32_t table_width;
  int32_t num_blocks;
  int32_t heads;
  int32_t kv_heads;
  int32_t group;  // heads / kv_heads
  int32_t head_dim;
  int32_t block_shift;
  int32_t window;  // 0: none
  int32_t sinks;
  int32_t causal;
  int32_t dtype;     // Dtype: kF16 or kBF16
  int32_t fill_tail; // write zeros (lse -inf) for tokens behind the last request
  float softmax_scale;
  void* workspace;
  int64_t workspace_bytes;
  int32_t* counters;  // zeroed kPagedCounterBytes that every launch leaves zero, or null
};
constexpr int64_t kPagedCounterBytes = 64 * 1024;
hipError_t launch_paged_attention(const PagedAttnArgs& a, hipStream_t stream);
int64_t paged_attention_workspace(int32_t tokens, int32_t requests, int32_t heads, int32_t kv_heads, int32_t head_dim,
                                  int64_t table_rows, int32_t prefix_len, int32_t window, int32_t sinks, bool causal);

}  // namespace hkv
