// Argument blocks and launchers of the paged-cache operators (paged_cache.cu, paged_attention.cu,
// paged_attention_tc.cu) and of the packed-prompt attention (packed.cu, prefill.cu, prefill_wide.cu).
#pragma once

#include <stdint.h>

#include <cuda_runtime.h>

namespace omni {

constexpr int kFp8 = 2;   // cache element type codes beside kBF16 / kF32: e4m3 codes with a scale byte per vector,
constexpr int kInt4 = 3;  // 4-bit codes with a bf16 scale per 32 dims (int4.cuh)

// A cache of pages [pages, kv_heads, page, dim] (K and V share their strides, in elements; of 4-bit pages in bytes); scale bytes
// [pages, kv_heads, page], bf16 scales [pages, kv_heads, page, dim / 32], contiguous, or null.
struct PageCache {
  void* k;
  void* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t pages, s_page, s_head, s_pos;
  int page, kv_heads, dim;
  int type;  // kBF16, kF32, kFp8 or kInt4
};

struct PagedRopeArgs {
  const void* qkv;
  int64_t qkv_stride;
  const float* cs;
  int64_t cs_positions;
  const int64_t* pos;
  const int64_t* slots;
  void* q_out;
  PageCache c;
  int n, heads;
  const void* q_norm;  // [dim] weights of the norms (paged_norm_rope_kv alone)
  const void* k_norm;
  float eps;
  int* status;
};
cudaError_t launch_paged_rope_kv(int dtype, const PagedRopeArgs& a, cudaStream_t stream);
cudaError_t launch_paged_norm_rope_kv(int dtype, const PagedRopeArgs& a, cudaStream_t stream);

struct PagedReadArgs {
  PageCache c;
  const int32_t* table;
  int64_t table_stride;
  int table_width, rows;
  const int64_t* offsets;
  int64_t tokens;
  void* k_out;
  void* v_out;
  int* status;
};
cudaError_t launch_paged_kv_read(int dtype, const PagedReadArgs& a, cudaStream_t stream);

struct PagedAttnArgs {
  const void* q;
  PageCache c;
  const int32_t* table;
  int64_t table_stride;
  int table_width;
  const int64_t* lengths;
  void* out;
  int rows, tokens, heads;
  float scale;
  void* workspace;
  int* status;
};
// Query columns of one unit (row, kv head) are its tokens * heads / kv_heads query vectors, cut into chunks.
size_t paged_attention_workspace(int dtype, int type, int rows, int tokens, int heads, int kv_heads, int dim, int page,
                                 int table_width);
cudaError_t launch_paged_attention(int dtype, const PagedAttnArgs& a, cudaStream_t stream);
// The tensor-core pass (paged_attention_tc.cu); cudaErrorNotSupported where the pages' strides have no tensor map or the
// call has 2^31 key tiles and more.
bool paged_tc_supported(int dtype, int type, int dim, int page);
size_t paged_tc_workspace(int dim);
cudaError_t launch_paged_attention_tc(const PagedAttnArgs& a, cudaStream_t stream);

// The pass over 4-bit pages (paged_attention_int4.cu): bf16 queries, head_dim from 64, every page size.
bool paged_int4_supported(int dtype, int type, int dim);
size_t paged_int4_workspace(int dim);
cudaError_t launch_paged_attention_int4(const PagedAttnArgs& a, cudaStream_t stream);

struct PackedArgs {
  const void* q;
  int64_t q_st, q_sh;  // q[token, head, :] strides (elements)
  const void* k;
  int64_t k_st, k_sh;
  const void* v;
  int64_t v_st, v_sh;
  void* out;  // [tokens, heads, dim] contiguous
  const int64_t* q_offsets;
  const int64_t* k_offsets;
  int64_t q_tokens, k_tokens;
  int seqs, heads, kv_heads, dim;
  float scale;
  unsigned* counters;  // zero on entry, left zero (tensor-core kernels)
  int* status;
};
// Tensor-core kernels, bf16 head_dim 64 and 128 (prefill.cu), 256 and 512 (prefill_wide.cu), at most 128 query heads per kv head;
// cudaErrorNotSupported where a tensor's strides have no tensor map.
size_t packed_workspace(int dtype, int64_t q_tokens, int heads, int kv_heads, int dim);
cudaError_t launch_packed_tc(const PackedArgs& a, cudaStream_t stream);
cudaError_t launch_packed_tc_wide(const PackedArgs& a, cudaStream_t stream);
// What the parts of the CUDA-core kernel's calls take (packed.cu).
size_t packed_parts_bytes(int dtype, int64_t q_tokens, int heads, int kv_heads, int dim);
cudaError_t launch_packed(int dtype, const PackedArgs& a, cudaStream_t stream);

}  // namespace omni
