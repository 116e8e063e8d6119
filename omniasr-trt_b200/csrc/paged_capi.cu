// extern "C" entry points of the paged-cache operators and the packed-prompt attention: argument checks and launches.

#include <stdarg.h>
#include <stdio.h>

#include "attention.cuh"
#include "omniasr_b200.h"
#include "paged.cuh"

namespace omni {
int set_last_error(int code, const char* message);
}

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return omni::set_last_error(code, buf);
}

int done(const char* name, cudaError_t e) {
  if (e != cudaSuccess) return fail(OMNIASR_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
  return omni::set_last_error(OMNIASR_OK, "");
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
int esize(int type) { return type == OMNIASR_F32 ? 4 : type == OMNIASR_BF16 ? 2 : 1; }
bool stride_ok(int64_t stride, int type) { return stride >= 0 && stride * esize(type) % 16 == 0; }

// dtype, head_dim and head counts; `type`: the cache's element type (dtype itself, or fp8).
int check(const char* name, int dtype, int type, int dim, int heads, int kv_heads) {
  if (dtype != OMNIASR_BF16 && dtype != OMNIASR_F32) return fail(OMNIASR_ERR_UNSUPPORTED, "%s: dtype %d", name, dtype);
  if (type != dtype && type != OMNIASR_FP8)
    return fail(OMNIASR_ERR_UNSUPPORTED, "%s: cache type %d with dtype %d (the same, or fp8)", name, type, dtype);
  if (!omni::dim_supported(dtype, dim))
    return fail(OMNIASR_ERR_UNSUPPORTED, "%s: head_dim %d (supported: 16, 32, 64, 128, 256, 512)", name, dim);
  if (kv_heads <= 0 || heads <= 0 || heads > 65535 || heads % kv_heads)
    return fail(OMNIASR_ERR_ARGUMENT, "%s: heads %d, kv_heads %d (a multiple, at most 65535)", name, heads, kv_heads);
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(OMNIASR_ERR_DEVICE, "no CUDA device");
  if (!omniasr_device_supported(dev))
    return fail(OMNIASR_ERR_DEVICE, "device %d is not compute capability 10.0 (sm_100a code)", dev);
  return OMNIASR_OK;
}

int check_pages(const char* name, const omni::PageCache& c) {
  if (!c.k || !c.v || !aligned16(c.k) || !aligned16(c.v))
    return fail(OMNIASR_ERR_ARGUMENT, "%s: page pointers must be 16-byte aligned", name);
  if (c.pages <= 0 || c.page <= 0 || c.pages > 0x7fffffffll)
    return fail(OMNIASR_ERR_ARGUMENT, "%s: %lld pages of %d positions", name, (long long)c.pages, c.page);
  if (!stride_ok(c.s_page, c.type) || !stride_ok(c.s_head, c.type) || !stride_ok(c.s_pos, c.type))
    return fail(OMNIASR_ERR_ARGUMENT, "%s: page strides (%lld, %lld, %lld) must keep 16-byte alignment", name,
                (long long)c.s_page, (long long)c.s_head, (long long)c.s_pos);
  if (c.page > 1 && c.s_pos < c.dim) return fail(OMNIASR_ERR_ARGUMENT, "%s: positions overlap", name);
  if (c.type == OMNIASR_FP8 && (!c.k_scale || !c.v_scale))
    return fail(OMNIASR_ERR_ARGUMENT, "%s: an fp8 cache needs its scale bytes", name);
  if (c.type == OMNIASR_FP8 && (!aligned16(c.k_scale) || !aligned16(c.v_scale)))
    return fail(OMNIASR_ERR_ARGUMENT, "%s: scale bytes must be 16-byte aligned", name);
  return OMNIASR_OK;
}

omni::PageCache cache_of(const void* k, const void* v, const void* ks, const void* vs, int64_t pages, int page, int64_t s_page,
                         int64_t s_head, int64_t s_pos, int kv_heads, int dim, int type) {
  omni::PageCache c;
  c.k = const_cast<void*>(k);
  c.v = const_cast<void*>(v);
  c.k_scale = reinterpret_cast<uint8_t*>(const_cast<void*>(ks));
  c.v_scale = reinterpret_cast<uint8_t*>(const_cast<void*>(vs));
  c.pages = pages;
  c.page = page;
  c.s_page = s_page;
  c.s_head = s_head;
  c.s_pos = s_pos;
  c.kv_heads = kv_heads;
  c.dim = dim;
  c.type = type;
  return c;
}

}  // namespace

extern "C" {

int omniasr_paged_rope_kv(const void* qkv, int64_t qkv_stride, const float* cs, int64_t cs_positions, const int64_t* pos,
                          const int64_t* slots, void* q_out, void* k_pages, void* v_pages, void* k_scale, void* v_scale,
                          int64_t pages, int page, int64_t stride_page, int64_t stride_head, int64_t stride_pos, int n,
                          int heads, int kv_heads, int dim, int dtype, int cache_type, int* status, cudaStream_t stream) {
  const char* name = "paged_rope_kv";
  if (int e = check(name, dtype, cache_type, dim, heads, kv_heads)) return e;
  if (n < 0 || cs_positions < 0) return fail(OMNIASR_ERR_ARGUMENT, "%s: n %d", name, n);
  omni::PagedRopeArgs a;
  a.c = cache_of(k_pages, v_pages, k_scale, v_scale, pages, page, stride_page, stride_head, stride_pos, kv_heads, dim, cache_type);
  if (int e = check_pages(name, a.c)) return e;
  if (n == 0) return done(name, cudaSuccess);
  if (!qkv || !cs || !pos || !slots || !q_out) return fail(OMNIASR_ERR_ARGUMENT, "%s: null pointer", name);
  if (!aligned16(qkv) || !aligned16(cs) || !aligned16(q_out) || !stride_ok(qkv_stride, dtype))
    return fail(OMNIASR_ERR_ARGUMENT, "%s: qkv, cs and q must keep 16-byte alignment", name);
  a.qkv = qkv;
  a.qkv_stride = qkv_stride;
  a.cs = cs;
  a.cs_positions = cs_positions;
  a.pos = pos;
  a.slots = slots;
  a.q_out = q_out;
  a.n = n;
  a.heads = heads;
  a.status = status;
  return done(name, omni::launch_paged_rope_kv(dtype, a, stream));
}

int omniasr_paged_kv_read(const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale, int64_t pages,
                          int page, int64_t stride_page, int64_t stride_head, int64_t stride_pos, const int32_t* table,
                          int64_t table_stride, int table_width, int rows, const int64_t* offsets, int64_t tokens,
                          void* k_out, void* v_out, int kv_heads, int dim, int dtype, int cache_type, int* status,
                          cudaStream_t stream) {
  const char* name = "paged_kv_read";
  if (int e = check(name, dtype, cache_type, dim, kv_heads, kv_heads)) return e;
  if (rows < 0 || tokens < 0 || table_width < 0 || tokens > 0x7fffffffll)
    return fail(OMNIASR_ERR_ARGUMENT, "%s: %d rows, %lld tokens", name, rows, (long long)tokens);
  omni::PagedReadArgs a;
  a.c = cache_of(k_pages, v_pages, k_scale, v_scale, pages, page, stride_page, stride_head, stride_pos, kv_heads, dim, cache_type);
  if (int e = check_pages(name, a.c)) return e;
  if (tokens == 0) return done(name, cudaSuccess);
  if (rows == 0) return fail(OMNIASR_ERR_ARGUMENT, "%s: %lld tokens of no rows", name, (long long)tokens);
  if (!table || !offsets || !k_out || !v_out) return fail(OMNIASR_ERR_ARGUMENT, "%s: null pointer", name);
  if (!aligned16(k_out) || !aligned16(v_out)) return fail(OMNIASR_ERR_ARGUMENT, "%s: outputs must be 16-byte aligned", name);
  a.table = table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.rows = rows;
  a.offsets = offsets;
  a.tokens = tokens;
  a.k_out = k_out;
  a.v_out = v_out;
  a.status = status;
  return done(name, omni::launch_paged_kv_read(dtype, a, stream));
}

size_t omniasr_paged_attention_workspace(int dtype, int cache_type, int rows, int tokens, int heads, int kv_heads, int dim,
                                         int page, int table_width) {
  if (!omni::dim_supported(dtype, dim) || rows < 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || page <= 0 ||
      table_width < 0)
    return 0;
  if (omni::paged_tc_supported(dtype, cache_type, dim, page)) return omni::paged_tc_workspace(dim);
  return omni::paged_attention_workspace(dtype, cache_type, rows ? rows : 1, tokens, heads, kv_heads, dim, page, table_width);
}

int omniasr_paged_attention(const void* q, const void* k_pages, const void* v_pages, const void* k_scale, const void* v_scale,
                            int64_t pages, int page, int64_t stride_page, int64_t stride_head, int64_t stride_pos,
                            const int32_t* table, int64_t table_stride, int table_width, const int64_t* lengths, void* out,
                            int rows, int tokens, int heads, int kv_heads, int dim, float scale, int dtype, int cache_type,
                            void* workspace, size_t workspace_bytes, int* status, cudaStream_t stream) {
  const char* name = "paged_attention";
  if (int e = check(name, dtype, cache_type, dim, heads, kv_heads)) return e;
  if (rows < 0 || rows > 65535 || tokens <= 0 || table_width < 0)
    return fail(OMNIASR_ERR_ARGUMENT, "%s: %d rows (at most 65535) of %d tokens", name, rows, tokens);
  if ((int64_t)table_width * page > 0x7fffff00ll)
    return fail(OMNIASR_ERR_ARGUMENT, "%s: %d pages of %d positions per row", name, table_width, page);
  if ((int64_t)tokens * heads > 65535)
    return fail(OMNIASR_ERR_ARGUMENT, "%s: %d tokens x %d heads per row (at most 65535)", name, tokens, heads);
  omni::PagedAttnArgs a;
  a.c = cache_of(k_pages, v_pages, k_scale, v_scale, pages, page, stride_page, stride_head, stride_pos, kv_heads, dim, cache_type);
  if (int e = check_pages(name, a.c)) return e;
  if (rows == 0) return done(name, cudaSuccess);
  if (!q || !out || !lengths || (!table && table_width)) return fail(OMNIASR_ERR_ARGUMENT, "%s: null pointer", name);
  if (!aligned16(q) || !aligned16(out)) return fail(OMNIASR_ERR_ARGUMENT, "%s: q and out must be 16-byte aligned", name);
  const size_t need = omniasr_paged_attention_workspace(dtype, cache_type, rows, tokens, heads, kv_heads, dim, page, table_width);
  if (!workspace || !aligned16(workspace) || workspace_bytes < need)
    return fail(OMNIASR_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes, need);
  a.q = q;
  a.table = table;
  a.table_stride = table_stride;
  a.table_width = table_width;
  a.lengths = lengths;
  a.out = out;
  a.rows = rows;
  a.tokens = tokens;
  a.heads = heads;
  a.scale = scale;
  a.workspace = workspace;
  a.status = status;
  if (omni::paged_tc_supported(dtype, cache_type, dim, page)) {
    const cudaError_t e = omni::launch_paged_attention_tc(a, stream);
    if (e == cudaErrorNotSupported)
      return fail(OMNIASR_ERR_UNSUPPORTED, "%s: page strides (%lld, %lld, %lld), or rows of that many keys", name,
                  (long long)stride_page, (long long)stride_head, (long long)stride_pos);
    return done(name, e);
  }
  return done(name, omni::launch_paged_attention(dtype, a, stream));
}

size_t omniasr_packed_attention_workspace(int64_t q_tokens, int heads, int kv_heads, int dim, int dtype) {
  if (!omni::dim_supported(dtype, dim) || q_tokens < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads) return 0;
  return omni::packed_workspace(dtype, q_tokens, heads, kv_heads, dim);
}

int omniasr_packed_attention(const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k, int64_t k_stride_tok,
                             int64_t k_stride_head, const void* v, int64_t v_stride_tok, int64_t v_stride_head, void* out,
                             const int64_t* q_offsets, const int64_t* k_offsets, int64_t q_tokens, int64_t k_tokens, int seqs,
                             int heads, int kv_heads, int dim, float scale, int dtype, void* workspace, size_t workspace_bytes,
                             int* status, cudaStream_t stream) {
  const char* name = "packed_attention";
  if (int e = check(name, dtype, dtype, dim, heads, kv_heads)) return e;
  if (seqs < 0 || q_tokens < 0 || k_tokens < 0 || q_tokens > 0x7fffffffll || k_tokens > 0x7fffffffll)
    return fail(OMNIASR_ERR_ARGUMENT, "%s: %d sequences, %lld queries, %lld keys", name, seqs, (long long)q_tokens,
                (long long)k_tokens);
  if (q_tokens == 0) return done(name, cudaSuccess);
  if (!q || !out || !q_offsets || !k_offsets || (k_tokens && (!k || !v)) || seqs == 0)
    return fail(OMNIASR_ERR_ARGUMENT, "%s: null pointer, or queries of no sequence", name);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(OMNIASR_ERR_ARGUMENT, "%s: pointers must be 16-byte aligned", name);
  const int64_t strides[6] = {q_stride_tok, q_stride_head, k_stride_tok, k_stride_head, v_stride_tok, v_stride_head};
  for (int64_t st : strides)
    if (!stride_ok(st, dtype)) return fail(OMNIASR_ERR_ARGUMENT, "%s: strides must keep 16-byte alignment", name);
  const size_t need = omniasr_packed_attention_workspace(q_tokens, heads, kv_heads, dim, dtype);
  if (!workspace || !aligned16(workspace) || workspace_bytes < need)
    return fail(OMNIASR_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", name, workspace_bytes, need);
  omni::PackedArgs a;
  a.q = q;
  a.q_st = q_stride_tok;
  a.q_sh = q_stride_head;
  a.k = k;
  a.k_st = k_stride_tok;
  a.k_sh = k_stride_head;
  a.v = v;
  a.v_st = v_stride_tok;
  a.v_sh = v_stride_head;
  a.out = out;
  a.q_offsets = q_offsets;
  a.k_offsets = k_offsets;
  a.q_tokens = q_tokens;
  a.k_tokens = k_tokens;
  a.seqs = seqs;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = dim;
  a.scale = scale;
  a.counters = reinterpret_cast<unsigned*>(workspace);
  a.status = status;
  return done(name, omni::launch_packed(dtype, a, stream));
}

}  // extern "C"
