// The Python calls of the paged cache and the packed prompts, as one native step each: argument checks, output allocation
// and the C ABI call (include/omniasr_b200.h). Through ctypes a call takes the host about 12 us, which is what a small call
// then waits for; here about half. kernels.py holds the functions' documentation, the status words and the workspaces.

#include <ATen/ATen.h>
#include <torch/csrc/utils/pybind.h>

#include <string>

#include "omniasr_b200.h"

namespace py = pybind11;

namespace {

using Opt = std::optional<at::Tensor>;

[[noreturn]] void refuse(const char* name, const std::string& what) { throw py::value_error(std::string(name) + ": " + what); }

void done(const char* fn, int code) {
  if (code == OMNIASR_OK) return;
  const std::string msg = omniasr_last_error();
  if (code == OMNIASR_ERR_ARGUMENT || code == OMNIASR_ERR_UNSUPPORTED || code == OMNIASR_ERR_WORKSPACE)
    throw py::value_error(std::string(fn) + ": " + msg);
  py::object error = py::module_::import("omniasr_b200._lib").attr("KernelError")(fn, code, msg);
  PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(error.ptr())), error.ptr());
  throw py::error_already_set();
}

int code_of(at::ScalarType t) { return t == at::kBFloat16 ? OMNIASR_BF16 : t == at::kFloat ? OMNIASR_F32 : -1; }

int dtype_of(const char* name, const at::Tensor& t) {
  const int code = code_of(t.scalar_type());
  if (code < 0) refuse(name, "dtype " + std::string(c10::toString(t.scalar_type())) + " (supported: bfloat16, float32)");
  return code;
}

// int64, contiguous (index tensors are torch.long; others are converted).
at::Tensor index_of(const at::Tensor& t) {
  if (t.scalar_type() == at::kLong && t.is_contiguous()) return t;
  return t.to(at::kLong).contiguous();
}

void same_device(const char* name, const at::Tensor& a, std::initializer_list<const at::Tensor*> others) {
  if (!a.is_cuda()) refuse(name, "tensors must be on a CUDA device");
  for (const at::Tensor* t : others)
    if (t->device() != a.device()) refuse(name, "tensors must be on one device");
}

// The stride of a dimension; nothing reads that of an extent of one, where PyTorch leaves any number.
int64_t stride_of(const at::Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

struct Pages {
  const void *k, *v, *ks, *vs;
  int64_t pages, kv, page, dim, sp, sh, st;
  int type;
};

Pages pages_of(const char* name, const at::Tensor& k, const at::Tensor& v, const Opt& ks, const Opt& vs, int dtype) {
  bool same = k.dim() == 4 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type();
  for (int64_t i = 0; same && i < 3; ++i) same = stride_of(k, i) == stride_of(v, i);
  if (!same || k.stride(3) != 1 || v.stride(3) != 1)
    refuse(name, "k and v pages must be [pages, kv_heads, page, D] views of one dtype with the same strides and unit stride in D");
  const bool int4 = k.scalar_type() == at::kByte;  // 4-bit codes, two to a byte
  Pages p{k.data_ptr(), v.data_ptr(), nullptr, nullptr, k.size(0), k.size(1), k.size(2), int4 ? 2 * k.size(3) : k.size(3),
          stride_of(k, 0), stride_of(k, 1), stride_of(k, 2), 0};
  if (k.scalar_type() == at::kFloat8_e4m3fn) {
    for (const Opt* s : {&ks, &vs}) {
      if (!*s || (*s)->scalar_type() != at::kByte || (*s)->sizes() != k.sizes().slice(0, 3) || !(*s)->is_contiguous())
        refuse(name, "float8_e4m3fn pages need contiguous uint8 scales [pages, kv_heads, page]");
    }
    same_device(name, k, {&v, &*ks, &*vs});
    p.ks = ks->data_ptr();
    p.vs = vs->data_ptr();
    p.type = OMNIASR_FP8;
    return p;
  }
  if (int4) {
    const int64_t shape[4] = {k.size(0), k.size(1), k.size(2), p.dim / 32};
    for (const Opt* s : {&ks, &vs}) {
      if (!*s || (*s)->scalar_type() != at::kBFloat16 || (*s)->sizes() != at::IntArrayRef(shape, 4) || !(*s)->is_contiguous())
        refuse(name, "uint8 pages (4-bit codes) need contiguous bfloat16 scales [pages, kv_heads, page, D / 32]");
    }
    same_device(name, k, {&v, &*ks, &*vs});
    p.ks = ks->data_ptr();
    p.vs = vs->data_ptr();
    p.type = OMNIASR_INT4;
    return p;
  }
  p.type = code_of(k.scalar_type());
  if (p.type != dtype)
    refuse(name, "pages of " + std::string(c10::toString(k.scalar_type())) +
                     " (supported: the queries' dtype, float8_e4m3fn, uint8 of 4-bit codes)");
  if (ks || vs) refuse(name, "scales belong to float8_e4m3fn and uint8 pages");
  return p;
}

void check_table(const char* name, const at::Tensor& t, int64_t rows) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) < rows || (t.size(1) > 1 && t.stride(1) != 1))
    refuse(name, "page_table must be int32 [rows, width] with unit inner stride");
}

int* status_of(int64_t p) { return reinterpret_cast<int*>(p); }
cudaStream_t stream_of(int64_t p) { return reinterpret_cast<cudaStream_t>(p); }

// paged_rope_kv, and paged_norm_rope_kv where the norms' weights are given.
at::Tensor rope(const char* name, const at::Tensor& qkv, const Opt& q_norm, const Opt& k_norm, double eps, const at::Tensor& cs_in,
                const at::Tensor& pos_in, const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots_in, int64_t heads,
                int64_t kv_heads, const Opt& ks, const Opt& vs, int64_t status, int64_t stream) {
  const int dtype = dtype_of(name, qkv);
  const Pages p = pages_of(name, k, v, ks, vs, dtype);
  const int64_t n = qkv.dim() == 2 ? qkv.size(0) : 0;
  if (p.kv != kv_heads || qkv.dim() != 2 || qkv.size(1) != (heads + 2 * kv_heads) * p.dim || (n && qkv.stride(1) != 1))
    refuse(name, "qkv must be [N, (heads + 2 * kv_heads) * D] with unit inner stride");
  if (pos_in.numel() != n || slots_in.numel() != n) refuse(name, "pos and slots must hold one entry per token");
  if (cs_in.dim() != 3 || cs_in.size(1) != p.dim / 2 || cs_in.size(2) != 2) refuse(name, "cs must be [P, D / 2, 2]");
  if (q_norm) {
    for (const Opt* w : {&q_norm, &k_norm})
      if ((*w)->dim() != 1 || (*w)->size(0) != p.dim || (*w)->scalar_type() != qkv.scalar_type() || (*w)->stride(0) != 1)
        refuse(name, "q_norm and k_norm must be contiguous [D] of qkv's dtype");
  }
  if (n > 0x7fffffff) refuse(name, "too many tokens");
  at::Tensor q = at::empty({n, heads, p.dim}, qkv.options());
  if (n == 0) return q;
  same_device(name, qkv, {&cs_in, &pos_in, &k, &v, &slots_in});
  const at::Tensor cs = cs_in.scalar_type() == at::kFloat && cs_in.is_contiguous() ? cs_in : cs_in.to(at::kFloat).contiguous();
  const at::Tensor pos = index_of(pos_in), slots = index_of(slots_in);
  void *kp = const_cast<void*>(p.k), *vp = const_cast<void*>(p.v), *ksp = const_cast<void*>(p.ks), *vsp = const_cast<void*>(p.vs);
  if (q_norm) {
    same_device(name, qkv, {&*q_norm, &*k_norm});
    done("omniasr_paged_norm_rope_kv",
         omniasr_paged_norm_rope_kv(qkv.data_ptr(), stride_of(qkv, 0), q_norm->data_ptr(), k_norm->data_ptr(), (float)eps,
                                    cs.data_ptr<float>(), cs.size(0), pos.data_ptr<int64_t>(), slots.data_ptr<int64_t>(),
                                    q.data_ptr(), kp, vp, ksp, vsp, p.pages, (int)p.page, p.sp, p.sh, p.st, (int)n, (int)heads,
                                    (int)kv_heads, (int)p.dim, dtype, p.type, status_of(status), stream_of(stream)));
  } else {
    done("omniasr_paged_rope_kv",
         omniasr_paged_rope_kv(qkv.data_ptr(), stride_of(qkv, 0), cs.data_ptr<float>(), cs.size(0), pos.data_ptr<int64_t>(),
                               slots.data_ptr<int64_t>(), q.data_ptr(), kp, vp, ksp, vsp, p.pages, (int)p.page, p.sp, p.sh, p.st,
                               (int)n, (int)heads, (int)kv_heads, (int)p.dim, dtype, p.type, status_of(status), stream_of(stream)));
  }
  return q;
}

at::Tensor paged_rope_kv(const at::Tensor& qkv, const at::Tensor& cs, const at::Tensor& pos, const at::Tensor& k,
                         const at::Tensor& v, const at::Tensor& slots, int64_t heads, int64_t kv_heads, const Opt& ks,
                         const Opt& vs, int64_t status, int64_t stream) {
  return rope("paged_rope_kv", qkv, std::nullopt, std::nullopt, 0., cs, pos, k, v, slots, heads, kv_heads, ks, vs, status, stream);
}

at::Tensor paged_norm_rope_kv(const at::Tensor& qkv, const at::Tensor& q_norm, const at::Tensor& k_norm, const at::Tensor& cs,
                              const at::Tensor& pos, const at::Tensor& k, const at::Tensor& v, const at::Tensor& slots,
                              int64_t heads, int64_t kv_heads, double eps, const Opt& ks, const Opt& vs, int64_t status,
                              int64_t stream) {
  return rope("paged_norm_rope_kv", qkv, q_norm, k_norm, eps, cs, pos, k, v, slots, heads, kv_heads, ks, vs, status, stream);
}

std::pair<at::Tensor, at::Tensor> paged_kv_read(const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                                                const at::Tensor& offsets_in, int64_t tokens, const Opt& ks, const Opt& vs,
                                                at::ScalarType kind, int64_t status, int64_t stream) {
  const char* name = "paged_kv_read";
  const int dtype = code_of(kind);
  if (dtype < 0) refuse(name, "dtype " + std::string(c10::toString(kind)) + " (supported: bfloat16, float32)");
  const Pages p = pages_of(name, k, v, ks, vs, dtype);
  const int64_t rows = offsets_in.numel() - 1;
  if (rows < 0 || rows > 0x7fffffff) refuse(name, "offsets must hold rows + 1 entries");
  check_table(name, table, rows);
  if (tokens < 0) refuse(name, "a negative number of tokens");
  at::Tensor ko = at::empty({tokens, p.kv, p.dim}, k.options().dtype(kind)), vo = at::empty_like(ko);
  if (tokens == 0) return {ko, vo};
  same_device(name, k, {&v, &table, &offsets_in});
  const at::Tensor offsets = index_of(offsets_in);
  done("omniasr_paged_kv_read",
       omniasr_paged_kv_read(p.k, p.v, p.ks, p.vs, p.pages, (int)p.page, p.sp, p.sh, p.st, table.data_ptr<int32_t>(), table.stride(0),
                             (int)table.size(1), (int)rows, offsets.data_ptr<int64_t>(), tokens, ko.data_ptr(), vo.data_ptr(),
                             (int)p.kv, (int)p.dim, dtype, p.type, status_of(status), stream_of(stream)));
  return {ko, vo};
}

// The result, or the bytes of workspace that the call needs where `ws` is smaller (nothing has run then).
py::object paged_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& table,
                           const at::Tensor& lengths_in, double scale, int64_t tokens, const Opt& ks, const Opt& vs, int64_t status,
                           int64_t stream, const Opt& ws) {
  const char* name = "paged_attention";
  if (q.dim() != 3 || !q.is_contiguous()) refuse(name, "q must be contiguous [B * tokens, heads, D]");
  const int dtype = dtype_of(name, q);
  const Pages p = pages_of(name, k, v, ks, vs, dtype);
  const int64_t rows_q = q.size(0), heads = q.size(1), dim = q.size(2);
  if (p.dim != dim) refuse(name, "q and the pages differ in head_dim");
  if (tokens < 1 || rows_q % tokens || lengths_in.numel() * tokens != rows_q)
    refuse(name, std::to_string(rows_q) + " queries are not " + std::to_string(lengths_in.numel()) + " rows of " +
                     std::to_string(tokens) + " tokens");
  const int64_t rows = rows_q / tokens;
  check_table(name, table, rows);
  if (rows == 0) return py::cast(at::empty_like(q));
  if (rows > 0x7fffffff || heads > 0x7fffffff || tokens > 0x7fffffff || table.size(1) > 0x7fffffff) refuse(name, "sizes past 2^31");
  same_device(name, q, {&k, &v, &table, &lengths_in});
  const size_t need = omniasr_paged_attention_workspace(dtype, p.type, (int)rows, (int)tokens, (int)heads, (int)p.kv, (int)dim,
                                                        (int)p.page, (int)table.size(1));
  if (!ws || (size_t)ws->numel() < need) return py::int_(need);
  const at::Tensor lengths = index_of(lengths_in);
  at::Tensor out = at::empty_like(q);
  done("omniasr_paged_attention",
       omniasr_paged_attention(q.data_ptr(), p.k, p.v, p.ks, p.vs, p.pages, (int)p.page, p.sp, p.sh, p.st, table.data_ptr<int32_t>(),
                               table.stride(0), (int)table.size(1), lengths.data_ptr<int64_t>(), out.data_ptr(), (int)rows,
                               (int)tokens, (int)heads, (int)p.kv, (int)dim, (float)scale, dtype, p.type, ws->data_ptr(), ws->numel(),
                               status_of(status), stream_of(stream)));
  return py::cast(out);
}

py::object packed_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_offsets_in,
                            const Opt& k_offsets_in, std::optional<double> scale, int64_t status, int64_t stream, const Opt& ws) {
  const char* name = "packed_attention";
  if (q.dim() != 3 || k.dim() != 3 || v.sizes() != k.sizes() || q.size(2) != k.size(2))
    refuse(name, "q [Tq, heads, D], k and v [Tk, kv_heads, D]");
  if (k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type()) refuse(name, "q, k and v must share a dtype");
  const int64_t tq = q.size(0), heads = q.size(1), dim = q.size(2), tk = k.size(0), kv = k.size(1);
  if ((tq && q.stride(2) != 1) || (tk && (k.stride(2) != 1 || v.stride(2) != 1))) refuse(name, "unit stride in D");
  const int dtype = dtype_of(name, q);
  const at::Tensor& ko_in = k_offsets_in ? *k_offsets_in : q_offsets_in;
  const int64_t seqs = q_offsets_in.numel() - 1;
  if (seqs < 0 || ko_in.numel() != seqs + 1) refuse(name, "q_offsets and k_offsets must hold sequences + 1 entries");
  if (tq == 0) return py::cast(at::empty({tq, heads, dim}, q.options()));
  if (seqs > 0x7fffffff || heads > 0x7fffffff || kv > 0x7fffffff) refuse(name, "sizes past 2^31");
  same_device(name, q, {&k, &v, &q_offsets_in, &ko_in});
  const size_t need = omniasr_packed_attention_workspace(tq, (int)heads, (int)kv, (int)dim, dtype);
  if (!ws || (size_t)ws->numel() < need) return py::int_(need);
  const at::Tensor qo = index_of(q_offsets_in), ko = index_of(ko_in);
  at::Tensor out = at::empty({tq, heads, dim}, q.options());
  const double s = scale ? *scale : 1.0 / std::sqrt((double)dim);
  done("omniasr_packed_attention",
       omniasr_packed_attention(q.data_ptr(), stride_of(q, 0), stride_of(q, 1), k.data_ptr(), stride_of(k, 0), stride_of(k, 1),
                                v.data_ptr(), stride_of(v, 0), stride_of(v, 1), out.data_ptr(), qo.data_ptr<int64_t>(),
                                ko.data_ptr<int64_t>(), tq, tk, (int)seqs, (int)heads, (int)kv, (int)dim, (float)s, dtype,
                                ws->data_ptr(), ws->numel(), status_of(status), stream_of(stream)));
  return py::cast(out);
}

// Whether rows of a and of b (2-D, unit inner stride, one element size) share memory. Columns of one buffer's rows that lie side by side
// do not.
bool rows_overlap(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const int64_t es = a.element_size(), la = stride_of(a, 0), lb = stride_of(b, 0);
  const int64_t pa = reinterpret_cast<int64_t>(a.data_ptr()) / es, pb = reinterpret_cast<int64_t>(b.data_ptr()) / es;
  if (pa + (a.size(0) - 1) * la + a.size(1) <= pb || pb + (b.size(0) - 1) * lb + b.size(1) <= pa) return false;
  if (la != lb || la <= 0) return true;
  const int64_t at = ((pb - pa) % la + la) % la;  // where b's rows begin in a's
  return at < a.size(1) || at + b.size(1) > la;
}

at::Tensor decode_gemm_int4(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scales, int64_t wrows, int64_t k,
                            int64_t group, int64_t mode, const Opt& residual, const Opt& out, int64_t stream) {
  const char* name = "decode_gemm_int4";
  if (x.scalar_type() != at::kBFloat16 || x.dim() != 2 || x.size(1) != k || (k > 1 && x.size(0) && x.stride(1) != 1))
    refuse(name, "x must be bfloat16 [rows, " + std::to_string(k) + "] with unit inner stride");
  const int64_t rows = x.size(0), n = mode == OMNIASR_GEMM_SWIGLU ? wrows / 2 : wrows;
  if (mode == OMNIASR_GEMM_SWIGLU && wrows % 2) refuse(name, "swiglu needs the rows of [gate; inner]");
  auto bf16_rows = [&](const at::Tensor& t, const char* what) {
    if (t.scalar_type() != at::kBFloat16 || t.dim() != 2 || t.size(0) != rows || t.size(1) != n || (n > 1 && rows && t.stride(1) != 1))
      refuse(name, std::string(what) + " must be bfloat16 [rows, n] with unit inner stride");
  };
  if ((mode == OMNIASR_GEMM_RESIDUAL) != residual.has_value()) refuse(name, "a residual belongs to the residual mode, and that to it");
  if (residual) bf16_rows(*residual, "residual");
  if (out) bf16_rows(*out, "out");
  if (out && (rows_overlap(x, *out) || (residual && (residual->data_ptr() != out->data_ptr() ||
                                                     stride_of(*residual, 0) != stride_of(*out, 0)) && rows_overlap(*residual, *out))))
    refuse(name, "out must not share memory with x, nor with the residual unless it is the residual");
  if (rows > 64) refuse(name, "at most 64 rows");
  if (group != 32 && group != 64 && group != 128) refuse(name, "groups of 32, 64 or 128 columns");
  const int64_t tiles = (wrows + 7) / 8;
  if (wrows < 0 || codes.scalar_type() != at::kByte || !codes.is_contiguous() || codes.numel() != tiles * ((k + 127) / 128) * 512 ||
      scales.scalar_type() != at::kBFloat16 || !scales.is_contiguous() || scales.numel() != tiles * ((k + group - 1) / group) * 8)
    refuse(name, "codes and scales are not those of " + std::to_string(wrows) + " x " + std::to_string(k) + " weights (int4_weights)");
  at::Tensor y = out ? *out : at::empty({rows, n}, x.options());
  if (rows == 0 || n == 0) return y;
  same_device(name, x, {&codes, &scales, &y});
  if (residual) same_device(name, x, {&*residual});
  done("omniasr_decode_gemm_int4",
       omniasr_decode_gemm_int4(x.data_ptr(), stride_of(x, 0), (int)rows, codes.data_ptr(), scales.data_ptr(), (int)n, (int)k,
                                (int)group, (int)mode, residual ? residual->data_ptr() : nullptr,
                                residual ? stride_of(*residual, 0) : 0, y.data_ptr(), stride_of(y, 0), stream_of(stream)));
  return y;
}

struct Tables {
  int64_t requests;
  at::Tensor rows, want;
};

Tables tables_of(const char* name, const at::Tensor& rows, const at::Tensor& want, int64_t page, const at::Tensor& length,
                 const at::Tensor& table, const at::Tensor& free, const at::Tensor& free_count) {
  if (rows.dim() != 1 || want.sizes() != rows.sizes()) refuse(name, "rows and their numbers must be [requests]");
  if (length.scalar_type() != at::kLong || length.dim() != 1 || !length.is_contiguous())
    refuse(name, "length must be contiguous int64 [sequences]");
  if (table.scalar_type() != at::kInt || table.dim() != 2 || table.size(0) != length.size(0) || (table.size(1) > 1 && table.stride(1) != 1))
    refuse(name, "table must be int32 [sequences, width] with unit inner stride");
  if (free.scalar_type() != at::kInt || free.dim() != 1 || !free.is_contiguous()) refuse(name, "free must be contiguous int32 [pages]");
  if (free_count.scalar_type() != at::kLong || free_count.numel() != 1) refuse(name, "free_count must be one int64");
  if (page < 1 || page > 0x7fffffff || table.size(1) > 0x7fffffff) refuse(name, "pages of " + std::to_string(page) + " positions");
  if (rows.size(0) > 0x7fffffff) refuse(name, "too many requests");
  same_device(name, length, {&rows, &want, &table, &free, &free_count});
  return {rows.size(0), index_of(rows), index_of(want)};
}

// (A table of one row or none may have any stride.)
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

py::object paged_plan(const at::Tensor& rows, const at::Tensor& fresh, int64_t tokens, int64_t page, const at::Tensor& length,
                      const at::Tensor& table, const at::Tensor& free, const at::Tensor& free_count, std::optional<int64_t> width,
                      std::optional<int64_t> positions, int64_t status, int64_t stream, const Opt& ws) {
  const char* name = "paged_plan";
  const Tables t = tables_of(name, rows, fresh, page, length, table, free, free_count);
  const int64_t w = width ? *width : table.size(1);
  if (tokens < 0 || tokens > 0x7fffffff) refuse(name, std::to_string(tokens) + " tokens");
  if (w < 0 || w > table.size(1)) refuse(name, "a width of " + std::to_string(w) + " of a table of " + std::to_string(table.size(1)));
  if (positions && *positions < 1) refuse(name, std::to_string(*positions) + " positions");
  if (!ws) return py::int_(OMNIASR_PLAN_WORKSPACE);
  const int64_t b = t.requests;
  const auto i64 = length.options();
  // One allocation for the int64 outputs: positions, slots, lengths, offsets.
  const std::vector<at::Tensor> parts = at::empty({2 * tokens + 3 * b + 2}, i64).unsafe_split_with_sizes({tokens, tokens, b, b + 1, b + 1});
  const at::Tensor &pos = parts[0], &slots = parts[1], &lengths = parts[2], &qo = parts[3], &ko = parts[4];
  at::Tensor out = at::empty({b, w}, table.options()), taken = at::empty({b}, i64.dtype(at::kBool));
  done("omniasr_paged_plan",
       omniasr_paged_plan_within(t.rows.data_ptr<int64_t>(), t.want.data_ptr<int64_t>(), (int)b, tokens, (int)page,
                                 length.data_ptr<int64_t>(), length.size(0), table.data_ptr<int32_t>(), row_stride(table),
                                 (int)table.size(1), free.data_ptr<int32_t>(), free_count.data_ptr<int64_t>(), free.size(0),
                                 positions.value_or(INT64_MAX), pos.data_ptr<int64_t>(), slots.data_ptr<int64_t>(),
                                 out.data_ptr<int32_t>(), (int)w, lengths.data_ptr<int64_t>(), qo.data_ptr<int64_t>(),
                                 ko.data_ptr<int64_t>(), reinterpret_cast<uint8_t*>(taken.data_ptr()), ws->data_ptr(), ws->numel(),
                                 status_of(status), stream_of(stream)));
  return py::make_tuple(pos, slots, out, lengths, qo, ko, taken);
}

py::object paged_trim(const at::Tensor& rows, const at::Tensor& keep, int64_t page, const at::Tensor& length, const at::Tensor& table,
                      const at::Tensor& free, const at::Tensor& free_count, int64_t status, int64_t stream, const Opt& ws) {
  const char* name = "paged_trim";
  const Tables t = tables_of(name, rows, keep, page, length, table, free, free_count);
  if (!ws) return py::int_(OMNIASR_PLAN_WORKSPACE);
  done("omniasr_paged_trim",
       omniasr_paged_trim(t.rows.data_ptr<int64_t>(), t.want.data_ptr<int64_t>(), (int)t.requests, (int)page, length.data_ptr<int64_t>(),
                          length.size(0), table.data_ptr<int32_t>(), row_stride(table), (int)table.size(1), free.data_ptr<int32_t>(),
                          free_count.data_ptr<int64_t>(), free.size(0), ws->data_ptr(), ws->numel(), status_of(status),
                          stream_of(stream)));
  return py::none();
}

}  // namespace

PYBIND11_MODULE(_omniasr_torch, m) {
  m.def("paged_rope_kv", &paged_rope_kv);
  m.def("paged_norm_rope_kv", &paged_norm_rope_kv);
  m.def("paged_kv_read", &paged_kv_read);
  m.def("paged_attention", &paged_attention);
  m.def("packed_attention", &packed_attention);
  m.def("decode_gemm_int4", &decode_gemm_int4);
  m.def("paged_plan", &paged_plan);
  m.def("paged_trim", &paged_trim);
}
