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
  Pages p{k.data_ptr(), v.data_ptr(), nullptr, nullptr, k.size(0), k.size(1), k.size(2), k.size(3),
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
  p.type = code_of(k.scalar_type());
  if (p.type != dtype)
    refuse(name, "pages of " + std::string(c10::toString(k.scalar_type())) + " (supported: the queries' dtype, float8_e4m3fn)");
  if (ks || vs) refuse(name, "scales belong to float8_e4m3fn pages");
  return p;
}

void check_table(const char* name, const at::Tensor& t, int64_t rows) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) < rows || (t.size(1) > 1 && t.stride(1) != 1))
    refuse(name, "page_table must be int32 [rows, width] with unit inner stride");
}

int* status_of(int64_t p) { return reinterpret_cast<int*>(p); }
cudaStream_t stream_of(int64_t p) { return reinterpret_cast<cudaStream_t>(p); }

at::Tensor paged_rope_kv(const at::Tensor& qkv, const at::Tensor& cs_in, const at::Tensor& pos_in, const at::Tensor& k,
                         const at::Tensor& v, const at::Tensor& slots_in, int64_t heads, int64_t kv_heads, const Opt& ks,
                         const Opt& vs, int64_t status, int64_t stream) {
  const char* name = "paged_rope_kv";
  const int dtype = dtype_of(name, qkv);
  const Pages p = pages_of(name, k, v, ks, vs, dtype);
  const int64_t n = qkv.dim() == 2 ? qkv.size(0) : 0;
  if (p.kv != kv_heads || qkv.dim() != 2 || qkv.size(1) != (heads + 2 * kv_heads) * p.dim || (n && qkv.stride(1) != 1))
    refuse(name, "qkv must be [N, (heads + 2 * kv_heads) * D] with unit inner stride");
  if (pos_in.numel() != n || slots_in.numel() != n) refuse(name, "pos and slots must hold one entry per token");
  if (cs_in.dim() != 3 || cs_in.size(1) != p.dim / 2 || cs_in.size(2) != 2) refuse(name, "cs must be [P, D / 2, 2]");
  if (n > 0x7fffffff) refuse(name, "too many tokens");
  at::Tensor q = at::empty({n, heads, p.dim}, qkv.options());
  if (n == 0) return q;
  same_device(name, qkv, {&cs_in, &pos_in, &k, &v, &slots_in});
  const at::Tensor cs = cs_in.scalar_type() == at::kFloat && cs_in.is_contiguous() ? cs_in : cs_in.to(at::kFloat).contiguous();
  const at::Tensor pos = index_of(pos_in), slots = index_of(slots_in);
  done("omniasr_paged_rope_kv",
       omniasr_paged_rope_kv(qkv.data_ptr(), stride_of(qkv, 0), cs.data_ptr<float>(), cs.size(0), pos.data_ptr<int64_t>(),
                             slots.data_ptr<int64_t>(), q.data_ptr(), const_cast<void*>(p.k), const_cast<void*>(p.v),
                             const_cast<void*>(p.ks), const_cast<void*>(p.vs), p.pages, (int)p.page, p.sp, p.sh, p.st, (int)n,
                             (int)heads, (int)kv_heads, (int)p.dim, dtype, p.type, status_of(status), stream_of(stream)));
  return q;
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

}  // namespace

PYBIND11_MODULE(_omniasr_torch, m) {
  m.def("paged_rope_kv", &paged_rope_kv);
  m.def("paged_kv_read", &paged_kv_read);
  m.def("paged_attention", &paged_attention);
  m.def("packed_attention", &packed_attention);
}
