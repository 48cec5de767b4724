// Host side of shard_b200.fp4 and shard_b200.route for torch: one call checks its tensors, allocates its outputs through
// torch and enqueues the C-ABI entry on the tensors' current stream. A call for one decoded token is bound by
// its host side: through ctypes, with the checks and allocations in Python, quantising a row takes 8.3 us and
// a product 8.7.
//
// The functions take positional arguments, raise ValueError for tensors that the operators refuse, and return the
// entry's status (an int) where it is not SB_OK; the Python wrappers document them.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include "../../include/shard_b200.h"

namespace {

using at::Tensor;

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) throw torch::TypeError(c10::str(what, ": expected a tensor"));
  return THPVariable_Unpack(o);
}

// a tensor or None
const Tensor* optional(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

#define REFUSE(...) TORCH_CHECK_VALUE(false, __VA_ARGS__)

void same_device(const char* what, const Tensor& ref, const Tensor& t) {
  if (t.device() != ref.device())
    REFUSE(what, ": tensors on ", t.device(), " and ", ref.device());
}

// sb_dtype, or -1
int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? SB_BF16 : t == at::kHalf ? SB_F16 : t == at::kFloat ? SB_F32 : -1;
}
at::ScalarType dtype_of(int code) { return code == SB_BF16 ? at::kBFloat16 : code == SB_F16 ? at::kHalf : at::kFloat; }

void* current_stream(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

Tensor empty(at::IntArrayRef size, at::ScalarType type, const Tensor& like) {
  return at::empty(size, at::TensorOptions().dtype(type).device(like.device()));
}

const int32_t* int_vector(const char* what, const char* name, const Tensor& ref, const Tensor& t) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || !t.is_contiguous())
    REFUSE(what, ": ", name, " must be a contiguous int32 vector");
  same_device(what, ref, t);
  return t.data_ptr<int32_t>();
}

const float* float_values(const char* what, const char* name, const Tensor& ref, const Tensor& t, int64_t n) {
  if (t.scalar_type() != at::kFloat || !t.is_contiguous() || t.numel() != n)
    REFUSE(what, ": ", name, " must be contiguous fp32 with ", n, " values");
  same_device(what, ref, t);
  return t.data_ptr<float>();
}

int64_t as_int(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
// a C int of the entries: what lies outside is refused as the nearest one is
int as_c_int(PyObject* o) {
  const int64_t v = as_int(o);
  return (int)(v < INT32_MIN ? INT32_MIN : v > INT32_MAX ? INT32_MAX : v);
}
double as_float(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
void* as_ptr(PyObject* o) { return o == Py_None ? nullptr : reinterpret_cast<void*>(as_int(o)); }
bool as_bool(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}

PyObject* status(int rc) { return PyLong_FromLong(rc); }

void count(const char* what, Py_ssize_t n, Py_ssize_t want) {
  if (n != want) throw torch::TypeError(c10::str(what, ": ", want, " arguments, not ", n));
}

// quant(x, fmt, tensor_scale, rows, offsets) -> (buffer, rows, k, one scale per row, end of the codes, end of the
// scales, address, leading sizes) | status
PyObject* quant(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count("quant", nargs, 5);
  const Tensor& x = tensor(args[0], "quant");
  const int fmt = (int)as_int(args[1]);
  const Tensor *scale = optional(args[2], "quant"), *rows = optional(args[3], "quant"), *off = optional(args[4], "quant");
  const int dt = dtype_code(x.scalar_type());
  if (dt < 0 || !x.is_cuda() || x.dim() < 1) REFUSE("quant: x must be a CUDA tensor of bf16, fp16 or fp32");
  const bool nv = fmt == SB_FMT_NVFP4;
  const int64_t k = x.size(-1);
  if (k < 1) REFUSE("quant: rows of no values");
  Tensor z = x;
  if (x.dim() != 2) z = x.reshape({x.numel() / k, k});
  if (k > 1 && z.stride(1) != 1) z = z.contiguous();
  const int64_t m = z.size(0);
  int64_t p = m, groups = 0;
  const int32_t *rp = nullptr, *op = nullptr;
  const float* tp = nullptr;
  if (rows) {
    rp = int_vector("quant", "rows", x, *rows);
    p = rows->numel();
  }
  if (off) {
    op = int_vector("quant", "offsets", x, *off);
    groups = off->numel() - 1;
    if (groups < 1) REFUSE("quant: offsets must hold at least two values");
  }
  if (scale) {
    if (!nv) REFUSE("quant: MXFP4 has no tensor scale");
    tp = float_values("quant", "tensor_scale", x, *scale, 1);
  }
  // one allocation: codes, scale atoms, the rows' tensor scales
  const bool per_row = nv && !scale;
  const int64_t end = p * ((k + 31) / 32) * 16, atoms_end = end + (int64_t)sb_fp4_scale_bytes(fmt, 1, p, k, groups);
  Tensor buf = empty({per_row ? atoms_end + 4 * p : atoms_end}, at::kByte, x);
  uint8_t* base = buf.data_ptr<uint8_t>();
  const size_t need = rows ? sb_fp4_quant_workspace_bytes(fmt, m, p, k) : 0;
  Tensor ws;
  if (need) ws = empty({(int64_t)need}, at::kByte, x);
  // (a gather of no rows has no pointer, which the entry takes for none: no source rows, then)
  const int64_t src = rows && p == 0 ? 0 : m;
  const int rc = sb_fp4_quant(fmt, z.data_ptr(), dt, src, k, m > 1 ? z.stride(0) : k, rp, p, tp, op, groups, base, base + end,
                              per_row ? reinterpret_cast<float*>(base + atoms_end) : nullptr, need ? ws.data_ptr() : nullptr, need,
                              current_stream(x));
  if (rc != SB_OK) return status(rc);
  const int64_t lead = rows ? 1 : x.dim() - 1;
  THPObjectPtr shape(PyTuple_New(lead));
  if (!shape) throw python_error();
  for (int64_t i = 0; i < lead; ++i) PyTuple_SET_ITEM(shape.get(), i, PyLong_FromLongLong(rows ? p : x.size(i)));
  return Py_BuildValue("(NLLOLLLN)", THPVariable_Wrap(std::move(buf)), (long long)p, (long long)k, per_row ? Py_True : Py_False,
                       (long long)end, (long long)atoms_end, (long long)reinterpret_cast<intptr_t>(base), shape.release());
  END_HANDLE_TH_ERRORS
}

at::DimVector sizes(PyObject* lead, int64_t last) {
  at::DimVector s;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(lead); ++i) s.push_back(as_int(PyTuple_GET_ITEM(lead, i)));
  s.push_back(last);
  return s;
}

// dequant(buffer, fmt, codes, scales, ts, one per row, rows, k, leading sizes, dtype) -> y | status
PyObject* dequant(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count("dequant", nargs, 10);
  const Tensor& buf = tensor(args[0], "dequant");
  const int64_t k = as_int(args[7]);
  const int dt = (int)as_int(args[9]);
  Tensor y = empty(sizes(args[8], k), dtype_of(dt), buf);
  const int rc = sb_fp4_dequant((int)as_int(args[1]), as_ptr(args[2]), as_ptr(args[3]), (const float*)as_ptr(args[4]),
                                as_bool(args[5]), as_int(args[6]), k, y.data_ptr(), dt, current_stream(buf));
  return rc != SB_OK ? status(rc) : THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// The output of a product: `out` if given, checked, else new rows of `n` (of the leading sizes `lead`, or [m]).
Tensor output(const char* what, PyObject* out, int64_t m, int64_t n, PyObject* lead, at::ScalarType type, const Tensor& like,
              int64_t* ld) {
  *ld = n;
  if (out == Py_None) return lead ? empty(sizes(lead, n), type, like) : empty({m, n}, type, like);
  const Tensor& t = tensor(out, what);
  if (t.dim() != 2 || t.size(0) != m || t.size(1) != n || t.scalar_type() != type || t.device() != like.device() ||
      (n > 1 && t.numel() > 0 && t.stride(1) != 1) || (m > 1 && t.stride(0) < n))
    REFUSE(what, ": out must be [", m, ", ", n, "] of out_dtype on ", like.device(),
           ", with contiguous rows that do not overlap");
  if (m > 1) *ld = t.stride(0);
  return t;
}

// gemm(a buffer, fmt, a codes, scales, ts, per row, m, leading sizes, k, w codes, scales, ts, per row, n, dtype, out)
// -> y | status
PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count("gemm", nargs, 16);
  const Tensor& buf = tensor(args[0], "gemm");
  const int64_t m = as_int(args[6]), n = as_int(args[13]);
  const int dt = (int)as_int(args[14]);
  int64_t ld = 0;
  Tensor y = output("gemm", args[15], m, n, args[7], dtype_of(dt), buf, &ld);
  const int rc = sb_fp4_gemm((int)as_int(args[1]), as_ptr(args[2]), as_ptr(args[3]), (const float*)as_ptr(args[4]),
                             as_bool(args[5]), m, as_ptr(args[9]), as_ptr(args[10]), (const float*)as_ptr(args[11]),
                             as_bool(args[12]), n, as_int(args[8]), y.data_ptr(), dt, ld, current_stream(buf));
  return rc != SB_OK ? status(rc) : THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// grouped_gemm(a buffer, fmt, a codes, scales, ts, per row, m, k, offsets, w codes, scales, ts, scales a matrix,
// matrices, n, swiglu, limit, row weight, dtype, out) -> y | status
PyObject* grouped_gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count("grouped_gemm", nargs, 20);
  const Tensor& buf = tensor(args[0], "grouped_gemm");
  const int64_t m = as_int(args[6]), n = as_int(args[14]);
  const int32_t* off = int_vector("grouped_gemm", "offsets", buf, tensor(args[8], "grouped_gemm"));
  const bool swiglu = as_bool(args[15]);
  const Tensor* weight = optional(args[17], "grouped_gemm");
  const float* wp = weight ? float_values("grouped_gemm", "row_weight", buf, *weight, m) : nullptr;
  const int dt = (int)as_int(args[18]);
  int64_t ld = 0;
  Tensor y = output("grouped_gemm", args[19], m, swiglu ? n / 2 : n, nullptr, dtype_of(dt), buf, &ld);
  const int rc = sb_fp4_grouped_gemm((int)as_int(args[1]), as_ptr(args[2]), as_ptr(args[3]), (const float*)as_ptr(args[4]),
                                     as_bool(args[5]), m, off, as_ptr(args[9]), as_ptr(args[10]),
                                     (const float*)as_ptr(args[11]), (int)as_int(args[12]), as_int(args[13]), n,
                                     as_int(args[7]), swiglu, (float)as_float(args[16]), wp, y.data_ptr(), dt, ld,
                                     current_stream(buf));
  return rc != SB_OK ? status(rc) : THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// topk(logits, k, bias, score, n_group, topk_group, group_score, renormalize, scale) -> (weights, ids) | status
PyObject* topk(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count("topk", nargs, 9);
  Tensor l = tensor(args[0], "topk");
  const int dt = dtype_code(l.scalar_type());
  if (dt < 0 || !l.is_cuda() || l.dim() != 2) REFUSE("topk: logits must be a CUDA tensor [T, E] of bf16, fp16 or fp32");
  const int64_t t = l.size(0), e = l.size(1);
  const int k = as_c_int(args[1]);
  const Tensor* bias = optional(args[2], "topk");
  const float* bp = bias ? float_values("topk", "bias", l, *bias, e) : nullptr;
  if (e > 1 && l.stride(1) != 1) l = l.contiguous();
  const int64_t room = k < 0 || k > e ? 0 : k;   // (the entry refuses such k)
  Tensor w = empty({t, room}, at::kFloat, l), ids = empty({t, room}, at::kLong, l);
  const int rc = sb_route_topk(l.data_ptr(), dt, t, e, t > 1 ? l.stride(0) : e, bp, k, as_c_int(args[3]),
                               as_c_int(args[4]), as_c_int(args[5]), as_c_int(args[6]), as_bool(args[7]),
                               (float)as_float(args[8]), w.data_ptr<float>(), ids.data_ptr<int64_t>(), current_stream(l));
  if (rc != SB_OK) return status(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(w)), THPVariable_Wrap(std::move(ids)));
  END_HANDLE_TH_ERRORS
}

// expert_order(ids, n_experts) -> (offsets, tokens, places) | status
PyObject* expert_order(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count("expert_order", nargs, 2);
  const Tensor& ids = tensor(args[0], "expert_order");
  if (!ids.is_cuda() || ids.scalar_type() != at::kLong || ids.dim() != 2 || !ids.is_contiguous() || ids.size(1) < 1)
    REFUSE("expert_order: indices must be a contiguous CUDA int64 tensor [T, k]");
  const int64_t t = ids.size(0), k = ids.size(1), pairs = t * k, e = as_int(args[1]);
  const size_t need = sb_expert_order_workspace_bytes(pairs, e);   // (0 for an e that the entry refuses; e <= 1024)
  Tensor offsets = empty({e < 0 || e > 1024 ? 0 : e + 1}, at::kInt, ids), tokens = empty({pairs}, at::kInt, ids), places = empty({t, k}, at::kInt, ids);
  Tensor ws;
  if (need) ws = empty({(int64_t)need}, at::kByte, ids);
  const int rc = sb_expert_order(ids.data_ptr<int64_t>(), t, k > INT32_MAX ? 0 : (int)k, e, offsets.data_ptr<int32_t>(), tokens.data_ptr<int32_t>(),
                                 places.data_ptr<int32_t>(), need ? ws.data_ptr() : nullptr, need, current_stream(ids));
  if (rc != SB_OK) return status(rc);
  return Py_BuildValue("(NNN)", THPVariable_Wrap(std::move(offsets)), THPVariable_Wrap(std::move(tokens)),
                       THPVariable_Wrap(std::move(places)));
  END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(quant), METHOD(dequant), METHOD(gemm), METHOD(grouped_gemm), METHOD(topk),
                         METHOD(expert_order), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", "Host calls of shard_b200.fp4 and shard_b200.route.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&module); }
