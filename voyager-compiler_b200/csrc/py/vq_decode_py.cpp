// Python binding of the cached-decoding operators: argument checks, output
// allocation and the C ABI call in one native function each.
//
// A decoding step's calls take 2 - 10 us on the device; checked and called from
// Python through ctypes they took 13 us on the host, here 4.  The functions
// have positional arguments only; voyager_b200.fp8block and
// voyager_b200.kvcache give them their documented form.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <map>
#include <mutex>

#include "voyager_b200.h"

namespace {

using at::Tensor;
constexpr int64_t BLOCK = 128;
PyObject* g_check = nullptr;  // voyager_b200._lib.check(status, what)

Tensor tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
  return THPVariable_Unpack(o);
}
Tensor optional(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor(o, name); }

bool failed(int status, const char* what) {
  if (status == 0) return false;
  PyObject* r = PyObject_CallFunction(g_check, "is", status, what);
  Py_XDECREF(r);
  if (r) PyErr_Format(PyExc_RuntimeError, "%s: status %d", what, status);
  return true;
}

int float_code(at::ScalarType t) {
  return t == at::kBFloat16 ? VQ_BF16 : t == at::kFloat ? VQ_F32 : -1;
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// An output on t's device, past the dispatcher (which takes 0.4 us a tensor).
Tensor output(at::IntArrayRef sizes, at::ScalarType type, const Tensor& t) {
  return Tensor(at::detail::empty_cuda(sizes, type, t.device(), std::nullopt));
}

// The operators have no derivative.  Where one of `in` wants a gradient, a
// backward pass that reaches one of `out` raises instead of ending there.
void no_derivative(const char* what, std::initializer_list<const Tensor*> in, std::initializer_list<Tensor*> out) {
  if (!at::GradMode::is_enabled()) return;
  torch::autograd::edge_list edges;
  for (const Tensor* t : in)
    if (t->defined() && t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
  if (edges.empty()) return;
  const std::shared_ptr<torch::autograd::Node> fn(new torch::autograd::NotImplemented(what, std::move(edges)),
                                                  torch::autograd::deleteNode);
  for (Tensor* t : out)
    if (t->defined()) torch::autograd::set_history(*t, fn);
}

// Makes the tensor's device current where it is not.
struct On {
  c10::cuda::OptionalCUDAGuard guard;
  explicit On(const Tensor& t) {
    if (c10::cuda::current_device() != t.get_device()) guard.set_device(t.device());
  }
};

// t as [rows, cols] with dense rows that do not overlap (an expanded tensor's
// do): itself, a view, or a copy.
Tensor rows_of(const Tensor& t, int64_t cols) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, cols});
  const bool dense = r.stride(1) == 1 || cols == 1;
  return dense && (r.size(0) <= 1 || r.stride(0) >= cols) ? r : r.contiguous();
}

// x, residual or None, weight or None, eps, what -> (codes, scale, hidden or None)
PyObject* norm_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 5, "norm_quantize takes 5 arguments");
  const char* what = PyUnicode_AsUTF8(args[4]);
  const double eps = PyFloat_AsDouble(args[3]);
  if (!what || PyErr_Occurred()) return nullptr;
  const Tensor x = tensor(args[0], "x");
  Tensor residual = optional(args[1], "residual"), weight = optional(args[2], "weight"), hidden;
  const int code = float_code(x.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(code >= 0, what, ": bfloat16 or float32, not ", x.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(x.is_cuda(), what, ": the CUDA kernel needs CUDA tensors");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) > 0, what,
                    ": x needs a last dimension to normalise, got ", x.sizes());
  const int64_t cols = x.size(-1);
  On on(x);
  const Tensor x2 = rows_of(x, cols);
  const int64_t rows = x2.size(0), ldx = std::max(x2.stride(0), cols);
  int64_t ldr = 0;
  if (weight.defined()) {
    TORCH_CHECK_VALUE(weight.scalar_type() == x.scalar_type() && weight.device() == x.device() &&
                          weight.dim() == 1 && weight.size(0) == cols,
                      what, ": weight must be ", x.scalar_type(), " [", cols, "] on ", x.device());
    weight = weight.contiguous();
  }
  if (residual.defined()) {
    TORCH_CHECK_VALUE(residual.scalar_type() == x.scalar_type() && residual.device() == x.device() &&
                          residual.sizes() == x.sizes(),
                      what, ": residual must be ", x.scalar_type(), " ", x.sizes(), " on ", x.device());
    residual = rows_of(residual, cols);
    ldr = std::max(residual.stride(0), cols);
    hidden = output(x.sizes(), x.scalar_type(), x);
  }
  c10::SmallVector<int64_t, 6> ss(x.sizes().begin(), x.sizes().end());
  ss.back() = (cols + BLOCK - 1) / BLOCK;
  Tensor codes = output(x.sizes(), at::kFloat8_e4m3fn, x);
  Tensor scale = output(ss, at::kFloat, x);
  const int st = vq_norm_quantize_fp8(x2.data_ptr(), ldx, ptr(residual), ldr, ptr(weight), code, rows, cols,
                                      (float)eps, codes.data_ptr(), scale.data_ptr<float>(), ptr(hidden),
                                      stream_of(x));
  if (failed(st, what)) return nullptr;
  no_derivative(what, {&x, &residual, &weight}, {&codes, &scale, &hidden});
  PyObject* out = PyTuple_New(3);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(codes)));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(scale)));
  if (hidden.defined()) {
    PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(hidden)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(out, 2, Py_None);
  }
  return out;
  END_HANDLE_TH_ERRORS
}

// codes, scale, w_codes, w_scale, bias or None -> out
PyObject* linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "fp8block.linear";
  TORCH_CHECK_TYPE(n == 5, "linear takes 5 arguments");
  Tensor c = tensor(args[0], "codes"), s = tensor(args[1], "scale"), w = tensor(args[2], "w_codes"),
         ws = tensor(args[3], "w_scale"), bias = optional(args[4], "bias");
  TORCH_CHECK_NOT_IMPLEMENTED(c.scalar_type() == at::kFloat8_e4m3fn && w.scalar_type() == at::kFloat8_e4m3fn,
                              what, " takes float8_e4m3fn codes");
  TORCH_CHECK_NOT_IMPLEMENTED(s.scalar_type() == at::kFloat && ws.scalar_type() == at::kFloat, what,
                              " takes float32 scales");
  TORCH_CHECK_NOT_IMPLEMENTED(c.is_cuda(), what, ": the CUDA kernel needs CUDA tensors");
  TORCH_CHECK_VALUE(w.dim() == 2 && c.dim() >= 1 && c.size(-1) == w.size(1), what, ": ", c.sizes(),
                    " does not match a weight [N, K] ", w.sizes());
  const int64_t N = w.size(0), K = w.size(1);
  TORCH_CHECK_VALUE(K > 0 && K % 16 == 0 && N > 0, what, ": K = ", K,
                    " must be a positive multiple of 16 and N = ", N, " positive");
  const int64_t nk = (K + BLOCK - 1) / BLOCK, lead = c.dim() - 1;
  TORCH_CHECK_VALUE(s.dim() == c.dim() && s.size(-1) == nk && s.sizes().slice(0, lead) == c.sizes().slice(0, lead) &&
                        ws.dim() == 2 && ws.size(0) == (N + BLOCK - 1) / BLOCK && ws.size(1) == nk,
                    what, ": scales ", s.sizes(), " and ", ws.sizes(),
                    " are not one per 128 columns and one per 128 x 128 block");
  const auto dev = c.device();
  TORCH_CHECK_VALUE(s.device() == dev && w.device() == dev && ws.device() == dev, what,
                    ": operands on different devices");
  On on(c);
  if (bias.defined()) {
    TORCH_CHECK_VALUE(bias.scalar_type() == at::kBFloat16 && bias.dim() == 1 && bias.size(0) == N &&
                          bias.device() == dev,
                      what, ": bias must be bfloat16 [", N, "] on ", dev);
    bias = bias.contiguous();
  }
  c = c.contiguous(), s = s.contiguous(), w = w.contiguous(), ws = ws.contiguous();
  c10::SmallVector<int64_t, 6> os(c.sizes().begin(), c.sizes().end());
  os.back() = N;
  Tensor out = output(os, at::kBFloat16, c);
  const int st = vq_linear_fp8_block(c.data_ptr(), s.data_ptr<float>(), w.data_ptr(), ws.data_ptr<float>(),
                                     ptr(bias), c.numel() / K, N, K, out.data_ptr(), N, stream_of(c));
  if (failed(st, what)) return nullptr;
  no_derivative(what, {&c, &s, &w, &ws, &bias}, {&out});
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

struct Cache {
  Tensor kc, vc, ks, vs;
  int64_t pages, heads, page, dim;
  // args: k_codes, v_codes, k_scale, v_scale
  Cache(PyObject* const* a, const char* what)
      : kc(tensor(a[0], "k_codes")), vc(tensor(a[1], "v_codes")), ks(tensor(a[2], "k_scale")),
        vs(tensor(a[3], "v_scale")) {
    TORCH_CHECK_NOT_IMPLEMENTED(kc.scalar_type() == at::kFloat8_e4m3fn && vc.scalar_type() == at::kFloat8_e4m3fn &&
                                    ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat,
                                what, ": a cache is float8_e4m3fn codes and float32 scales");
    TORCH_CHECK_VALUE(kc.dim() == 4 && vc.sizes() == kc.sizes() && ks.sizes() == kc.sizes().slice(0, 2) &&
                          vs.sizes() == ks.sizes(),
                      what, ": cache codes ", kc.sizes(), ", ", vc.sizes(), " and scales ", ks.sizes(), ", ",
                      vs.sizes(), " are not one cache");
    pages = kc.size(0), heads = kc.size(1), page = kc.size(2), dim = kc.size(3);
    TORCH_CHECK_NOT_IMPLEMENTED((page == 32 || page == 64 || page == 128) && (dim == 64 || dim == 128), what,
                                ": page in (32, 64, 128) and head_dim in (64, 128), not ", page, " and ", dim);
    TORCH_CHECK_VALUE(kc.is_contiguous() && vc.is_contiguous() && ks.is_contiguous() && vs.is_contiguous(), what,
                      ": the cache's tensors must be contiguous");
    TORCH_CHECK_VALUE(vc.device() == kc.device() && ks.device() == kc.device() && vs.device() == kc.device(), what,
                      ": the cache's tensors are on different devices");
  }
};

// block_table, lengths, counts or None; their values stay on the device.
struct Plan {
  Tensor table, lengths, counts;
  Plan(PyObject* const* a, const char* what, int64_t B, const at::Device& dev)
      : table(tensor(a[0], "block_table")), lengths(tensor(a[1], "lengths")), counts(optional(a[2], "counts")) {
    one(table, "block_table", 2, what, B, dev);
    one(lengths, "lengths", 1, what, B, dev);
    if (counts.defined()) one(counts, "counts", 1, what, B, dev);
  }
  static void one(const Tensor& t, const char* name, int64_t dim, const char* what, int64_t B, const at::Device& dev) {
    TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == dim && t.size(0) == B && t.device() == dev &&
                          t.is_contiguous(),
                      what, ": ", name, " must be contiguous int32 with ", dim, " dimension(s), the first ", B,
                      ", on ", dev);
  }
};

// t [B, T, H, D] with a dense last dim and 16-byte rows, itself or a copy.
Tensor heads_of(const Tensor& t) {
  const int64_t eb = t.element_size();
  if (t.stride(3) == 1 &&
      (((int64_t)(uintptr_t)t.data_ptr() | t.stride(0) * eb | t.stride(1) * eb | t.stride(2) * eb) & 15) == 0)
    return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

// q, k, v, table, k_codes, v_codes, k_scale, v_scale, block_table, lengths,
// counts or None, interleaved -> q turned
PyObject* rope_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "rope_append";
  TORCH_CHECK_TYPE(n == 12, "rope_append takes 12 arguments");
  Tensor q = tensor(args[0], "q"), k = tensor(args[1], "k"), v = tensor(args[2], "v");
  const Tensor table = tensor(args[3], "table");
  const int interleaved = PyObject_IsTrue(args[11]);
  if (interleaved < 0) return nullptr;
  const int code = float_code(q.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(code >= 0 && k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type(),
                              what, ": q, k and v of one type, bfloat16 or float32");
  TORCH_CHECK_NOT_IMPLEMENTED(q.is_cuda(), what, ": the CUDA kernel needs CUDA tensors");
  const Cache c(args + 4, what);
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == c.dim && k.dim() == 4 && k.size(0) == q.size(0) &&
                        k.size(1) == q.size(1) && k.size(2) == c.heads && k.size(3) == c.dim && v.sizes() == k.sizes(),
                    what, ": q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes(), " do not match a cache of ",
                    c.heads, " heads of ", c.dim);
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2);
  TORCH_CHECK_VALUE(H > 0 && c.heads > 0 && H % c.heads == 0, what, ": ", H, " query heads do not group over ", c.heads, " kv heads");
  TORCH_CHECK_VALUE(table.scalar_type() == at::kFloat && table.dim() == 3 && table.size(2) == 2 && table.is_contiguous(),
                    what, ": table must be contiguous float32 [positions, rotary_dim / 2, 2]");
  const int64_t rot = 2 * table.size(1);
  TORCH_CHECK_VALUE(rot > 0 && rot % 16 == 0 && rot <= c.dim, what, ": rotary_dim = ", rot,
                    " must be a multiple of 16 up to ", c.dim);
  const auto dev = c.kc.device();
  TORCH_CHECK_VALUE(q.device() == dev && k.device() == dev && v.device() == dev && table.device() == dev, what,
                    ": operands on different devices");
  const Plan plan(args + 8, what, B, dev);
  const int64_t width = plan.table.size(1);
  TORCH_CHECK_VALUE(table.size(0) >= width * c.page, what, ": the table's ", table.size(0),
                    " positions do not cover the block table's ", width * c.page, " tokens");
  On on(q);
  q = heads_of(q), k = heads_of(k), v = heads_of(v);
  Tensor out = output({B, T, H, c.dim}, q.scalar_type(), q);
  const int64_t strides[9] = {q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1),
                              k.stride(2), v.stride(0), v.stride(1), v.stride(2)};
  const int st = vq_rope_append_kv8(
      q.data_ptr(), k.data_ptr(), v.data_ptr(), strides, code, table.data_ptr<float>(), table.size(0), (int)rot,
      interleaved, B, T, (int)H, (int)c.heads, (int)c.dim, plan.table.data_ptr(), width, plan.lengths.data_ptr(),
      ptr(plan.counts), c.pages, (int)c.page, out.data_ptr(), c.kc.data_ptr(), c.vc.data_ptr(),
      c.ks.data_ptr<float>(), c.vs.data_ptr<float>(), stream_of(q));
  if (failed(st, what)) return nullptr;
  no_derivative(what, {&q, &k, &v, &table}, {&out});
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// Zeroed counters for a call on the current stream; each call leaves them
// zero, and calls on one stream do not overlap, so they share them.  A
// captured call gets its own, which live and die with its graph; so does a call
// on the per-thread default stream, whose one handle names a stream of its own
// in every thread.  The map is never destroyed: the tensors outlive the CUDA
// context's end at exit.
Tensor join_counters(const Tensor& q, int64_t n) {
  const auto opt = q.options().dtype(at::kInt);
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None ||
      stream_of(q) == cudaStreamPerThread)
    return at::zeros({n}, opt);
  static std::mutex m;
  static auto* kept = new std::map<std::pair<int, void*>, Tensor>();
  std::lock_guard<std::mutex> lock(m);
  Tensor& t = (*kept)[{q.get_device(), stream_of(q)}];
  if (!t.defined() || t.numel() < n) t = at::zeros({std::max<int64_t>(n, 1024)}, opt);
  return t;
}

// q, k_codes, v_codes, k_scale, v_scale, block_table, lengths, counts or
// None, scale or None -> out
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* what = "attend";
  TORCH_CHECK_TYPE(n == 9, "attend takes 9 arguments");
  Tensor q = tensor(args[0], "q");
  TORCH_CHECK_NOT_IMPLEMENTED(q.scalar_type() == at::kBFloat16, what, ": q must be bfloat16, not ", q.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(q.is_cuda(), what, ": the CUDA kernel needs CUDA tensors");
  const Cache c(args + 1, what);
  TORCH_CHECK_VALUE(q.dim() == 4 && q.size(3) == c.dim && q.size(2) > 0 && c.heads > 0 && q.size(2) % c.heads == 0,
                    what, ": q ", q.sizes(), " does not match a cache of ", c.heads, " heads of ", c.dim);
  TORCH_CHECK_VALUE(q.device() == c.kc.device(), what, ": operands on different devices");
  const int64_t B = q.size(0), T = q.size(1), H = q.size(2);
  const Plan plan(args + 5, what, B, q.device());
  const double scale = args[8] == Py_None ? 1.0 / std::sqrt((double)c.dim) : PyFloat_AsDouble(args[8]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t width = plan.table.size(1);
  On on(q);
  q = heads_of(q);
  Tensor out = output({B, T, H, c.dim}, q.scalar_type(), q);
  int64_t floats = 0, counters = 0;
  if (failed(vq_attn_kv8_workspace(B, T, (int)H, (int)c.heads, (int)c.dim, (int)c.page, width, &floats, &counters),
             what))
    return nullptr;
  const Tensor done = join_counters(q, counters);
  const Tensor part = output({floats}, at::kFloat, q);
  const int64_t strides[3] = {q.stride(0), q.stride(1), q.stride(2)};
  const int st = vq_attn_kv8(q.data_ptr(), strides, B, T, (int)H, (int)c.heads, (int)c.dim, c.kc.data_ptr(),
                             c.vc.data_ptr(), c.ks.data_ptr<float>(), c.vs.data_ptr<float>(), c.pages, (int)c.page,
                             plan.table.data_ptr(), width, plan.lengths.data_ptr(), ptr(plan.counts), (float)scale,
                             part.data_ptr<float>(), floats, done.data_ptr<int>(), done.numel(), out.data_ptr(),
                             stream_of(q));
  if (failed(st, what)) return nullptr;
  no_derivative(what, {&q, &c.kc, &c.vc, &c.ks, &c.vs}, {&out});
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyObject* bind(PyObject*, PyObject* check) {
  Py_INCREF(check);
  Py_XSETREF(g_check, check);
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"bind", bind, METH_O, "bind(check): the function that raises a status"},
    {"norm_quantize", (PyCFunction)(void (*)(void))norm_quantize, METH_FASTCALL, nullptr},
    {"linear", (PyCFunction)(void (*)(void))linear, METH_FASTCALL, nullptr},
    {"rope_append", (PyCFunction)(void (*)(void))rope_append, METH_FASTCALL, nullptr},
    {"attend", (PyCFunction)(void (*)(void))attend, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_decode", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decode(void) { return PyModule_Create(&kModule); }
