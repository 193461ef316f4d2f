// CPython binding of the device-pointer operators (fa_dev_*) for torch tensors.
//
// Reads the tensors' addresses, shapes and strides, checks that they fit
// together and lie on the backend's device, and makes the C call.  The smallest
// operators take a few microseconds on the GPU; the same checks written in
// Python took twelve on the host.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "../../include/funasr_cuda.h"

namespace {

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};

[[noreturn]] void refuse(const char* name, const std::string& what) { throw Refused(std::string(name) + ": " + what); }

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(name, "expected a torch tensor");
  return THPVariable_Unpack(o);
}

// Tells autograd that a call has overwritten an output, as torch's own in-place operations do.
void written(PyObject* o) {
  if (o == Py_None) return;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int dtype_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return FA_DTYPE_F32;
    case at::kHalf: return FA_DTYPE_F16;
    case at::kBFloat16: return FA_DTYPE_BF16;
    default: refuse(name, "expected float32, float16 or bfloat16");
  }
}

void on_device(const at::Tensor& t, int device, const char* name) {
  if (!t.is_cuda() || t.get_device() != device)
    refuse(name, "on " + t.device().str() + ", not on the backend's device cuda:" + std::to_string(device));
}

std::string text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

// A strided tensor of `like`'s type and of `shape`, innermost dimension
// contiguous; the other strides go to `strides`.
void* rows(const at::Tensor& t, const at::Tensor& like, at::IntArrayRef shape, int device, int64_t* strides,
           const char* name) {
  if (t.scalar_type() != like.scalar_type()) refuse(name, "its type differs from the first tensor's");
  if (t.sizes() != shape) refuse(name, "expected shape " + text(shape) + ", got " + text(t.sizes()));
  const at::IntArrayRef st = t.strides();
  const size_t n = shape.size();
  if (st[n - 1] != 1 && shape[n - 1] > 1) refuse(name, "the innermost dimension must be contiguous");
  for (size_t i = 0; i + 1 < n; ++i) strides[i] = st[i];
  on_device(t, device, name);
  return t.data_ptr();
}

// A contiguous tensor of `type` with `count` elements (any number: -1); None gives null.
template <typename T>
T* flat(PyObject* o, at::ScalarType type, int64_t count, int device, const char* name) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type) refuse(name, std::string("expected ") + at::toString(type));
  if (!t.is_contiguous()) refuse(name, "not contiguous");
  if (count >= 0 && t.numel() != count)
    refuse(name, "expected " + std::to_string(count) + " elements, got " + std::to_string(t.numel()));
  on_device(t, device, name);
  return static_cast<T*>(t.data_ptr());
}

int64_t numel(PyObject* o, const char* name) { return o == Py_None ? 0 : tensor(o, name).numel(); }

void* workspace(PyObject* o, int device, int64_t* bytes) {
  *bytes = 0;
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, "workspace");
  if (!t.is_contiguous()) refuse("workspace", "not contiguous");
  on_device(t, device, "workspace");
  *bytes = (int64_t)t.nbytes();
  return t.data_ptr();
}

int small(int64_t n, const char* name) {
  if (n > INT32_MAX) refuse(name, "too long");
  return (int)n;
}

struct Call {  // the arguments that every function starts with, and the stream it ends with
  fa_backend* backend;
  int device;
  void* stream;
  Call(PyObject* const* args, Py_ssize_t n) {
    backend = static_cast<fa_backend*>(PyLong_AsVoidPtr(args[0]));
    device = (int)PyLong_AsLong(args[1]);
    // 0 is torch's default stream, which the C ABI names cudaStreamLegacy (1):
    // its null selects the backend's own stream.
    PyObject* s = args[n - 1];
    stream = s == Py_None ? nullptr : PyLong_AsVoidPtr(s);
    if (s != Py_None && stream == nullptr) stream = reinterpret_cast<void*>(1);
    if (PyErr_Occurred()) throw Refused("");
    // Autograd would take the outputs for constants.
    if (!at::GradMode::is_enabled()) return;
    for (Py_ssize_t i = 2; i < n; ++i)
      if (THPVariable_Check(args[i]) && THPVariable_Unpack(args[i]).requires_grad())
        throw Refused("a tensor requires grad, but this operator has no backward pass: call it under torch.no_grad() or "
                      "detach the tensor");
  }
};

float scale_of(PyObject* o, int64_t head_size) {
  if (o == Py_None) return (float)(1.0 / std::sqrt((double)head_size));
  const double v = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) throw Refused("");
  return (float)v;
}

template <typename F>
PyObject* guarded(Py_ssize_t n, Py_ssize_t expected, F&& f) {
  if (n != expected) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return PyLong_FromLong(f());
  } catch (const Refused& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

template <typename Args>
int enqueue(int (*fn)(fa_backend*, const Args*, void*), const Call& c, const Args& a,
            std::initializer_list<PyObject*> outputs) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = fn(c.backend, &a, c.stream);
  Py_END_ALLOW_THREADS
  if (rc == FA_OK)
    for (PyObject* o : outputs) written(o);
  return rc;
}

// backend, device, q, k, v, q_offsets, k_offsets, out, causal, scale, lse, workspace, stream
PyObject* attention_packed(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 13, [&] {
    const Call c(args, n);
    const at::Tensor &q = tensor(args[2], "q"), &k = tensor(args[3], "k"), &off = tensor(args[5], "q_offsets");
    if (q.dim() != 3 || k.dim() != 3) refuse("q, k", "expected three dimensions");
    fa_attention_packed_args a{};
    a.dtype = dtype_of(q, "q");
    const int64_t heads = q.size(1), size = q.size(2), kv_heads = k.size(1), sequences = off.numel() - 1;
    if (k.size(2) != size) refuse("k", "its head size differs from q's");
    if (sequences < 0) refuse("q_offsets", "empty");
    a.q = rows(q, q, q.sizes(), c.device, a.q_stride, "q");
    a.k = rows(k, q, k.sizes(), c.device, a.k_stride, "k");
    a.v = rows(tensor(args[4], "v"), q, k.sizes(), c.device, a.v_stride, "v");
    a.out = rows(tensor(args[7], "out"), q, q.sizes(), c.device, a.out_stride, "out");
    a.total_q = q.size(0);
    a.total_k = k.size(0);
    a.q_offsets = flat<int32_t>(args[5], at::kInt, sequences + 1, c.device, "q_offsets");
    a.k_offsets = flat<int32_t>(args[6], at::kInt, sequences + 1, c.device, "k_offsets");
    a.lse = flat<float>(args[10], at::kFloat, a.total_q * heads, c.device, "lse");
    a.workspace = workspace(args[11], c.device, &a.workspace_bytes);
    a.sequences = small(sequences, "q_offsets");
    a.heads = small(heads, "q");
    a.kv_heads = small(kv_heads, "k");
    a.head_size = small(size, "q");
    const int causal = PyObject_IsTrue(args[8]);
    if (causal < 0) throw Refused("");
    a.causal = causal;
    a.scale = scale_of(args[9], size);
    return enqueue(fa_dev_attention_packed, c, a, {args[7], args[10]});
  });
}

// backend, device, q, prefix_k, prefix_v, suffix_k, suffix_v, suffix_lens, out, scale, lse, workspace, stream
PyObject* attention_shared(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 13, [&] {
    const Call c(args, n);
    const at::Tensor &q = tensor(args[2], "q"), &pk = tensor(args[3], "prefix_k"), &sk = tensor(args[5], "suffix_k");
    if (q.dim() != 3 || pk.dim() != 3) refuse("q, prefix_k", "expected three dimensions");
    if (sk.dim() != 4) refuse("suffix_k", "expected four dimensions");
    fa_attention_shared_args a{};
    a.dtype = dtype_of(q, "q");
    const int64_t sequences = q.size(0), heads = q.size(1), size = q.size(2), kv_heads = pk.size(1);
    if (pk.size(2) != size) refuse("prefix_k", "its head size differs from q's");
    if (sk.size(0) != sequences || sk.size(2) != kv_heads || sk.size(3) != size)
      refuse("suffix_k", "expected (sequences, capacity, kv_heads, head size), got " + text(sk.sizes()));
    a.q = rows(q, q, q.sizes(), c.device, a.q_stride, "q");
    a.prefix_k = rows(pk, q, pk.sizes(), c.device, a.prefix_k_stride, "prefix_k");
    a.prefix_v = rows(tensor(args[4], "prefix_v"), q, pk.sizes(), c.device, a.prefix_v_stride, "prefix_v");
    a.suffix_k = rows(sk, q, sk.sizes(), c.device, a.suffix_k_stride, "suffix_k");
    a.suffix_v = rows(tensor(args[6], "suffix_v"), q, sk.sizes(), c.device, a.suffix_v_stride, "suffix_v");
    a.out = rows(tensor(args[8], "out"), q, q.sizes(), c.device, a.out_stride, "out");
    a.suffix_lens = flat<int32_t>(args[7], at::kInt, sequences, c.device, "suffix_lens");
    a.lse = flat<float>(args[10], at::kFloat, sequences * heads, c.device, "lse");
    a.workspace = workspace(args[11], c.device, &a.workspace_bytes);
    a.prefix_len = pk.size(0);
    a.suffix_capacity = sk.size(1);
    a.sequences = small(sequences, "q");
    a.heads = small(heads, "q");
    a.kv_heads = small(kv_heads, "prefix_k");
    a.head_size = small(size, "q");
    a.scale = scale_of(args[9], size);
    return enqueue(fa_dev_attention_shared, c, a, {args[8], args[10]});
  });
}

// backend, device, logits, out, tokens, history, history_offsets, prompt_lens, repetition, presence, frequency,
// bias_tokens, bias_values, bias_offsets, mask, mask_rows, stream
PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 17, [&] {
    const Call c(args, n);
    const at::Tensor& x = tensor(args[2], "logits");
    if (x.dim() != 2) refuse("logits", "expected two dimensions");
    fa_logits_args a{};
    a.dtype = dtype_of(x, "logits");
    const int64_t count = x.size(0), vocab = x.size(1);
    a.logits = rows(x, x, x.sizes(), c.device, &a.logits_stride, "logits");
    a.out = rows(tensor(args[3], "out"), x, x.sizes(), c.device, &a.out_stride, "out");
    a.tokens = flat<int32_t>(args[4], at::kInt, count, c.device, "tokens");
    if ((args[5] == Py_None) != (args[6] == Py_None)) refuse("history", "comes with history_offsets");
    if ((args[11] == Py_None) != (args[12] == Py_None) || (args[11] == Py_None) != (args[13] == Py_None))
      refuse("bias_tokens", "comes with bias_values and bias_offsets");
    a.history_total = numel(args[5], "history");
    a.bias_total = numel(args[11], "bias_tokens");
    a.history = flat<int32_t>(args[5], at::kInt, -1, c.device, "history");
    a.history_offsets = flat<int32_t>(args[6], at::kInt, count + 1, c.device, "history_offsets");
    a.prompt_lens = flat<int32_t>(args[7], at::kInt, count, c.device, "prompt_lens");
    a.repetition = flat<float>(args[8], at::kFloat, count, c.device, "repetition");
    a.presence = flat<float>(args[9], at::kFloat, count, c.device, "presence");
    a.frequency = flat<float>(args[10], at::kFloat, count, c.device, "frequency");
    a.bias_tokens = flat<int32_t>(args[11], at::kInt, -1, c.device, "bias_tokens");
    a.bias_values = flat<float>(args[12], at::kFloat, a.bias_total, c.device, "bias_values");
    a.bias_offsets = flat<int32_t>(args[13], at::kInt, count + 1, c.device, "bias_offsets");
    if (args[14] != Py_None) {
      const at::Tensor& m = tensor(args[14], "mask");
      if (m.dim() != 2 || m.size(1) != (vocab + 31) / 32 ||
          (m.scalar_type() != at::kInt && m.scalar_type() != at::kUInt32))
        refuse("mask", "expected 32-bit words [masks, ceil(vocab / 32)]");
      a.mask = static_cast<const uint32_t*>(rows(m, m, m.sizes(), c.device, &a.mask_stride, "mask"));
      a.mask_count = small(m.size(0), "mask");
    }
    a.mask_rows = flat<int32_t>(args[15], at::kInt, count, c.device, "mask_rows");
    a.rows = small(count, "logits");
    a.vocab = small(vocab, "logits");
    return enqueue(fa_dev_adjust_logits, c, a, {args[3], args[4]});
  });
}

#define FA_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FA_METHOD(attention_packed), FA_METHOD(attention_shared), FA_METHOD(adjust_logits),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops() { return PyModule_Create(&module); }
