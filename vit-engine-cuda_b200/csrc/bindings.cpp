// Python entry points of the serving operators (vit_cuda._serving): argument
// checks, output allocation and the call into libvitb200.so.
//
// One eager call through Python code and ctypes took 10-12 us on the host
// against 3-6 us on the GPU for a single token's step; these functions take
// their arguments by position from the interpreter's own vector and spend 4-5
// us, most of it the launch itself. The package opens libvitb200.so (ctypes) and
// hands the entry points' addresses to `bind`, so this module links only
// PyTorch.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/DispatchKeySet.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include "vitb200.h"

namespace {

constexpr int64_t kBlock = 128;  // columns (and, for weights, rows) that share one scale

struct Library {
  decltype(&vitb200_quantize_fp8) quantize = nullptr;
  decltype(&vitb200_layernorm_fp8) layernorm = nullptr;
  decltype(&vitb200_gemm_fp8) gemm = nullptr;
  decltype(&vitb200_cross_attention) attention = nullptr;
  decltype(&vitb200_cross_attention_workspace_bytes) attention_workspace = nullptr;
  PyObject* error = nullptr;  // raise_status(what, status)
} g_lib;

const at::Tensor& tensor_arg(PyObject* o, const char* op) {
  TORCH_CHECK(THPVariable_Check(o), op, ": all inputs must be CUDA tensors");
  return THPVariable_Unpack(o);
}

// The current device, after checking that every tensor given is on it.
c10::DeviceIndex on_device(const char* op, std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    TORCH_CHECK(!t || t->is_cuda(), op, ": all inputs must be CUDA tensors");
  const c10::DeviceIndex device = (*tensors.begin())->get_device();
  for (const at::Tensor* t : tensors)
    TORCH_CHECK(!t || t->get_device() == device, op,
                ": all inputs must be on the same CUDA device");
  const c10::DeviceIndex current = c10::cuda::current_device();
  TORCH_CHECK(device == current, op, ": inputs are on device ", int(device),
              " but the current CUDA device is ", int(current),
              " (run torch.cuda.set_device, or move tensors)");
  return device;
}

int type_code(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return VITB200_F32;
    case at::kHalf: return VITB200_F16;
    case at::kBFloat16: return VITB200_BF16;
    default: TORCH_CHECK(false, what, " must be float32, float16 or bfloat16");
  }
}

int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, c10::DeviceIndex device) {
  return at::detail::empty_cuda(sizes, type, at::Device(at::kCUDA, device), std::nullopt);
}

// A tensor read as [rows, last dim]: as it is where one stride (in elements)
// describes the rows, else a contiguous copy. The stride of a dimension of one means
// nothing, so one token of each sequence ([B, 1, K]) goes by its batch stride.
struct Rows {
  at::Tensor t;
  int64_t ld;
};
Rows rows_of(const at::Tensor& t) {
  const int64_t n = t.size(-1);
  if (t.is_contiguous()) return {t, n};
  if (t.stride(-1) == 1) {
    if (t.dim() == 2 && t.stride(0) >= n) return {t, t.stride(0)};
    if (t.dim() == 3) {
      const int64_t ld = t.size(1) == 1 ? t.stride(0) : t.stride(1);
      // (a padded [B, N, K] still has one stride)
      if (ld >= n && (t.size(0) == 1 || t.size(1) == 1 || t.stride(0) == t.size(1) * ld))
        return {t, ld};
    }
  }
  return {t.contiguous(), n};
}

// Empty codes of the given shape, rows a multiple of 16 bytes apart as the
// matrix product's loads need them.
Rows empty_codes(at::IntArrayRef shape, c10::DeviceIndex device) {
  const int64_t n = shape.back();
  const int64_t ld = (n + 15) / 16 * 16;
  if (ld == n) return {empty(shape, at::kFloat8_e4m3fn, device), ld};
  c10::SmallVector<int64_t, 5> padded(shape.begin(), shape.end());
  padded.back() = ld;
  return {empty(padded, at::kFloat8_e4m3fn, device).narrow(-1, 0, n), ld};
}

// rows_of codes, with rows and base aligned to 16 bytes (a padded copy if not).
Rows code_rows(const at::Tensor& q, c10::DeviceIndex device) {
  Rows r = rows_of(q);
  // One row counts as contiguous whatever its stride; nothing past it is read.
  if (q.numel() == q.size(-1)) r.ld = (r.ld + 15) / 16 * 16;
  if (r.ld % 16 == 0 && reinterpret_cast<uintptr_t>(r.t.data_ptr()) % 16 == 0) return r;
  Rows c = empty_codes(q.sizes(), device);
  c.t.view(at::kByte).copy_(q.view(at::kByte));
  return c;
}

void* stream_of(c10::DeviceIndex device) {
  return c10::cuda::getCurrentCUDAStream(device).stream();
}

// Turns a non-zero status into the package's exception; false with it set.
bool passed(int status, const char* what) {
  if (status == 0) return true;
  PyObject* r = PyObject_CallFunction(g_lib.error, "is", status, what);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, what);
  return false;
}

// Whether somebody looks on: a tracer, a dispatch or function mode, a transform
// (vmap, functionalize), or gradients. The functions below read memory behind the
// dispatcher's back, so such a call has to go to the registered operator instead.
bool watched_thread() {
  // BackendSelect and the like are always included, autocast's keys change nothing here
  const c10::DispatchKeySet keys = c10::impl::tls_local_dispatch_key_set().included_ -
                                   c10::default_included_set - c10::autocast_dispatch_keyset;
  return !keys.empty() || c10::impl::dispatch_mode_enabled() ||
         at::impl::torch_function_mode_enabled();
}
bool watched_arg(PyObject* o) {
  if (o == Py_None) return false;
  if (!THPVariable_CheckExact(o)) {  // a subclass or a proxy; anything else is refused later
    return THPVariable_Check(o) || PyObject_HasAttrString(o, "__torch_function__");
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  if (c10::GradMode::is_enabled() && t.requires_grad()) return true;
  TORCH_CHECK(!t._fw_grad(0).defined(), "vit_cuda: forward only, and an input has a tangent");
  // anything but a plain CUDA tensor (CPU tensors are refused later): fakes, wrappers,
  // views with a pending negation
  const c10::DispatchKeySet keys = t.key_set() - c10::autograd_dispatch_keyset_with_ADInplaceOrView -
                                   c10::autocast_dispatch_keyset;
  return keys != c10::DispatchKeySet(c10::DispatchKey::CUDA) &&
         keys != c10::DispatchKeySet(c10::DispatchKey::CPU);
}

// (tensors or None...) -> bool
PyObject* watched(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  bool yes = watched_thread();
  for (Py_ssize_t i = 0; i < n && !yes; ++i) yes = watched_arg(args[i]);
  return PyBool_FromLong(yes);
  END_HANDLE_TH_ERRORS
}

void check_count(Py_ssize_t n, Py_ssize_t want) {
  TORCH_CHECK(n == want && g_lib.gemm, "vit_cuda._serving: wrong call");
}

int64_t int_arg(PyObject* o, const char* what) {
  const int64_t v = PyLong_AsLongLong(o);
  TORCH_CHECK(!(v == -1 && PyErr_Occurred()) || (PyErr_Clear(), false), what,
              " must be an integer");
  return v;
}

float float_arg(PyObject* o, const char* what) {
  const double v = PyFloat_AsDouble(o);
  TORCH_CHECK(!(v == -1.0 && PyErr_Occurred()) || (PyErr_Clear(), false), what,
              " must be a number");
  return static_cast<float>(v);
}

PyObject* pair_of(at::Tensor a, at::Tensor b) {
  PyObject* x = THPVariable_Wrap(std::move(a));
  PyObject* y = THPVariable_Wrap(std::move(b));
  PyObject* t = PyTuple_Pack(2, x, y);
  Py_DECREF(x);
  Py_DECREF(y);
  return t;
}

// Codes and scales of X [..., K], with or without a LayerNorm (gamma != null).
PyObject* quantize(const char* op, const at::Tensor& X, const at::Tensor* gamma,
                   const at::Tensor* beta, float eps, int64_t block_rows) {
  const c10::DeviceIndex device = gamma ? on_device(op, {&X, gamma, beta}) : on_device(op, {&X});
  const int code = type_code(X.scalar_type(), "X");
  TORCH_CHECK(X.dim() >= 1 && X.size(-1) >= 1 && X.size(-1) <= (1 << 30),
              "X must be [..., K] with K >= 1");
  const int64_t K = X.size(-1), M = X.numel() / K;
  TORCH_CHECK(block_rows == 1 || block_rows == kBlock, "block_rows must be 1 or 128");
  TORCH_CHECK(block_rows == 1 || X.dim() == 2, "X must be 2D for 128 x 128 blocks");
  const Rows x = rows_of(X);
  const Rows q = empty_codes(X.sizes(), device);
  c10::SmallVector<int64_t, 5> shape(X.sizes().begin(), X.sizes().end());
  shape.back() = blocks(K);
  if (block_rows != 1) shape[0] = blocks(M);
  at::Tensor scales = empty(shape, at::kFloat, device);
  int st;
  if (gamma) {
    for (auto [t, name] : {std::pair{gamma, "gamma"}, std::pair{beta, "beta"}}) {
      TORCH_CHECK(t->scalar_type() == at::kFloat, name, " must be float32");
      TORCH_CHECK(t->numel() == K, name, " size mismatch");
    }
    const at::Tensor g = gamma->contiguous(), b = beta->contiguous();
    st = g_lib.layernorm(x.t.data_ptr(), code, M, static_cast<int>(K), x.ld,
                         static_cast<const float*>(g.data_ptr()),
                         static_cast<const float*>(b.data_ptr()), eps,
                         static_cast<uint8_t*>(q.t.data_ptr()), q.ld,
                         static_cast<float*>(scales.data_ptr()), stream_of(device));
  } else {
    st = g_lib.quantize(x.t.data_ptr(), code, M, static_cast<int>(K), x.ld,
                        static_cast<int>(block_rows), static_cast<uint8_t*>(q.t.data_ptr()), q.ld,
                        static_cast<float*>(scales.data_ptr()), stream_of(device));
  }
  return passed(st, op) ? pair_of(q.t, std::move(scales)) : nullptr;
}

// (X, block_rows)
PyObject* quantize_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  check_count(n, 2);
  return quantize("quantize_fp8", tensor_arg(args[0], "quantize_fp8"), nullptr, nullptr, 0.f,
                  int_arg(args[1], "block_rows"));
  END_HANDLE_TH_ERRORS
}

// (X, gamma, beta, eps)
PyObject* layernorm_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  check_count(n, 4);
  const char* op = "layernorm_fp8";
  return quantize(op, tensor_arg(args[0], op), &tensor_arg(args[1], op), &tensor_arg(args[2], op),
                  float_arg(args[3], "eps"), 1);
  END_HANDLE_TH_ERRORS
}

// (X, X_scale, W, W_scale, B, residual, gelu, out_dtype)
PyObject* gemm_fp8(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  check_count(n, 8);
  const char* op = "gemm_fp8";
  const at::Tensor &X = tensor_arg(args[0], op), &Xs = tensor_arg(args[1], op),
                   &W = tensor_arg(args[2], op), &Ws = tensor_arg(args[3], op);
  const at::Tensor* B = args[4] == Py_None ? nullptr : &tensor_arg(args[4], op);
  const at::Tensor* R = args[5] == Py_None ? nullptr : &tensor_arg(args[5], op);
  const int gelu = PyObject_IsTrue(args[6]);
  if (gelu < 0) return nullptr;
  TORCH_CHECK(THPDtype_Check(args[7]), "out_dtype must be a torch.dtype");
  const at::ScalarType out_type = reinterpret_cast<THPDtype*>(args[7])->scalar_type;
  const c10::DeviceIndex device = on_device(op, {&X, &Xs, &W, &Ws, B, R});
  TORCH_CHECK(X.scalar_type() == at::kFloat8_e4m3fn && W.scalar_type() == at::kFloat8_e4m3fn,
              "X and W must be float8_e4m3fn");
  TORCH_CHECK(Xs.scalar_type() == at::kFloat && Ws.scalar_type() == at::kFloat,
              "X_scale and W_scale must be float32");
  const int code = type_code(out_type, "out_dtype");
  TORCH_CHECK(X.dim() == 2 || X.dim() == 3, "X must be [N, K] or [B, N, K]");
  TORCH_CHECK(W.dim() == 2, "W must be [N_out, K]");
  const int64_t N = W.size(0), K = W.size(1), kb = blocks(K);
  TORCH_CHECK(K >= 1, "K must be at least 1");
  TORCH_CHECK(X.size(-1) == K, "W second dim must match K");
  c10::SmallVector<int64_t, 5> shape(X.sizes().begin(), X.sizes().end());
  shape.back() = kb;
  TORCH_CHECK(Xs.sizes() == at::IntArrayRef(shape), "X_scale must be [..., ", kb,
              "] (one scale per row and 128 columns)");
  TORCH_CHECK(Ws.dim() == 2 && Ws.size(0) == blocks(N) && Ws.size(1) == kb, "W_scale must be [",
              blocks(N), ", ", kb, "] (one scale per 128 x 128 block)");
  shape.back() = N;
  at::Tensor bias;
  if (B) {
    TORCH_CHECK(B->scalar_type() == at::kFloat, "B must be float32");
    TORCH_CHECK(B->numel() == N, "bias size mismatch");
    bias = B->contiguous();
  }
  Rows r{at::Tensor(), 0};
  if (R) {
    TORCH_CHECK(R->scalar_type() == out_type, "residual must have out_dtype");
    TORCH_CHECK(R->sizes() == at::IntArrayRef(shape), "residual shape mismatch");
    if (N > 0) r = rows_of(*R);
  }
  TORCH_CHECK(N <= INT32_MAX && K <= INT32_MAX, "N_out and K must fit 32 bits");
  const Rows x = code_rows(X, device), w = code_rows(W, device);
  const Rows xs = rows_of(Xs), ws = rows_of(Ws);
  at::Tensor Y = empty(shape, out_type, device);
  const int st = g_lib.gemm(
      static_cast<const uint8_t*>(x.t.data_ptr()), x.ld,
      static_cast<const float*>(xs.t.data_ptr()), xs.ld,
      static_cast<const uint8_t*>(w.t.data_ptr()), w.ld,
      static_cast<const float*>(ws.t.data_ptr()), ws.ld,
      bias.defined() ? static_cast<const float*>(bias.data_ptr()) : nullptr,
      r.t.defined() ? r.t.data_ptr() : nullptr, r.ld, Y.data_ptr(), N, code, X.numel() / K,
      static_cast<int>(K), static_cast<int>(N), gelu, stream_of(device));
  return passed(st, op) ? THPVariable_Wrap(std::move(Y)) : nullptr;
  END_HANDLE_TH_ERRORS
}

// A [B, N, E] operand of the attention, strides in elements: as it is where rows
// are contiguous and everything is 16-byte aligned, else a copy.
struct Operand {
  at::Tensor t;
  int64_t row, batch;
};
Operand operand(const at::Tensor& t, bool shared) {
  const int64_t B = t.size(0), N = t.size(1), E = t.size(2);
  const int64_t row = N > 1 ? t.stride(1) : E;
  const int64_t batch = B > 1 ? t.stride(0) : std::max<int64_t>(N, 1) * row;
  // (a stride of 0 is an expanded batch)
  if (t.stride(2) != 1 || row < E || row % 8 || batch < (shared && batch == 0 ? 0 : E) ||
      batch % 8 ||
      reinterpret_cast<uintptr_t>(t.data_ptr()) % 16)
    return {t.clone(at::MemoryFormat::Contiguous), E, std::max<int64_t>(N, 1) * E};
  return {t, row, batch};
}

// (Q, K, V, scale, heads, kv_heads, kv_lens)
PyObject* cross_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  check_count(n, 7);
  const char* op = "cross_attention";
  const at::Tensor &Q = tensor_arg(args[0], op), &K = tensor_arg(args[1], op),
                   &V = tensor_arg(args[2], op);
  const at::Tensor* L = args[6] == Py_None ? nullptr : &tensor_arg(args[6], op);
  const float scale = float_arg(args[3], "scale");
  const int64_t heads = int_arg(args[4], "heads");
  const int64_t kv_heads = args[5] == Py_None ? heads : int_arg(args[5], "kv_heads");
  const c10::DeviceIndex device = on_device(op, {&Q, &K, &V, L});
  const at::ScalarType type = Q.scalar_type();
  TORCH_CHECK(type == at::kHalf || type == at::kBFloat16,
              "Q must be float16 or bfloat16 (flash_attn_2 takes float32)");
  TORCH_CHECK(K.scalar_type() == type && V.scalar_type() == type,
              "Q, K and V must have the same type");
  TORCH_CHECK(Q.dim() == 3, "Q must be [B, Tq, heads * D]");
  TORCH_CHECK(K.dim() == 3 && K.size(0) == Q.size(0),
              "K must be [B, Tk, kv_heads * D] with Q's B");
  TORCH_CHECK(V.sizes() == K.sizes(), "V shape must match K shape");
  TORCH_CHECK(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0,
              "heads must be a positive multiple of kv_heads");
  const int64_t B = Q.size(0), Tq = Q.size(1), Tk = K.size(1), D = Q.size(2) / heads;
  TORCH_CHECK((D == 64 || D == 128) && Q.size(2) == heads * D,
              "Q's last dim must be heads * D with D 64 or 128");
  TORCH_CHECK(K.size(2) == kv_heads * D, "K's last dim must be kv_heads * D with Q's D");
  TORCH_CHECK(B <= INT32_MAX && Tq <= INT32_MAX && Tk <= INT32_MAX,
              "B, Tq and Tk must fit 32 bits");
  at::Tensor lens;
  if (L) {
    TORCH_CHECK(L->scalar_type() == at::kInt, "kv_lens must be int32");
    TORCH_CHECK(L->dim() == 1 && L->size(0) == B, "kv_lens must be [B]");
    lens = L->contiguous();
  }
  // An expanded batch (beams over one image) is read in place by the forms for up to 128
  // rows per key head; a longer prompt's copy is small next to its work.
  const bool shared = heads / kv_heads * Tq <= 128;
  const Operand q = operand(Q, shared), k = operand(K, shared), v = operand(V, shared);
  at::Tensor O = empty(Q.sizes(), type, device);
  at::Tensor workspace;
  const size_t bytes = g_lib.attention_workspace(
      static_cast<int>(B), static_cast<int>(Tq), static_cast<int>(Tk), static_cast<int>(heads),
      static_cast<int>(kv_heads), static_cast<int>(D));
  if (bytes > 0) workspace = empty({static_cast<int64_t>(bytes)}, at::kByte, device);
  const int st = g_lib.attention(
      q.t.data_ptr(), k.t.data_ptr(), v.t.data_ptr(), O.data_ptr(), type_code(type, "Q"),
      static_cast<int>(B), static_cast<int>(Tq), static_cast<int>(Tk), static_cast<int>(heads),
      static_cast<int>(kv_heads), static_cast<int>(D), q.row, q.batch, k.row, k.batch, v.row,
      v.batch, lens.defined() ? static_cast<const int*>(lens.data_ptr()) : nullptr, scale,
      bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(device));
  return passed(st, op) ? THPVariable_Wrap(std::move(O)) : nullptr;
  END_HANDLE_TH_ERRORS
}

// (quantize, layernorm, gemm, attention, attention_workspace: addresses in
// libvitb200.so; raise_status)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 6, "bind takes five addresses and a function");
  void* at[5];
  for (int i = 0; i < 5; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "bind: null address");
      return nullptr;
    }
  }
  g_lib.quantize = reinterpret_cast<decltype(g_lib.quantize)>(at[0]);
  g_lib.layernorm = reinterpret_cast<decltype(g_lib.layernorm)>(at[1]);
  g_lib.attention = reinterpret_cast<decltype(g_lib.attention)>(at[3]);
  g_lib.attention_workspace = reinterpret_cast<decltype(g_lib.attention_workspace)>(at[4]);
  Py_INCREF(args[5]);
  Py_XDECREF(g_lib.error);
  g_lib.error = args[5];
  g_lib.gemm = reinterpret_cast<decltype(g_lib.gemm)>(at[2]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define VITB200_METHOD(f) \
  {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {VITB200_METHOD(bind),         VITB200_METHOD(watched),
                          VITB200_METHOD(quantize_fp8), VITB200_METHOD(layernorm_fp8),
                          VITB200_METHOD(gemm_fp8),     VITB200_METHOD(cross_attention),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) {
  PyObject* m = PyModule_Create(&kModule);
  // (a module of another PyTorch may still find all its symbols)
  if (m && PyModule_AddStringConstant(m, "BUILT_FOR", VITB200_BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
