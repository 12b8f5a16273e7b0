// Host side of one forward call on torch tensors: the checks of ForwardPlan and gq_linear.forward, the output, the
// workspace and the C struct in native code, then the C entry point whose address the caller hands in.  Host code only; nothing is kept
// from one call for the next.  The steps take 14 to 16 us in Python beside the 7 us of the entry point's two launches, 4 to 6 here, and a decode
// call's kernels 11 to 17: 2560 -> 6144, one row, 4 adapters of rank 64 23.3 -> 12.4 us a call; 12288 -> 4096, 16 rows, 4-bit codes 25.2 -> 18.1.
//
// Every function returns the output tensor (grouped_bwd: a tuple of two; grad_table: the table's bytes and the adapters; accumulation_stream: a number), an int (the entry point's status, not OK), or None for anything out of the ordinary -- a wrong
// dtype, shape or device, a tensor subclass or mode, a tensor that is not contiguous, one that requires a gradient, a geometry that
// the library refuses -- and the caller then goes the general way, which converts, differentiates or raises.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TensorSubclassLikeUtils.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>

#include <algorithm>
#include <vector>

#include "bf16_api.h"

namespace {

constexpr int64_t kMaxRank = 64, kMaxAdapters = 64;

struct Args {
  PyObject* const* p;
  bool ok = true;
  // an ordinary tensor, or null where the argument is None
  const at::Tensor* tensor(int i) {
    if (p[i] == Py_None) return nullptr;
    if (!THPVariable_CheckExact(p[i])) { ok = false; return nullptr; }
    return &THPVariable_Unpack(p[i]);
  }
  int64_t integer(int i) {
    const int64_t v = PyLong_AsLongLong(p[i]);
    if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); ok = false; }
    return v;
  }
  void* address(int i) { return reinterpret_cast<void*>(static_cast<uintptr_t>(integer(i))); }
};

bool plain(const at::Tensor& t, at::ScalarType type, c10::Device device) {
  return t.layout() == at::kStrided && !t.is_nested() && t.scalar_type() == type && t.device() == device && t.is_contiguous() && t.unsafeGetTensorImpl()->has_storage() &&
         !at::isTensorSubclassLike(t) && !(c10::GradMode::is_enabled() && t.requires_grad());
}

// Rows of K from x; 0 where the call is not an ordinary one.
int64_t rows_of(const at::Tensor* x, int64_t k, int64_t min_dim) {
  if (!x || !x->is_cuda() || x->layout() != at::kStrided || x->is_nested() || x->dim() < min_dim || k <= 0 || x->size(-1) != k || x->numel() == 0) return 0;
  if (c10::impl::TorchDispatchModeTLS::any_modes_set() || !plain(*x, at::kBFloat16, x->device())) return 0;
  if (c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getDevice() != x->device()) return 0;
  const int64_t rows = x->numel() / k;
  return rows <= 0x7fffffff ? rows : 0;
}

struct Lora {
  int64_t adapters = 0, rank = 0;
  const void *a = nullptr, *b = nullptr;
  const float* scaling = nullptr;
};
// A [(n,) K, r], B [(n,) r, N], scaling float32 [n]; false where they are not plain or do not fit.
bool lora_of(const at::Tensor* a, const at::Tensor* b, const at::Tensor* s, int64_t k, int64_t n, c10::Device device, Lora& l) {
  if (!a && !b) return true;
  if (!a || !b || !s || a->dim() != b->dim() || (a->dim() != 2 && a->dim() != 3)) return false;
  if (!plain(*a, at::kBFloat16, device) || !plain(*b, at::kBFloat16, device) || !plain(*s, at::kFloat, device)) return false;
  l.adapters = a->dim() == 3 ? a->size(0) : 1;
  l.rank = a->size(-1);
  if (l.adapters < 1 || l.adapters > kMaxAdapters || l.rank < 1 || l.rank > kMaxRank || a->size(-2) != k || b->size(-2) != l.rank || b->size(-1) != n ||
      (b->dim() == 3 && b->size(0) != l.adapters) || s->dim() != 1 || s->size(0) != l.adapters)
    return false;
  l.a = a->const_data_ptr();
  l.b = b->const_data_ptr();
  l.scaling = s->const_data_ptr<float>();
  return true;
}

// Allocations and launches may wait for the GPU: other Python threads go on meanwhile.
struct WithoutGil {
  PyThreadState* const state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

PyObject* finish(at::Tensor&& out, int status) {
  return status == 0 ? THPVariable_Wrap(std::move(out)) : PyLong_FromLong(status);
}

// dense(x, packed, scales, k, n, a, b, scaling, adapter_indices, gamma, residual, flags, eps, entry, workspace_bytes, forward_path,
// stream)
PyObject* dense(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc != 17) { PyErr_SetString(PyExc_TypeError, "dense takes 17 arguments"); return nullptr; }
  HANDLE_TH_ERRORS
  Args arg{argv};
  const at::Tensor *x = arg.tensor(0), *packed = arg.tensor(1), *scales = arg.tensor(2), *a = arg.tensor(5), *b = arg.tensor(6),
                   *s = arg.tensor(7), *idx = arg.tensor(8), *gamma = arg.tensor(9), *residual = arg.tensor(10);
  const int64_t k = arg.integer(3), n = arg.integer(4), flags = arg.integer(11);
  const double eps = PyFloat_Check(argv[12]) ? PyFloat_AS_DOUBLE(argv[12]) : -1.0;
  const auto entry = reinterpret_cast<int (*)(const mi355_w8a8_problem*, void*)>(arg.address(13));
  const auto bytes_of = reinterpret_cast<uint64_t (*)(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t)>(arg.address(14));
  const auto path_of = reinterpret_cast<int (*)(uint32_t, uint32_t, uint32_t, uint32_t)>(arg.address(15));
  void* const stream = arg.address(16);
  if (!arg.ok || !entry || !bytes_of || !path_of || !packed || !scales || n <= 0 || eps < 0.0) Py_RETURN_NONE;
  const int64_t m = rows_of(x, k, 2);
  if (m == 0) Py_RETURN_NONE;
  const c10::Device device = x->device();
  if (!plain(*packed, at::kByte, device) || !plain(*scales, at::kFloat, device)) Py_RETURN_NONE;
  Lora lora;
  if (!lora_of(a, b, s, k, n, device, lora)) Py_RETURN_NONE;
  const bool swiglu = (flags & MI355_W8A8_FLAG_SWIGLU) != 0;
  if (swiglu && n % 2) Py_RETURN_NONE;
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = swiglu ? n / 2 : n;
  if (gamma && (!plain(*gamma, at::kFloat, device) || gamma->dim() != 1 || gamma->size(0) != k)) Py_RETURN_NONE;
  if (residual && (!plain(*residual, at::kBFloat16, device) || residual->sizes() != at::IntArrayRef(shape))) Py_RETURN_NONE;
  if (idx && (!lora.adapters || !plain(*idx, at::kInt, device) || idx->numel() == 0 || m % idx->numel())) Py_RETURN_NONE;
  const uint64_t bytes = bytes_of((uint32_t)m, (uint32_t)k, (uint32_t)n, (uint32_t)lora.adapters, (uint32_t)lora.rank, (uint32_t)flags);
  if (bytes == 0) Py_RETURN_NONE;
  at::Tensor out;
  int status;
  {
    const WithoutGil released;
    // One index per example, whose rows follow each other: the routing launch of the tiled paths reads it as it is (the decode
    // kernels take an index per row, and every path an aligned array).
    at::Tensor rows_idx;
    uint32_t per = 1;
    if (idx) {
      rows_idx = *idx;
      const int64_t rows = m / idx->numel();
      if (rows > 1) {
        const int path = path_of((uint32_t)m, (uint32_t)k, (uint32_t)n, (uint32_t)flags);
        if (path == MI355_W8A8_PATH_SKINNY || path == MI355_W8A8_PATH_SKINNY_CHUNKS || (reinterpret_cast<uintptr_t>(idx->const_data_ptr()) & 15u))
          rows_idx = idx->reshape({-1, 1}).expand({idx->numel(), rows}).contiguous();
        else
          per = (uint32_t)rows;
      }
    }
    out = at::empty(shape, x->options().requires_grad(false));
    const at::Tensor ws = at::empty({(int64_t)bytes}, packed->options().requires_grad(false));
    mi355_w8a8_problem_z whole{};
    whole.rows_per_index = per;
    mi355_w8a8_problem& p = whole.call;
    p.struct_size = sizeof(whole);
    p.flags = (uint32_t)flags;
    p.m = (uint32_t)m; p.k = (uint32_t)k; p.n = (uint32_t)n;
    p.n_adapters = (uint32_t)lora.adapters; p.rank = (uint32_t)lora.rank;
    p.rms_eps = (float)eps;
    p.x = x->const_data_ptr();
    p.w_packed = packed->const_data_ptr(); p.w_scales = scales->const_data_ptr<float>();
    p.lora_a = lora.a; p.lora_b = lora.b; p.lora_scaling = lora.scaling;
    p.adapter_indices = idx ? rows_idx.const_data_ptr<int32_t>() : nullptr;
    p.rms_gamma = gamma ? gamma->const_data_ptr<float>() : nullptr;
    p.residual = residual ? residual->const_data_ptr() : nullptr;
    p.out = out.mutable_data_ptr();
    p.workspace = ws.mutable_data_ptr();
    p.workspace_bytes = bytes;
    // (what the kernels touch was allocated for the stream they are enqueued on, or is held by the caller)
    status = entry(&p, stream);
  }
  return finish(std::move(out), status);
  END_HANDLE_TH_ERRORS
}

// group_scaled(x, packed, scales, k, k_pad, n, group, weight_bits, activation_bits, a, b, scaling, entry, workspace_bytes, stream)
PyObject* group_scaled(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc != 15) { PyErr_SetString(PyExc_TypeError, "group_scaled takes 15 arguments"); return nullptr; }
  HANDLE_TH_ERRORS
  Args arg{argv};
  const at::Tensor *x = arg.tensor(0), *packed = arg.tensor(1), *scales = arg.tensor(2), *a = arg.tensor(9), *b = arg.tensor(10),
                   *s = arg.tensor(11);
  const int64_t k = arg.integer(3), k_pad = arg.integer(4), n = arg.integer(5), group = arg.integer(6), wbits = arg.integer(7),
                abits = arg.integer(8);
  const auto entry = reinterpret_cast<int (*)(const mi355_w8a8_gq_problem*, void*)>(arg.address(12));
  const auto bytes_of = reinterpret_cast<uint64_t (*)(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t)>(arg.address(13));
  void* const stream = arg.address(14);
  if (!arg.ok || !entry || !bytes_of || !packed || !scales || n <= 0 || k_pad <= 0 || group <= 0) Py_RETURN_NONE;
  const int64_t m = rows_of(x, k, 1);
  if (m == 0) Py_RETURN_NONE;
  const c10::Device device = x->device();
  if (!plain(*packed, at::kByte, device) || !plain(*scales, at::kFloat, device)) Py_RETURN_NONE;
  Lora lora;
  if (!lora_of(a, b, s, k, n, device, lora)) Py_RETURN_NONE;
  const uint64_t bytes = bytes_of((uint32_t)m, (uint32_t)k_pad, (uint32_t)group, (uint32_t)lora.adapters, (uint32_t)lora.rank);
  if (bytes == 0) Py_RETURN_NONE;
  at::DimVector shape(x->sizes().begin(), x->sizes().end());
  shape.back() = n;
  at::Tensor out;
  int status;
  {
    const WithoutGil released;
    out = at::empty(shape, x->options().requires_grad(false));
    const at::Tensor ws = at::empty({(int64_t)bytes}, packed->options().requires_grad(false));
    mi355_w8a8_gq_problem p{};
    p.struct_size = sizeof(p);
    p.m = (uint32_t)m; p.k = (uint32_t)k; p.k_pad = (uint32_t)k_pad; p.n = (uint32_t)n;
    p.group_size = (uint32_t)group; p.weight_bits = (uint32_t)wbits; p.activation_bits = (uint32_t)abits;
    p.n_adapters = (uint32_t)lora.adapters; p.rank = (uint32_t)lora.rank;
    p.x = x->const_data_ptr();
    p.w_packed = packed->const_data_ptr(); p.w_scales = scales->const_data_ptr<float>();
    p.lora_a = lora.a; p.lora_b = lora.b; p.lora_scaling = lora.scaling;
    p.out = out.mutable_data_ptr();
    p.workspace = ws.mutable_data_ptr();
    p.workspace_bytes = bytes;
    status = entry(&p, stream);
  }
  return finish(std::move(out), status);
  END_HANDLE_TH_ERRORS
}

// A tensor that the bf16 operators take as it is: plain and, for the kernels' 16-byte loads, aligned.
bool whole(const at::Tensor* t, at::ScalarType type, c10::Device device, int64_t dim) {
  return t && plain(*t, type, device) && t->dim() == dim && (reinterpret_cast<uintptr_t>(t->const_data_ptr()) & 15u) == 0;
}
// The device of an ordinary call on t: the current one.
bool here(const at::Tensor* t) {
  return t && t->is_cuda() && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getDevice() == t->device();
}
// no flags but those of the tiles: the type of dw is that of the tensor made here
bool grouped_flags(int64_t flags) {
  return (flags & ~(int64_t)(MI355_W8A8_FLAG_BF16_GROUPED_TILE_256X256 | MI355_W8A8_FLAG_BF16_GROUPED_TILE_128X256 |
                             MI355_W8A8_FLAG_BF16_GROUPED_TILE_64X128)) == 0;
}
bool grouped_dims(int64_t m, int64_t k, int64_t n, int64_t g) {
  return m > 0 && m <= (1 << 20) && k > 0 && n > 0 && k % 8 == 0 && n % 8 == 0 && k <= MI355_W8A8_BF16_GROUPED_MAX_FEATURES &&
         n <= MI355_W8A8_BF16_GROUPED_MAX_FEATURES && g > 0 && g <= 1024;
}

// grouped(x, weight, group_sizes, flags, entry, workspace_bytes, stream)
PyObject* grouped(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc != 7) { PyErr_SetString(PyExc_TypeError, "grouped takes 7 arguments"); return nullptr; }
  HANDLE_TH_ERRORS
  Args arg{argv};
  const at::Tensor *x = arg.tensor(0), *w = arg.tensor(1), *sizes = arg.tensor(2);
  const int64_t flags = arg.integer(3);
  const auto entry = reinterpret_cast<int (*)(const mi355_w8a8_bf16_grouped_problem*, void*)>(arg.address(4));
  const auto bytes_of = reinterpret_cast<uint64_t (*)(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t)>(arg.address(5));
  void* const stream = arg.address(6);
  if (!arg.ok || !entry || !bytes_of || !grouped_flags(flags) || !here(x)) Py_RETURN_NONE;
  const c10::Device device = x->device();
  if (!whole(x, at::kBFloat16, device, 2) || !whole(w, at::kBFloat16, device, 3) || !sizes || !plain(*sizes, at::kInt, device) || sizes->dim() != 1) Py_RETURN_NONE;
  const int64_t m = x->size(0), k = x->size(1), n = w->size(2), g = w->size(0);
  if (w->size(1) != k || sizes->size(0) != g || !grouped_dims(m, k, n, g)) Py_RETURN_NONE;
  at::Tensor out, ws;
  int status;
  {
    const WithoutGil released;
    out = at::empty({m, n}, x->options().requires_grad(false));
    mi355_w8a8_bf16_grouped_problem p{};
    p.struct_size = sizeof(p);
    p.flags = (uint32_t)flags;
    p.m = (uint32_t)m; p.k = (uint32_t)k; p.n = (uint32_t)n; p.n_groups = (uint32_t)g;
    p.x = x->const_data_ptr(); p.weight = w->const_data_ptr(); p.group_sizes = sizes->const_data_ptr<int32_t>();
    p.out = out.mutable_data_ptr();
    p.workspace_bytes = bytes_of(p.m, p.k, p.n, p.n_groups, p.flags);
    if (p.workspace_bytes) {
      ws = at::empty({(int64_t)p.workspace_bytes}, x->options().requires_grad(false).dtype(at::kByte));
      p.workspace = ws.mutable_data_ptr();
    }
    status = entry(&p, stream);
  }
  return finish(std::move(out), status);
  END_HANDLE_TH_ERRORS
}

// grouped_bwd(x, dy, weight, group_sizes, need_dx, need_dw, f32, flags, entry, workspace_bytes, stream)
PyObject* grouped_bwd(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc != 11) { PyErr_SetString(PyExc_TypeError, "grouped_bwd takes 11 arguments"); return nullptr; }
  HANDLE_TH_ERRORS
  Args arg{argv};
  const at::Tensor *x = arg.tensor(0), *dy = arg.tensor(1), *w = arg.tensor(2), *sizes = arg.tensor(3);
  const bool need_dx = argv[4] == Py_True, need_dw = argv[5] == Py_True, f32 = argv[6] == Py_True;
  const int64_t flags = arg.integer(7);
  const auto entry = reinterpret_cast<int (*)(const mi355_w8a8_bf16_grouped_bwd_problem*, void*)>(arg.address(8));
  const auto bytes_of = reinterpret_cast<uint64_t (*)(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t)>(arg.address(9));
  void* const stream = arg.address(10);
  if (!arg.ok || !entry || !bytes_of || !grouped_flags(flags) || !here(dy) || !x || !w) Py_RETURN_NONE;
  const c10::Device device = dy->device();
  if (!whole(dy, at::kBFloat16, device, 2) || !whole(x, at::kBFloat16, device, 2) || !whole(w, at::kBFloat16, device, 3) || !sizes ||
      !plain(*sizes, at::kInt, device) || sizes->dim() != 1)
    Py_RETURN_NONE;
  const int64_t m = dy->size(0), k = w->size(1), n = w->size(2), g = w->size(0);
  if (dy->size(1) != n || x->size(0) != m || x->size(1) != k || sizes->size(0) != g || !grouped_dims(m, k, n, g)) Py_RETURN_NONE;
  at::Tensor dx, dw, ws;
  int status;
  {
    const WithoutGil released;
    if (need_dx) dx = at::empty({m, k}, dy->options().requires_grad(false));
    if (need_dw) dw = at::empty({g, k, n}, dy->options().requires_grad(false).dtype(f32 ? at::kFloat : at::kBFloat16));
    mi355_w8a8_bf16_grouped_bwd_problem p{};
    p.struct_size = sizeof(p);
    p.flags = (uint32_t)flags | (f32 ? MI355_W8A8_FLAG_BF16_GROUPED_DW_F32 : 0u);
    p.m = (uint32_t)m; p.k = (uint32_t)k; p.n = (uint32_t)n; p.n_groups = (uint32_t)g;
    p.x = x->const_data_ptr(); p.dy = dy->const_data_ptr(); p.weight = w->const_data_ptr(); p.group_sizes = sizes->const_data_ptr<int32_t>();
    p.dx = need_dx ? dx.mutable_data_ptr() : nullptr;
    p.dw = need_dw ? dw.mutable_data_ptr() : nullptr;
    p.workspace_bytes = bytes_of(p.m, p.k, p.n, p.n_groups, p.flags, need_dx, need_dw);
    if (p.workspace_bytes) {
      ws = at::empty({(int64_t)p.workspace_bytes}, dy->options().requires_grad(false).dtype(at::kByte));
      p.workspace = ws.mutable_data_ptr();
    }
    status = entry(&p, stream);
  }
  if (status) return PyLong_FromLong(status);
  PyObject* const a = need_dx ? THPVariable_Wrap(std::move(dx)) : (Py_INCREF(Py_None), Py_None);
  PyObject* const b = need_dw ? THPVariable_Wrap(std::move(dw)) : (Py_INCREF(Py_None), Py_None);
  return a && b ? Py_BuildValue("(NN)", a, b) : nullptr;
  END_HANDLE_TH_ERRORS
}

// The index side of an embedding call; false where it is not an ordinary one.  shape: the table's.
bool embedding_call(const at::Tensor* ids, const at::Tensor* adapters, PyObject* scale, at::IntArrayRef shape, at::ScalarType type, c10::Device device,
                    mi355_w8a8_embedding_problem& p) {
  const int64_t dim = (int64_t)shape.size();
  if ((dim != 2 && dim != 3) || (type != at::kBFloat16 && type != at::kFloat) || !ids) return false;
  const bool wide = ids->scalar_type() == at::kLong;
  if (!plain(*ids, wide ? at::kLong : at::kInt, device)) return false;
  const int64_t n = ids->numel(), vocab = shape[dim - 2], width = shape[dim - 1], adapted = dim == 3 ? shape[0] : 0, rows = adapted ? adapted : 1;
  if (n <= 0 || n > (1 << 20) || vocab <= 0 || width <= 0 || width > (int64_t)MI355_W8A8_EMBEDDING_MAX_WIDTH || vocab > (int64_t)MI355_W8A8_EMBEDDING_MAX_ROWS ||
      rows > (int64_t)MI355_W8A8_EMBEDDING_MAX_ROWS / vocab || (dim == 3 && adapted <= 0))
    return false;
  if (adapters ? dim != 3 || !plain(*adapters, at::kInt, device) || adapters->numel() != n : adapted > 1) return false;
  p.scale = 1.0f;
  if (PyFloat_Check(scale)) {
    p.scale = (float)PyFloat_AS_DOUBLE(scale);
    if (!(p.scale - p.scale == 0.0f)) return false;
  } else if (THPVariable_CheckExact(scale)) {
    const at::Tensor& t = THPVariable_Unpack(scale);
    if (dim != 3 || !plain(t, at::kFloat, device) || t.dim() != 1 || t.size(0) != adapted) return false;
    p.scales = t.const_data_ptr<float>();
  } else if (scale != Py_None) {
    return false;
  }
  p.struct_size = sizeof(p);
  p.flags = (type == at::kFloat ? MI355_W8A8_FLAG_EMBEDDING_F32 : 0u) | (wide ? MI355_W8A8_FLAG_EMBEDDING_IDS64 : 0u);
  p.n_tokens = (uint32_t)n; p.vocab = (uint32_t)vocab; p.width = (uint32_t)width; p.n_adapters = (uint32_t)adapted;
  p.ids = ids->const_data_ptr();
  p.adapter_indices = adapters ? adapters->const_data_ptr<int32_t>() : nullptr;
  return true;
}

// embedding(table, ids, scale, adapter_indices, entry, stream)
PyObject* embedding(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc != 6) { PyErr_SetString(PyExc_TypeError, "embedding takes 6 arguments"); return nullptr; }
  HANDLE_TH_ERRORS
  Args arg{argv};
  const at::Tensor *table = arg.tensor(0), *ids = arg.tensor(1), *adapters = arg.tensor(3);
  const auto entry = reinterpret_cast<int (*)(const mi355_w8a8_embedding_problem*, void*)>(arg.address(4));
  void* const stream = arg.address(5);
  if (!arg.ok || !entry || !here(table) || !plain(*table, table->scalar_type(), table->device())) Py_RETURN_NONE;
  mi355_w8a8_embedding_problem p{};
  if (!embedding_call(ids, adapters, argv[2], table->sizes(), table->scalar_type(), table->device(), p)) Py_RETURN_NONE;
  at::DimVector shape(ids->sizes().begin(), ids->sizes().end());
  shape.push_back(p.width);
  at::Tensor out;
  int status;
  {
    const WithoutGil released;
    out = at::empty(shape, table->options().requires_grad(false));
    p.table = table->const_data_ptr();
    p.out = out.mutable_data_ptr();
    status = entry(&p, stream);
  }
  return finish(std::move(out), status);
  END_HANDLE_TH_ERRORS
}

// embedding_bwd(d_out, ids, table_shape, scale, adapter_indices, entry, workspace_bytes, stream)
PyObject* embedding_bwd(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc != 8) { PyErr_SetString(PyExc_TypeError, "embedding_bwd takes 8 arguments"); return nullptr; }
  HANDLE_TH_ERRORS
  Args arg{argv};
  const at::Tensor *d = arg.tensor(0), *ids = arg.tensor(1), *adapters = arg.tensor(4);
  const auto entry = reinterpret_cast<int (*)(const mi355_w8a8_embedding_problem*, void*)>(arg.address(5));
  const auto bytes_of = reinterpret_cast<uint64_t (*)(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t)>(arg.address(6));
  void* const stream = arg.address(7);
  if (!arg.ok || !entry || !bytes_of || !here(d) || !ids || !plain(*d, d->scalar_type(), d->device()) || !PyTuple_CheckExact(argv[2])) Py_RETURN_NONE;
  at::DimVector table;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(argv[2]); ++i) {
    PyObject* const v = PyTuple_GET_ITEM(argv[2], i);
    if (!PyLong_CheckExact(v)) Py_RETURN_NONE;
    table.push_back(PyLong_AsLongLong(v));
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
  }
  mi355_w8a8_embedding_problem p{};
  if (!embedding_call(ids, adapters, argv[3], table, d->scalar_type(), d->device(), p)) Py_RETURN_NONE;
  at::DimVector shape(ids->sizes().begin(), ids->sizes().end());
  shape.push_back(p.width);
  if (d->sizes() != at::IntArrayRef(shape)) Py_RETURN_NONE;
  const uint64_t bytes = bytes_of(p.n_tokens, p.vocab, p.width, p.n_adapters, p.flags);
  if (bytes == 0) Py_RETURN_NONE;
  at::Tensor out;
  int status;
  {
    const WithoutGil released;
    out = at::empty(table, d->options().requires_grad(false));
    const at::Tensor ws = at::empty({(int64_t)bytes}, d->options().requires_grad(false).dtype(at::kByte));
    p.d_out = d->const_data_ptr();
    p.out = out.mutable_data_ptr();
    p.workspace = ws.mutable_data_ptr();
    p.workspace_bytes = bytes;
    status = entry(&p, stream);
  }
  return finish(std::move(out), status);
  END_HANDLE_TH_ERRORS
}

// accumulation_stream(leaf) -> number of the stream (0: the default one) on which autograd adds to the leaf's gradient as long as one of its graphs
// lives, or None where none does.
PyObject* accumulation_stream(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc != 1 || !THPVariable_Check(argv[0])) { PyErr_SetString(PyExc_TypeError, "accumulation_stream takes a tensor"); return nullptr; }
  HANDLE_TH_ERRORS
  const auto node = torch::autograd::impl::try_get_grad_accumulator(THPVariable_Unpack(argv[0]));
  const auto stream = node ? node->stream() : std::nullopt;
  if (!stream) Py_RETURN_NONE;
  return PyLong_FromLongLong(stream->id());
  END_HANDLE_TH_ERRORS
}

// A tensor of a gradient table: its values lie behind each other.
bool whole_gradient(const at::Tensor& t, c10::Device device) {
  return t.layout() == at::kStrided && !t.is_nested() && t.device() == device && t.is_contiguous() && t.unsafeGetTensorImpl()->has_storage() &&
         !at::isTensorSubclassLike(t) && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat);
}

// grad_table(grads, outs, per_adapter), lists of tensors (outs: or None) -> (bytes of the C table, adapters), or None where something is not
// ordinary: an output that overlaps anything but its own gradient, whose place it may have, is not.
PyObject* grad_table(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc != 3) { PyErr_SetString(PyExc_TypeError, "grad_table takes 3 arguments"); return nullptr; }
  HANDLE_TH_ERRORS
  if (!PyList_CheckExact(argv[0]) || (argv[1] != Py_None && !PyList_CheckExact(argv[1])) || c10::impl::TorchDispatchModeTLS::any_modes_set()) Py_RETURN_NONE;
  const Py_ssize_t n = PyList_GET_SIZE(argv[0]);
  const bool written = argv[1] != Py_None, per_adapter = argv[2] == Py_True;
  if (n < 1 || n > (Py_ssize_t)MI355_W8A8_GRAD_MAX_TENSORS || (written && PyList_GET_SIZE(argv[1]) != n)) Py_RETURN_NONE;
  struct Span { uintptr_t from, to; Py_ssize_t of; };
  std::vector<Span> outs;
  std::vector<mi355_w8a8_grad_tensor> table((size_t)n);
  int64_t adapters = 1;
  c10::Device device(c10::DeviceType::CPU);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* const item = PyList_GET_ITEM(argv[0], i);
    if (!THPVariable_Check(item)) Py_RETURN_NONE;
    const at::Tensor& g = THPVariable_Unpack(item);
    if (i == 0) {
      device = g.device();
      if (!device.is_cuda()) Py_RETURN_NONE;
      if (per_adapter) adapters = g.dim() ? g.size(0) : 0;
      if (adapters < 1 || adapters > 65535) Py_RETURN_NONE;
    }
    if (!whole_gradient(g, device) || (per_adapter && (g.dim() == 0 || g.size(0) != adapters))) Py_RETURN_NONE;
    mi355_w8a8_grad_tensor& t = table[(size_t)i];
    t = mi355_w8a8_grad_tensor{g.const_data_ptr(), nullptr, (uint64_t)(g.numel() / adapters),
                               g.scalar_type() == at::kFloat ? MI355_W8A8_GRAD_F32 : MI355_W8A8_GRAD_BF16, 0u};
    if (!written) continue;
    PyObject* const target = PyList_GET_ITEM(argv[1], i);
    if (!THPVariable_Check(target)) Py_RETURN_NONE;
    const at::Tensor& o = THPVariable_Unpack(target);
    if (!whole_gradient(o, device) || o.scalar_type() != g.scalar_type() || o.sizes() != g.sizes()) Py_RETURN_NONE;
    t.out = const_cast<void*>(o.const_data_ptr());
    const uintptr_t from = reinterpret_cast<uintptr_t>(t.out);
    if (o.numel()) outs.push_back({from, from + (uintptr_t)o.nbytes(), i});
  }
  std::sort(outs.begin(), outs.end(), [](const Span& a, const Span& b) { return a.from < b.from; });
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i].from < outs[i - 1].to) Py_RETURN_NONE;
  for (const Span& own : outs) {  // every gradient with values has an output of the same size
    const uintptr_t from = reinterpret_cast<uintptr_t>(table[(size_t)own.of].grad), to = from + (own.to - own.from);
    if (from == own.from) continue;
    auto behind = std::lower_bound(outs.begin(), outs.end(), to, [](const Span& a, uintptr_t end) { return a.from < end; });
    if (behind != outs.begin() && (behind - 1)->to > from) Py_RETURN_NONE;
  }
  return Py_BuildValue("(y#L)", reinterpret_cast<const char*>(table.data()), (Py_ssize_t)(table.size() * sizeof(mi355_w8a8_grad_tensor)), (long long)adapters);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"dense", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dense)), METH_FASTCALL, "One forward call of the per-channel linear."},
    {"group_scaled", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(group_scaled)), METH_FASTCALL,
     "One forward call of the group-scaled linear."},
    {"grouped", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(grouped)), METH_FASTCALL, "One call of the bf16 products grouped by expert."},
    {"grouped_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(grouped_bwd)), METH_FASTCALL, "Their two gradients."},
    {"embedding", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(embedding)), METH_FASTCALL, "One lookup of embedding rows."},
    {"embedding_bwd", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(embedding_bwd)), METH_FASTCALL, "The table's gradient."},
    {"accumulation_stream", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(accumulation_stream)), METH_FASTCALL,
     "The stream on which autograd adds to a leaf's gradient."},
    {"grad_table", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(grad_table)), METH_FASTCALL, "The C table of gradients and their outputs."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "mi355_w8a8_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_mi355_w8a8_host() {
  PyObject* const m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", MI355_TORCH_VERSION) != 0) {  // (its C++ ABI is this one's: _native.host)
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
