// Host side of the serving operators: argument checks, result tensors and the library calls of paged.py,
// rotary.py, verify.py and int4.py. Those calls last a few microseconds on the device; checked and marshalled in Python they took 13
// to 15 microseconds of the host. A Python extension module on torch's tensors, no device code; the C
// ABI's entry points are handed over by address.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <cmath>
#include <sstream>

#include "../../include/strassen_mi355x.h"

namespace {

using at::Tensor;

// A refused argument, raised as ValueError (or TypeError).
struct Refused : std::exception {
  std::string message;
  PyObject* type;
  Refused(std::string m, PyObject* t) : message(std::move(m)), type(t) {}
  const char* what() const noexcept override { return message.c_str(); }
};

template <class... Args>
[[noreturn]] void refuse(const Args&... args) {
  std::ostringstream s;
  (s << ... << args);
  throw Refused(s.str(), PyExc_ValueError);
}

// A Python exception is set already.
struct Raised {};

struct Library {
  decltype(&smx_paged_plan) plan;
  decltype(&smx_paged_write) write;
  decltype(&smx_paged_attention_lse) attention;
  decltype(&smx_paged_attention_workspace_bytes) attention_bytes;
  decltype(&smx_paged_key_weights) weights;
  decltype(&smx_paged_key_weights_workspace_bytes) weights_bytes;
  decltype(&smx_paged_evict) evict;
  decltype(&smx_paged_evict_workspace_bytes) evict_bytes;
  decltype(&smx_rotary) rotary;
  decltype(&smx_verify_drafts) verify;
  decltype(&smx_verify_workspace_bytes) verify_bytes;
  decltype(&smx_int4_matmul) int4;
  decltype(&smx_int4_workspace_bytes) int4_bytes;
  decltype(&smx_last_error) error;
  PyObject* raw_stream;  // device index -> the handle of torch's current stream there
} lib;

// What smx_* returned, with the exceptions of _lib.check.
void check(int rc) {
  if (rc == SMX_OK) return;
  throw Refused(lib.error(), rc == SMX_ERR_INVALID || rc == SMX_ERR_UNSUPPORTED ? PyExc_ValueError : PyExc_RuntimeError);
}

void* stream_of(const at::Device& device) {
  PyObject* const index = PyLong_FromLong(device.index());
  if (!index) throw Raised();
  PyObject* const handle = PyObject_CallOneArg(lib.raw_stream, index);
  Py_DECREF(index);
  if (!handle) throw Raised();
  void* const stream = PyLong_AsVoidPtr(handle);
  Py_DECREF(handle);
  if (PyErr_Occurred()) throw Raised();
  return stream;
}

std::string shape_of(const Tensor& t) {
  std::ostringstream s;
  s << t.scalar_type() << " [";
  for (int64_t i = 0; i < t.dim(); ++i) s << (i ? ", " : "") << t.size(i);
  s << "]";
  return s.str();
}

// Tensors whose memory is not what they stand for: fake and other dispatching types, batched and
// differentiated ones of torch.func, views that negate when they are read, sparse layouts.
bool plain(const Tensor& t) {
  using c10::DispatchKey;
  constexpr c10::DispatchKeySet kOthers({DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper,
                                         DispatchKey::Batched, DispatchKey::Functionalize, DispatchKey::Conjugate,
                                         DispatchKey::Negative, DispatchKey::ZeroTensor});
  return t.layout() == at::kStrided && !t.key_set().has_any(kOthers);
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o))
    throw Refused(std::string(name) + " must be a tensor, got " + Py_TYPE(o)->tp_name, PyExc_TypeError);
  const Tensor& t = THPVariable_Unpack(o);
  if (!plain(t)) refuse(name, " must be a plain strided tensor, the kernels read its memory (got ", Py_TYPE(o)->tp_name, ")");
  return t;
}

// The call wrote to t: a backward pass that kept its values finds out.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A call that is traced would run once, on the tensors at hand, and be missing from what is traced.
void not_traced() {
  using c10::impl::TorchDispatchModeKey;
  using Modes = c10::impl::TorchDispatchModeTLS;
  if (!c10::impl::dispatch_mode_enabled()) return;
  for (const auto mode : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
    if (Modes::get_mode(mode)) refuse("serving operators cannot be traced (", c10::impl::to_string(mode), " mode)");
}

const Tensor& on_device(PyObject* o, const char* name) {
  const Tensor& t = tensor(o, name);
  if (!t.is_cuda()) refuse("the gfx950 kernel needs tensors on the HIP device (got ", name, " on ", t.device(), ")");
  return t;
}

const Tensor& on_device(PyObject* o, const char* name, const at::Device& device) {
  const Tensor& t = on_device(o, name);
  if (t.device() != device) refuse(name, " is on ", t.device(), ", the call on ", device);
  return t;
}

bool given(PyObject* o) { return o != Py_None; }

void no_gradients(std::initializer_list<PyObject*> tensors) {
  const c10::AutogradState& state = c10::AutogradState::get_tls_state();
  const bool backward = state.get_grad_mode(), forward = state.get_fw_grad_mode();
  for (PyObject* const o : tensors) {
    if (!given(o) || !THPVariable_Check(o)) continue;
    const Tensor& t = THPVariable_Unpack(o);
    if (backward && t.requires_grad())
      refuse("serving operators record no gradients: call them under torch.no_grad()");
    if (forward && t._fw_grad(0).defined())  // (torch has one level of forward-mode tangents)
      refuse("serving operators carry no forward-mode gradients: unpack the dual tensor first");
  }
}

int64_t integer(PyObject* o, const char* name, int64_t low, int64_t high) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised();
  if (v < low || v > high) refuse(name, " must be ", low, " to ", high, ", got ", v);
  return v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}

template <class F>
PyObject* guarded(F f) {
  try {
    not_traced();
    const at::AutoDispatchBelowADInplaceOrView below;  // nothing here records gradients
    return f();
  } catch (const Raised&) {
  } catch (const Refused& e) {
    PyErr_SetString(e.type, e.message.c_str());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// ---------------------------------------------------------------------------
// Plans
// ---------------------------------------------------------------------------

struct Plan {
  Tensor tables, memory;  // what the addresses below lie in
  at::Device device;
  int64_t page_size, num_pages, max_context;
  int64_t* slots;
  smx_paged_step step;
};

constexpr const char* kPlan = "strassen_tpu_amd.PagedPlan";

const Plan& plan_of(PyObject* o) {
  const auto* p = static_cast<const Plan*>(PyCapsule_GetPointer(o, kPlan));
  if (!p) throw Raised();
  return *p;
}

int32_t* int32_list(const Tensor& t, const char* name, int64_t length) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != length || !t.is_contiguous())
    refuse(name, " must be a contiguous int32 tensor of shape (", length, ",), got ", shape_of(t));
  return t.mutable_data_ptr<int32_t>();
}

const int32_t* table_rows(const Tensor& tables, int64_t requests) {
  if (tables.scalar_type() != at::kInt || tables.dim() != 2 || tables.size(0) != requests || !tables.size(1) ||
      (tables.size(1) > 1 && tables.stride(1) != 1) || (requests > 1 && tables.stride(0) < tables.size(1)))
    refuse("block_tables must be int32 [", requests, ", width] with rows apart from each other, got ", shape_of(tables));
  return tables.const_data_ptr<int32_t>();
}

// (context_lens, new_lens, block_tables, page_size, num_pages, tokens, free_pages, max_new, max_context) ->
// (capsule, requests, max_new, max_context, starts, rows, context, status, positions, slots, used, needed)
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    const Tensor& context_lens = on_device(a[0], "context_lens");
    const at::Device device = context_lens.device();
    if (context_lens.dim() != 1 || !context_lens.size(0)) refuse("context_lens must hold one length per request");
    const int64_t requests = context_lens.size(0);
    const int32_t* const context = int32_list(context_lens, "context_lens", requests);
    const int32_t* const fresh = int32_list(on_device(a[1], "new_lens", device), "new_lens", requests);
    const Tensor& tables = on_device(a[2], "block_tables", device);
    table_rows(tables, requests);
    const int64_t page_size = integer(a[3], "page_size", INT32_MIN, INT32_MAX);
    const int64_t num_pages = integer(a[4], "num_pages", INT32_MIN, INT32_MAX);
    const int64_t tokens = integer(a[5], "tokens", 1, SMX_PAGED_MAX_TOKENS);
    const int64_t width = std::min<int64_t>(tables.size(1), INT32_MAX);
    const int32_t* free = nullptr;
    int64_t free_count = 0;
    if (given(a[6])) {
      const Tensor& list = on_device(a[6], "free_pages", device);
      if (list.dim() != 1) refuse("free_pages must be a list of page numbers");
      free_count = list.size(0);
      if (free_count > INT32_MAX) refuse("free_pages is too long");
      free = int32_list(list, "free_pages", free_count);
      if (!free_count) free = fresh;  // an empty list too is a list: no request gets a new page
    }
    const int64_t max_new = given(a[7]) ? integer(a[7], "max_new", INT32_MIN, INT32_MAX) : tokens;
    const int64_t max_context = given(a[8]) ? integer(a[8], "max_context", INT32_MIN, INT32_MAX)
                                            : std::max<int64_t>(0, std::min<int64_t>(width * page_size, SMX_PAGED_MAX_CONTEXT));
    // one allocation for the small tensors: slots (int64) first, then the int32 ones
    const c10::DeviceGuard guard(device);
    const int64_t sizes[] = {2 * tokens, requests + 1, requests, requests, requests, tokens, 1, 1};
    int64_t total = 0;
    for (const int64_t s : sizes) total += s;
    const Tensor memory = at::empty({total}, context_lens.options());
    Tensor parts[8];
    int32_t* at[8];
    int64_t from = 0;
    int32_t* const base = memory.mutable_data_ptr<int32_t>();
    for (int i = 0; i < 8; ++i) {
      // a view of the memory, made directly (narrow() and view() take 3 us for the eight)
      parts[i] = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(memory.storage()), memory.key_set(),
                                                          c10::scalarTypeToTypeMeta(i ? at::kInt : at::kLong));
      c10::TensorImpl* const view = parts[i].unsafeGetTensorImpl();
      view->set_storage_offset(memory.storage_offset() + from);  // the int64 one lies at the front
      view->set_sizes_contiguous({i ? sizes[i] : tokens});
      at[i] = base + from;
      from += sizes[i];
    }
    auto* p = new Plan{tables, memory, device, page_size, num_pages, max_context, reinterpret_cast<int64_t*>(at[0]), {}};
    PyObject* const capsule = PyCapsule_New(p, kPlan, [](PyObject* c) {
      delete static_cast<Plan*>(PyCapsule_GetPointer(c, kPlan));
    });
    if (!capsule) {
      delete p;
      throw Raised();
    }
    try {
      const int64_t stride = requests > 1 ? tables.stride(0) : width;
      auto* const entries = tables.mutable_data_ptr<int32_t>();
      p->step = smx_paged_step{(int32_t)requests, (int32_t)tokens, (int32_t)max_new, entries, stride, at[1], at[2], at[3], at[5]};
      check(lib.plan((int32_t)std::min<int64_t>(requests, INT32_MAX), (int32_t)width, (int32_t)page_size, (int32_t)num_pages,
                     (int32_t)tokens, (int32_t)max_new, (int32_t)max_context, context, fresh, entries, stride, free,
                     (int32_t)free_count, at[1], at[2], at[3], at[5], p->slots, at[4], at[6], stream_of(device)));
      if (free) written(tables);
      PyObject* const result = PyTuple_New(12);
      if (!result) throw Raised();
      PyTuple_SET_ITEM(result, 0, capsule);
      const int64_t numbers[] = {requests, max_new, max_context};
      for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(result, 1 + i, PyLong_FromLongLong(numbers[i]));
      const int order[] = {1, 2, 3, 4, 5, 0, 6, 7};
      for (int i = 0; i < 8; ++i) PyTuple_SET_ITEM(result, 4 + i, THPVariable_Wrap(std::move(parts[order[i]])));
      return result;
    } catch (...) {
      Py_DECREF(capsule);
      throw;
    }
  });
}

// ---------------------------------------------------------------------------
// Caches and heads
// ---------------------------------------------------------------------------

// A cache's layout; of a plan's sizes where one is given.
smx_paged_cache cache_layout(const Tensor& k, const Tensor& v, const Plan* plan) {
  for (const Tensor* x : {&k, &v})
    if (x->scalar_type() != at::kBFloat16 || x->dim() != 4)
      refuse(x == &k ? "k_cache" : "v_cache", " must be a bf16 tensor [pages, page_size, kv_heads, head_dim], got ", shape_of(*x));
  if (k.sizes() != v.sizes()) refuse("k_cache and v_cache must have the same shape and strides");
  int64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    // the stride of a dimension of one is no stride: nothing steps over it
    strides[i] = k.size(i) == 1 ? k.size(3) : k.stride(i);
    if (k.size(i) != 1 && k.stride(i) != v.stride(i)) refuse("k_cache and v_cache must have the same shape and strides");
  }
  if (plan && (k.size(1) != plan->page_size || k.size(0) != plan->num_pages))
    refuse("the plan is of ", plan->num_pages, " pages of ", plan->page_size, " tokens, the cache of ", k.size(0), " of ", k.size(1));
  if (k.stride(3) != 1 || v.stride(3) != 1) refuse("cache heads must be contiguous runs");
  if (k.size(0) > INT32_MAX || k.size(1) > INT32_MAX || k.size(2) > 65535 || k.size(3) > 65535)
    refuse("too many pages, or too many or too wide heads: ", shape_of(k));
  return smx_paged_cache{k.mutable_data_ptr(), v.mutable_data_ptr(), strides[0], strides[1], strides[2],
                         (int32_t)k.size(0), (int32_t)k.size(1), (int32_t)k.size(2), (int32_t)k.size(3)};
}

smx_paged_cache cache_of(PyObject* k, PyObject* v, const Plan& plan) {
  return cache_layout(on_device(k, "k_cache", plan.device), on_device(v, "v_cache", plan.device), &plan);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Head rows [tokens, heads, head_dim]; rows that the kernels cannot take as they lie (not 16-byte aligned
// runs) are laid out first in `hold`, or refused without it. heads < 0: any number.
smx_heads heads_of(PyObject* o, const char* name, const Plan& plan, int64_t heads, int64_t head_dim, Tensor* hold) {
  const Tensor* x = &on_device(o, name, plan.device);
  if (x->scalar_type() != at::kBFloat16 || x->dim() != 3 || x->size(0) != plan.step.tokens || x->size(2) != head_dim ||
      (heads >= 0 && x->size(1) != heads)) {
    std::ostringstream want;
    if (heads >= 0) want << heads; else want << "heads";
    refuse(name, " must be a bf16 tensor of shape (", plan.step.tokens, ", ", want.str(), ", ", head_dim, "), got ", shape_of(*x));
  }
  auto stride = [](const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
  if (x->stride(2) != 1 || stride(*x, 0) % 8 || stride(*x, 1) % 8 || !aligned16(x->data_ptr())) {
    if (!hold) refuse(name, " rows must be 16-byte aligned runs");
    *hold = x->clone(at::MemoryFormat::Contiguous);
    x = hold;
  }
  if (x->size(1) > INT32_MAX) refuse(name, " has too many heads");
  return smx_heads{x->mutable_data_ptr(), stride(*x, 0), stride(*x, 1), (int32_t)x->size(1)};
}

// x contiguous, 16-byte aligned, bf16 or float32 (laid out anew in `hold` where it is not).
const Tensor& laid_out(const Tensor& x, Tensor* hold) {
  const bool typed = x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat;
  if (typed && x.is_contiguous() && aligned16(x.data_ptr())) return x;
  *hold = (typed ? x : x.to(at::kFloat)).clone(at::MemoryFormat::Contiguous);
  return *hold;
}

const void* scale_of(PyObject* o, const char* name, const Plan& plan, int64_t head_dim, int32_t bit, int32_t* dtypes,
                     Tensor* hold) {
  if (!given(o)) return nullptr;
  const Tensor& x = on_device(o, name, plan.device);
  if (x.dim() != 1 || x.size(0) != head_dim) refuse(name, " must have shape (", head_dim, ",), got ", shape_of(x));
  const Tensor& y = laid_out(x, hold);
  if (y.scalar_type() == at::kFloat) *dtypes |= bit;
  return y.data_ptr();
}

// (k, v, k_cache, v_cache, plan, q, rope_cos, rope_sin, q_scale, k_scale, eps) -> q' or None
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    no_gradients({a[0], a[1], a[2], a[3], a[5], a[6], a[7], a[8], a[9]});
    const Plan& plan = plan_of(a[4]);
    const smx_paged_cache cache = cache_of(a[2], a[3], plan);
    const int64_t head_dim = cache.head_dim;
    const c10::DeviceGuard guard(plan.device);
    Tensor hold[7];
    const smx_heads k = heads_of(a[0], "k", plan, cache.kv_heads, head_dim, &hold[0]);
    const smx_heads v = heads_of(a[1], "v", plan, cache.kv_heads, head_dim, &hold[1]);
    if (given(a[6]) != given(a[7])) refuse("rope_cos= and rope_sin= go together");
    smx_heads q{};
    Tensor out;
    if (given(a[5])) {
      q = heads_of(a[5], "q", plan, -1, head_dim, &hold[2]);
      out = at::empty({plan.step.tokens, q.heads, head_dim}, plan.memory.options().dtype(at::kBFloat16));
    } else if (given(a[8])) {
      refuse("q_scale= without q=");
    }
    int32_t dtypes = 0, rope_rows = 0;
    int64_t rope_stride = 0;
    const void *cos = nullptr, *sin = nullptr;
    if (given(a[6])) {
      const Tensor& c = on_device(a[6], "rope_cos", plan.device);
      const Tensor& s = on_device(a[7], "rope_sin", plan.device);
      for (const Tensor* x : {&c, &s}) {
        const char* const name = x == &c ? "rope_cos" : "rope_sin";
        if (x->dim() != 2 || (x->size(1) != head_dim / 2 && x->size(1) != head_dim) || x->sizes() != c.sizes())
          refuse(name, " must have rows of ", head_dim / 2, " or ", head_dim, " values, got ", shape_of(*x));
        if (x->size(0) < plan.max_context)
          refuse(name, " holds ", x->size(0), " positions, the plan's requests up to ", plan.max_context);
      }
      if (c.scalar_type() != s.scalar_type() || (c.scalar_type() != at::kBFloat16 && c.scalar_type() != at::kFloat))
        refuse("RoPE tables must both be bf16 or float32");
      cos = laid_out(c, &hold[3]).data_ptr(), sin = laid_out(s, &hold[4]).data_ptr();
      rope_rows = (int32_t)std::min<int64_t>(c.size(0), INT32_MAX), rope_stride = c.size(1);
      if (c.scalar_type() == at::kFloat) dtypes |= SMX_PAGED_ROPE_F32;
    }
    const void* const q_scale = scale_of(a[8], "q_scale", plan, head_dim, SMX_PAGED_Q_SCALE_F32, &dtypes, &hold[5]);
    const void* const k_scale = scale_of(a[9], "k_scale", plan, head_dim, SMX_PAGED_K_SCALE_F32, &dtypes, &hold[6]);
    check(lib.write(&cache, plan.step.tokens, plan.step.positions, plan.slots, out.defined() ? &q : nullptr, &k, &v, cos, sin,
                    rope_rows, rope_stride, q_scale, k_scale, dtypes, (float)real(a[10]),
                    out.defined() ? out.mutable_data_ptr() : nullptr, stream_of(plan.device)));
    for (PyObject* const o : {a[2], a[3]}) written(tensor(o, "cache"));
    if (!out.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(std::move(out));
  });
}

double scale_given(PyObject* o, int64_t head_dim) {
  const double scale = given(o) ? real(o) : 1.0 / std::sqrt((double)head_dim);
  if (!(std::isfinite(scale) && scale > 0)) refuse("scale must be positive and finite, got ", scale);
  return scale;
}

int32_t window_given(PyObject* o) {
  if (!given(o)) return 0;
  if (!PyLong_Check(o)) refuse("window must be a positive number of tokens");
  return (int32_t)integer(o, "window", 1, INT32_MAX);
}

// A float32 tensor that lies dense, of this shape.
float* dense_floats(const Tensor& t, const char* name, at::IntArrayRef shape) {
  if (t.scalar_type() != at::kFloat || t.sizes() != shape || !t.is_contiguous()) {
    std::ostringstream want;
    for (size_t i = 0; i < shape.size(); ++i) want << (i ? ", " : "") << shape[i];
    refuse(name, " must be a contiguous float32 tensor of shape [", want.str(), "], got ", shape_of(t));
  }
  return t.mutable_data_ptr<float>();
}

// (q, k_cache, v_cache, plan, scale, window, out, lse) -> out
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    no_gradients({a[0], a[1], a[2], a[6], a[7]});
    const Plan& plan = plan_of(a[3]);
    const smx_paged_cache cache = cache_of(a[1], a[2], plan);
    const int64_t head_dim = cache.head_dim;
    const c10::DeviceGuard guard(plan.device);
    Tensor hold, out;
    const smx_heads q = heads_of(a[0], "q", plan, -1, head_dim, &hold);
    const double scale = scale_given(a[4], head_dim);
    const int32_t window = window_given(a[5]);
    float* const lse = given(a[7]) ? dense_floats(on_device(a[7], "lse", plan.device), "lse", {plan.step.tokens, q.heads}) : nullptr;
    smx_heads rows;
    const bool own = !given(a[6]);
    if (own) {
      out = at::empty({plan.step.tokens, q.heads, head_dim}, plan.memory.options().dtype(at::kBFloat16));
      rows = smx_heads{out.mutable_data_ptr(), q.heads * head_dim, head_dim, q.heads};
    } else {
      rows = heads_of(a[6], "out", plan, q.heads, head_dim, nullptr);
    }
    int64_t need = 0;
    check(lib.attention_bytes((int32_t)head_dim, &need));
    const Tensor workspace = at::empty({need}, plan.memory.options().dtype(at::kByte));
    check(lib.attention(&cache, &plan.step, &q, &rows, (float)scale, window, own, lse, workspace.mutable_data_ptr(), need,
                        stream_of(plan.device)));
    if (lse) written(tensor(a[7], "lse"));
    if (own) return THPVariable_Wrap(std::move(out));
    written(tensor(a[6], "out"));
    Py_INCREF(a[6]);
    return a[6];
  });
}

// (q, k_cache, key_weights, plan, lse, scale, window) -> None
PyObject* key_weights(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    no_gradients({a[0], a[1], a[2], a[4]});
    const Plan& plan = plan_of(a[3]);
    const smx_paged_cache cache = cache_of(a[1], a[1], plan);  // (values are not read)
    const c10::DeviceGuard guard(plan.device);
    Tensor hold;
    smx_heads q = heads_of(a[0], "q", plan, -1, cache.head_dim, &hold);
    // rows that are too far from each other for the kernel's offsets (heads of some 10 million tokens outside the tokens) are
    // laid out too
    if (q.token_stride > 1 << 25 || q.head_stride > (1 << 29) / std::max(1, q.heads / std::max(1, cache.kv_heads))) {
      hold = tensor(a[0], "q").clone(at::MemoryFormat::Contiguous);
      q = smx_heads{hold.mutable_data_ptr(), q.heads * (int64_t)cache.head_dim, cache.head_dim, q.heads};
    }
    const Tensor& weights = on_device(a[2], "key_weights", plan.device);
    float* const to = dense_floats(weights, "key_weights", {cache.num_pages, cache.kv_heads, cache.page_size});
    const float* const lse = dense_floats(on_device(a[4], "lse", plan.device), "lse", {plan.step.tokens, q.heads});
    const double scale = scale_given(a[5], cache.head_dim);
    const int32_t window = window_given(a[6]);
    int64_t need = 0;
    check(lib.weights_bytes(&need));
    const Tensor workspace = at::empty({need}, plan.memory.options().dtype(at::kByte));
    check(lib.weights(&cache, &plan.step, &q, lse, (float)scale, window, to, workspace.mutable_data_ptr(), need,
                      stream_of(plan.device)));
    written(weights);
    Py_RETURN_NONE;
  });
}

// (k_cache, v_cache, key_weights, context_lens, block_tables, keep, recent, max_context) -> lens
PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    no_gradients({a[0], a[1], a[2]});
    const Tensor& k = on_device(a[0], "k_cache");
    const at::Device device = k.device();
    const Tensor &v = on_device(a[1], "v_cache", device), &weights = on_device(a[2], "key_weights", device);
    const smx_paged_cache cache = cache_layout(k, v, nullptr);
    float* const received = dense_floats(weights, "key_weights", {cache.num_pages, cache.kv_heads, cache.page_size});
    const Tensor& context_lens = on_device(a[3], "context_lens", device);
    if (context_lens.dim() != 1 || !context_lens.size(0)) refuse("context_lens must hold one length per request");
    const int64_t requests = context_lens.size(0);
    const int32_t* const context = int32_list(context_lens, "context_lens", requests);
    const Tensor& tables = on_device(a[4], "block_tables", device);
    const int32_t* const entries = table_rows(tables, requests);
    const int64_t width = std::min<int64_t>(tables.size(1), INT32_MAX), stride = requests > 1 ? tables.stride(0) : width;
    const int32_t* keep_lens = nullptr;
    int64_t keep = -1;
    if (THPVariable_Check(a[5]))
      keep_lens = int32_list(on_device(a[5], "keep", device), "keep", requests);
    else
      keep = integer(a[5], "keep", 0, INT32_MAX);
    const int64_t recent = integer(a[6], "recent", 0, INT32_MAX);
    const int64_t holds = std::min<int64_t>(width * cache.page_size, SMX_PAGED_MAX_CONTEXT);
    const int64_t max_context = given(a[7]) ? integer(a[7], "max_context", 0, INT32_MAX) : holds;
    const c10::DeviceGuard guard(device);
    int64_t need = 0;
    check(lib.evict_bytes((int32_t)std::min<int64_t>(requests, INT32_MAX), cache.kv_heads, (int32_t)keep, (int32_t)max_context, &need));
    Tensor lens = at::empty({requests}, context_lens.options());
    const Tensor workspace = at::empty({need}, context_lens.options().dtype(at::kByte));
    check(lib.evict(&cache, received, (int32_t)requests, (int32_t)width, context, entries, stride, keep_lens, (int32_t)keep,
                    (int32_t)recent, (int32_t)max_context, lens.mutable_data_ptr<int32_t>(), workspace.mutable_data_ptr(), need,
                    stream_of(device)));
    for (const Tensor* x : {&k, &v, &weights}) written(*x);
    return THPVariable_Wrap(std::move(lens));
  });
}

// ---------------------------------------------------------------------------
// Rotary positions
// ---------------------------------------------------------------------------

// (x, positions, frequencies, interleaved, amplitude, norm, eps, out) -> out
PyObject* rotary(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    no_gradients({a[0], a[1], a[2], a[5], a[7]});
    const Tensor* x = &on_device(a[0], "x");
    const at::Device device = x->device();
    if ((x->scalar_type() != at::kBFloat16 && x->scalar_type() != at::kFloat) || x->dim() != 3)
      refuse("x must be bf16 or float32 heads [tokens, heads, head_dim], got ", shape_of(*x));
    const int64_t tokens = x->size(0), heads = x->size(1), head_dim = x->size(2);
    if (heads > INT32_MAX || head_dim > INT32_MAX) refuse("too many or too wide heads: ", shape_of(*x));
    int32_t flags = 0;
    if (x->scalar_type() == at::kFloat) flags |= SMX_ROTARY_F32;
    const c10::DeviceGuard guard(device);
    Tensor hold[4], out;
    const Tensor* positions = &on_device(a[1], "positions", device);
    if (positions->dim() != 1 || positions->size(0) != tokens ||
        (positions->scalar_type() != at::kInt && positions->scalar_type() != at::kLong))
      refuse("positions must be int32 or int64 of shape (", tokens, ",), got ", shape_of(*positions));
    if (!positions->is_contiguous()) positions = &(hold[0] = positions->contiguous());
    if (positions->scalar_type() == at::kLong) flags |= SMX_ROTARY_POSITIONS_I64;
    const Tensor* frequencies = &on_device(a[2], "frequencies", device);
    if (frequencies->dim() != 1 || (frequencies->scalar_type() != at::kFloat && frequencies->scalar_type() != at::kDouble))
      refuse("frequencies must be a list of float64 or float32 values, got ", shape_of(*frequencies));
    if (frequencies->size(0) < 1 || 2 * frequencies->size(0) > head_dim)
      refuse("frequencies must be 1 to head_dim / 2 = ", head_dim / 2, " values, one for each pair, got ", frequencies->size(0));
    if (!frequencies->is_contiguous()) frequencies = &(hold[1] = frequencies->contiguous());
    if (frequencies->scalar_type() == at::kFloat) flags |= SMX_ROTARY_FREQUENCIES_F32;
    const int interleaved = PyObject_IsTrue(a[3]);
    if (interleaved < 0) throw Raised();
    if (interleaved) flags |= SMX_ROTARY_INTERLEAVED;
    const void* norm = nullptr;
    if (given(a[5])) {
      const Tensor& w = on_device(a[5], "norm", device);
      if (w.dim() != 1 || w.size(0) != head_dim) refuse("norm must have shape (", head_dim, ",), got ", shape_of(w));
      const Tensor& y = laid_out(w, &hold[2]);
      if (y.scalar_type() == at::kFloat) flags |= SMX_ROTARY_NORM_F32;
      norm = y.data_ptr();
    }
    auto stride = [](const Tensor& t, int i) { return t.size(i) > 1 ? t.stride(i) : 0; };
    const bool own = !given(a[7]);
    if (own) {
      out = at::empty({tokens, heads, head_dim}, x->options());
    } else {
      out = on_device(a[7], "out", device);
      if (out.scalar_type() != x->scalar_type() || out.sizes() != x->sizes() || out.stride(2) != 1)
        refuse("out must be like x, ", shape_of(*x), ", with contiguous heads, got ", shape_of(out));
    }
    const double amplitude = real(a[4]), eps = real(a[6]);
    if (tokens) {
      if (x->stride(2) != 1) x = &(hold[3] = x->clone(at::MemoryFormat::Contiguous));
      const smx_heads from{x->data_ptr(), stride(*x, 0), stride(*x, 1), (int32_t)heads};
      const smx_heads to{out.mutable_data_ptr(), stride(out, 0), stride(out, 1), (int32_t)heads};
      check(lib.rotary((int32_t)std::min<int64_t>(tokens, INT32_MAX), (int32_t)head_dim, (int32_t)(2 * frequencies->size(0)), &from, &to,
                       positions->data_ptr(), frequencies->data_ptr(), norm, flags, (float)amplitude, (float)eps, own,
                       stream_of(device)));
    }
    if (own) return THPVariable_Wrap(std::move(out));
    written(out);
    Py_INCREF(a[7]);
    return a[7];
  });
}

// ---------------------------------------------------------------------------
// Verification of drafts
// ---------------------------------------------------------------------------

// (target, tokens, plan, accept, sample, draft) -> (tokens, counts)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    no_gradients({a[0], a[3], a[4], a[5]});
    const Plan& plan = plan_of(a[2]);
    const int64_t rows = plan.step.tokens, requests = plan.step.requests;
    const c10::DeviceGuard guard(plan.device);
    Tensor hold[5];
    const Tensor& target = on_device(a[0], "target", plan.device);
    if (target.dim() != 2 || target.size(0) != rows || !target.size(1) || target.size(1) > SMX_VERIFY_MAX_VOCAB ||
        (target.scalar_type() != at::kFloat && target.scalar_type() != at::kBFloat16))
      refuse("target must be float32 or bf16 probabilities [", rows, ", vocab], got ", shape_of(target));
    const int64_t vocab = target.size(1);
    // rows of probabilities behind each other (laid out anew where they are not)
    auto rows_of = [&](const Tensor& t, Tensor* copy) -> const Tensor& {
      if ((vocab == 1 || t.stride(1) == 1) && (rows == 1 || t.stride(0) >= vocab)) return t;
      return *copy = t.clone(at::MemoryFormat::Contiguous);
    };
    const Tensor& p = rows_of(target, &hold[0]);
    const Tensor* q = nullptr;
    if (given(a[5])) {
      const Tensor& draft = on_device(a[5], "draft", plan.device);
      if (draft.sizes() != target.sizes() || draft.scalar_type() != target.scalar_type())
        refuse("draft must be like target, ", shape_of(target), ", got ", shape_of(draft));
      q = &rows_of(draft, &hold[1]);
    }
    const Tensor* tokens = &on_device(a[1], "tokens", plan.device);
    if (tokens->dim() != 1 || tokens->size(0) != rows || (tokens->scalar_type() != at::kInt && tokens->scalar_type() != at::kLong))
      refuse("tokens must be int32 or int64 of shape (", rows, ",), got ", shape_of(*tokens));
    if (!tokens->is_contiguous()) tokens = &(hold[2] = tokens->contiguous());
    const float* numbers[2];
    for (int i = 0; i < 2; ++i) {
      const char* const name = i ? "sample" : "accept";
      const int64_t length = i ? requests : rows;
      const Tensor* u = &on_device(a[3 + i], name, plan.device);
      if (u->dim() != 1 || u->size(0) != length || u->scalar_type() != at::kFloat)
        refuse(name, " must be float32 of shape (", length, ",), got ", shape_of(*u));
      if (!u->is_contiguous()) u = &(hold[3 + i] = u->contiguous());
      numbers[i] = u->const_data_ptr<float>();
    }
    int32_t flags = 0;
    if (target.scalar_type() == at::kBFloat16) flags |= SMX_VERIFY_BF16;
    if (tokens->scalar_type() == at::kLong) flags |= SMX_VERIFY_TOKENS_I64;
    Tensor out = at::empty({rows}, tokens->options()), counts = at::empty({requests}, plan.memory.options());
    int64_t need = 0;
    check(lib.verify_bytes((int32_t)requests, (int32_t)vocab, &need));
    const Tensor workspace = at::empty({need}, plan.memory.options().dtype(at::kByte));
    check(lib.verify(&plan.step, (int32_t)vocab, p.data_ptr(), rows > 1 ? p.stride(0) : vocab, q ? q->data_ptr() : nullptr,
                     q && rows > 1 ? q->stride(0) : vocab, tokens->data_ptr(), numbers[0], numbers[1], flags, out.mutable_data_ptr(),
                     counts.mutable_data_ptr<int32_t>(), workspace.mutable_data_ptr(), need, stream_of(plan.device)));
    PyObject* const result = PyTuple_New(2);
    if (!result) throw Raised();
    PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(out)));
    PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(counts)));
    return result;
  });
}

// One of the two tensors of a weight laid out for int4_matmul.
void laid_out_for(const Tensor& t, const char* name, const at::Device& device, int64_t numel) {
  if (t.scalar_type() != at::kInt || t.device() != device || !t.is_contiguous() || t.numel() != numel)
    refuse(name, " is not that of int4_weight_layout (", numel, " contiguous int32 values on ", device, "), got ", shape_of(t), " on ",
           t.device());
}

// (x, codes, scales, k, n, group, swiglu, zeros, epilogue, residual, bias) -> the product
PyObject* int4(PyObject*, PyObject* const* a, Py_ssize_t) {
  return guarded([&]() -> PyObject* {
    no_gradients({a[0], a[9], a[10]});
    const Tensor &codes = tensor(a[1], "w.codes"), &scales = tensor(a[2], "w.scales");
    const at::Device device = codes.device();
    const Tensor* x = &on_device(a[0], "x");
    on_device(a[0], "x", device);
    // The operand's fields are a program's to change: its memory is what the kernels will read of it
    const int64_t k = integer(a[3], "w.k", 1, 1 << 22), width = integer(a[4], "w.n", 1, 1 << 24);
    const int64_t group = integer(a[5], "w.group", 32, 128);
    const int32_t swiglu = (int32_t)integer(a[6], "w.swiglu", 0, 1), zeros = (int32_t)integer(a[7], "w.zeros", 0, 1);
    if (128 % group) refuse("w.group must be 32, 64 or 128, got ", group);
    const int64_t k_tiles = (k + 127) / 128, columns = swiglu ? 2 * ((width / 2 + 15) / 16) : 2 * ((width + 31) / 32);
    laid_out_for(codes, "w.codes", device, columns * k_tiles * 256);
    laid_out_for(scales, "w.scales", device, columns * k_tiles * 16 * (128 / group));
    const int32_t epilogue = (int32_t)PyLong_AsLong(a[8]);
    if (PyErr_Occurred()) throw Raised();
    const smx_int4_weight w{codes.data_ptr(), scales.data_ptr(), k, width, (int32_t)group, swiglu, zeros};
    if (x->scalar_type() != at::kBFloat16 || x->dim() != 2) refuse("x must be a bf16 matrix, got ", shape_of(*x));
    const int64_t m = x->size(0), n = w.swiglu ? width / 2 : width;
    if (x->size(1) != k) refuse("inner dimensions disagree: ", x->size(1), " vs ", k);
    if ((epilogue == SMX_EPI_RESIDUAL_ADD) != given(a[9])) refuse("residual= goes with the residual_add epilogue");
    if ((epilogue == SMX_EPI_BIAS_ADD) != given(a[10])) refuse("bias= goes with the bias_add epilogue");
    const c10::DeviceGuard guard(device);
    Tensor hold[2];
    const Tensor* extra = nullptr;
    int64_t extra_row = 0;
    if (epilogue == SMX_EPI_RESIDUAL_ADD || epilogue == SMX_EPI_BIAS_ADD) {
      const bool residual = epilogue == SMX_EPI_RESIDUAL_ADD;
      const char* const name = residual ? "residual" : "bias";
      extra = &on_device(a[residual ? 9 : 10], name, device);
      if (residual ? extra->dim() != 2 || extra->size(0) != m || extra->size(1) != n : extra->dim() != 1 || extra->size(0) != n)
        refuse(name, " shape ", shape_of(*extra), " does not fit the output [", m, ", ", n, "]");
      if (extra->scalar_type() != at::kBFloat16 && extra->scalar_type() != at::kFloat) {
        hold[0] = extra->to(at::kFloat);
        extra = &hold[0];
      }
      if ((n > 1 && extra->stride(-1) != 1) || (residual && m > 1 && extra->stride(0) < n)) {
        hold[0] = extra->clone(at::MemoryFormat::Contiguous);
        extra = &hold[0];
      }
      extra_row = residual && m > 1 ? extra->stride(0) : n;
    }
    Tensor out = at::empty({m, n}, x->options());
    if (m) {
      int64_t row = m > 1 ? x->stride(0) : k;  // a single row has no stride
      if (x->stride(1) != 1 || row % 8 || row < k || row > 1 << 24 || !aligned16(x->data_ptr())) {
        hold[1] = x->clone(at::MemoryFormat::Contiguous);
        x = &hold[1];
        row = k;
      }
      int64_t need = 0;
      check(lib.int4_bytes(&w, m, &need));
      Tensor workspace;
      if (need) workspace = at::empty({need}, x->options().dtype(at::kByte));
      check(lib.int4(&w, m, x->data_ptr(), row, epilogue, extra ? extra->data_ptr() : nullptr, extra_row,
                     extra && extra->scalar_type() == at::kFloat, out.mutable_data_ptr(), n,
                     need ? workspace.mutable_data_ptr() : nullptr, need, stream_of(device)));
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// (addresses of the C ABI's entry points in Library's order, raw_stream)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kEntries = 14;
  void* at[kEntries];
  if (n != kEntries + 1) {
    PyErr_SetString(PyExc_TypeError, "the addresses of the library's entry points and the stream lookup");
    return nullptr;
  }
  for (int i = 0; i < kEntries; ++i) at[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  int i = 0;
  auto next = [&](auto& entry) { entry = reinterpret_cast<std::decay_t<decltype(entry)>>(at[i++]); };
  next(lib.plan), next(lib.write), next(lib.attention), next(lib.attention_bytes), next(lib.weights), next(lib.weights_bytes);
  next(lib.evict), next(lib.evict_bytes), next(lib.rotary), next(lib.verify), next(lib.verify_bytes), next(lib.int4);
  next(lib.int4_bytes), next(lib.error);
  Py_INCREF(a[kEntries]);
  lib.raw_stream = a[kEntries];
  Py_RETURN_NONE;
}

template <class F>
PyCFunction method(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f));
}

PyMethodDef methods[] = {{"plan", method(plan), METH_FASTCALL, nullptr},
                         {"write", method(write), METH_FASTCALL, nullptr},
                         {"attention", method(attention), METH_FASTCALL, nullptr},
                         {"key_weights", method(key_weights), METH_FASTCALL, nullptr},
                         {"evict", method(evict), METH_FASTCALL, nullptr},
                         {"rotary", method(rotary), METH_FASTCALL, nullptr},
                         {"verify", method(verify), METH_FASTCALL, nullptr},
                         {"int4", method(int4), METH_FASTCALL, nullptr},
                         {"bind", method(bind), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&module); }
