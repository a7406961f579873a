// The binding of the row kernels around the attention (recap_b200/block.py): checks the tensors of a call,
// allocates its outputs, fills the host struct of the C ABI and calls it on the tensors' device and its
// current stream.  In C++ because these kernels take a few microseconds on few tokens, where the same
// checks in Python took twice the launch: a call of rotate_qk on one token takes the host 6.2 us here,
// 12.8 us through ctypes (of it 3.3 us the launch, 2.7 us two allocations).  The entry points come from librecap_b200.so by address (bind()).
//
// Refused arguments raise ValueError, inputs that would lose their gradient RuntimeError; no C++
// exception leaves a function.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_like.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cstring>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/recap_b200.h"

namespace {

using at::Tensor;

using RotateFn = int (*)(const recap_rotate_qk_args*, const recap_rotary*, void*);
using NormFn = int (*)(const recap_norm_rows_args*, void*);
RotateFn g_rotate = nullptr;
NormFn g_norm = nullptr;
PyObject* g_check = nullptr;  // raises the error of a return code: check(rc, name)

PyObject *s_code, *s_eps, *s_weight, *s_bias, *s_spec;  // attribute names

struct Refuse {  // becomes a ValueError
  std::string what;
};
struct Recorded {};  // becomes the RuntimeError of an input that requires a gradient
struct Tangent {};   // becomes the RuntimeError of a dual input
struct Raised {};    // a Python error is set

[[noreturn]] void refuse(std::string what) { throw Refuse{std::move(what)}; }

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + (s.size() == 1 ? ",)" : ")");
}

// A tensor argument, or null for None.
const Tensor* tensor(PyObject* o, const char* what) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse(std::string(what) + " must be a tensor");
  return &THPVariable_Unpack(o);
}
const Tensor& given(PyObject* o, const char* what) {
  const Tensor* t = tensor(o, what);
  if (t == nullptr) refuse(std::string(what) + " must be a tensor");
  return *t;
}

// Neither a recorded input of a backward pass nor the tangent of a forward one, which is not cut by no_grad().
void no_gradient(const Tensor* t) {
  if (t == nullptr) return;
  if (t->requires_grad() && c10::GradMode::is_enabled()) throw Recorded{};
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t->_fw_grad(0).defined()) throw Tangent{};
}

int type_of(at::ScalarType t, const char* what) {
  if (t == at::kBFloat16) return RECAP_TYPE_BF16;
  if (t == at::kHalf) return RECAP_TYPE_F16;
  if (t == at::kFloat) return RECAP_TYPE_F32;
  refuse(std::string(what) + " must be bfloat16, float16 or float32, not " + c10::toString(t));
}

// Rows, modulations and parameters are moved 16 bytes at a time.
bool base_aligned(const Tensor* t) { return t == nullptr || reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16 == 0; }
void aligned(const Tensor* t, const char* what) {
  if (t == nullptr) return;
  bool good = base_aligned(t);
  const int64_t unit = 16 / static_cast<int64_t>(t->element_size());
  for (int64_t i = 0; i + 1 < t->dim(); ++i) good = good && (t->size(i) <= 1 || t->stride(i) % unit == 0);
  if (!good) refuse(std::string(what) + " must have a base and strides of multiples of 16 bytes");
}

at::ScalarType dtype_or(PyObject* o, at::ScalarType otherwise) {
  if (o == Py_None) return otherwise;
  if (!THPDtype_Check(o)) refuse("out_dtype must be a dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}

struct Attribute {  // a new reference, released at the end; `what`: the refusal of an object without it
  PyObject* o;
  Attribute(PyObject* of, PyObject* name, const char* what) : o(PyObject_GetAttr(of, name)) {
    if (o != nullptr) return;
    if (!PyErr_ExceptionMatches(PyExc_AttributeError)) throw Raised{};
    PyErr_Clear();
    refuse(what);
  }
  ~Attribute() { Py_XDECREF(o); }
  Attribute(const Attribute&) = delete;
};

constexpr const char* kNotANorm = "a norm must be a Norm";
constexpr const char* kNotARotary = "rotary must be an AxialRotary";

// A norm's kind, epsilon and parameters of n values each (recap_b200.Norm); holds the parameters.
struct NormParams {
  int code = RECAP_NORM_NONE, type = 0;
  float eps = 0.f;
  const void *weight = nullptr, *bias = nullptr;
  const Tensor* tensors[2] = {nullptr, nullptr};  // weight, bias
  std::optional<Attribute> held[2];

  void check_aligned() const {
    for (int i = 0; i < 2; ++i)
      if (!base_aligned(tensors[i])) refuse(std::string("a norm's ") + (i == 0 ? "weight" : "bias") + " must have a base of a multiple of 16 bytes");
  }

  void read(PyObject* norm, int64_t n_head, int64_t n_across, const at::Device& device) {
    {
      const Attribute c(norm, s_code, kNotANorm), e(norm, s_eps, kNotANorm);
      code = static_cast<int>(integer(c.o));
      eps = static_cast<float>(PyFloat_AsDouble(e.o));
      if (PyErr_Occurred()) throw Raised{};
    }
    const int64_t n = code == RECAP_NORM_RMS_ACROSS ? n_across : n_head;
    bool typed = false;
    for (int i = 0; i < 2; ++i) {
      const char* what = i == 0 ? "norm's weight" : "norm's bias";
      held[i].emplace(norm, i == 0 ? s_weight : s_bias, kNotANorm);
      const Tensor* t = tensors[i] = tensor(held[i]->o, what);
      if (t == nullptr) continue;
      no_gradient(t);
      if (t->numel() != n || !t->is_contiguous()) refuse(std::string("a ") + what + " must be " + std::to_string(n) + " contiguous values");
      if (t->device() != device) refuse(std::string("a ") + what + " is on " + t->device().str() + ", the rows on " + device.str());
      const int code_of = type_of(t->scalar_type(), what);
      if (typed && code_of != type) refuse("a norm's weight and bias differ in type");
      type = code_of;
      typed = true;
      (i == 0 ? weight : bias) = t->const_data_ptr();
    }
  }
};

// ------------------------------------------------------------------------------ overlap

// Whether two tensors share no element, as far as that can be told.  Dim by dim, the widest steps first: x's elements lie at
// i step + u and y's at away + j step + v, with u and v what the dims within add, each tensor's by its own strides.  Where
// the spans of u and of v, moved by what `away` leaves over a step, lie in one window of a step, elements are equal only for i
// and j that step alike: the tensors are apart if no i and j do, or if those spans do not meet; else the dims within tell.  So
// the parts of a packed projection or of a joint sequence are told apart, and so are tensors whose dims within differ.
bool apart(const Tensor& x, const Tensor& y) {
  if (x.numel() == 0 || y.numel() == 0) return true;
  const int64_t size = static_cast<int64_t>(x.element_size());
  const auto span = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    const int64_t at = reinterpret_cast<int64_t>(t.const_data_ptr());
    return std::pair<int64_t, int64_t>(at, at + (last + 1) * static_cast<int64_t>(t.element_size()));
  };
  const auto [x0, x1] = span(x);
  const auto [y0, y1] = span(y);
  if (x1 <= y0 || y1 <= x0) return true;
  if (x.dim() != y.dim() || x.scalar_type() != y.scalar_type() || (y0 - x0) % size) return false;
  std::vector<std::array<int64_t, 4>> dims;  // strides, sizes; a dim of one element takes the other's stride
  for (int64_t i = 0; i < x.dim(); ++i)
    if (x.size(i) > 1 || y.size(i) > 1)
      dims.push_back({x.size(i) > 1 ? x.stride(i) : y.stride(i), y.size(i) > 1 ? y.stride(i) : x.stride(i), x.size(i), y.size(i)});
  std::sort(dims.rbegin(), dims.rend());
  int64_t away = (y0 - x0) / size;
  for (size_t i = 0; i < dims.size(); ++i) {
    const auto [step, other, n, m] = dims[i];
    if (step != other || step == 0) return false;
    int64_t inner_x = 1, inner_y = 1;
    for (size_t j = i + 1; j < dims.size(); ++j) {
      inner_x += (dims[j][2] - 1) * dims[j][0];
      inner_y += (dims[j][3] - 1) * dims[j][1];
    }
    int64_t at = away / step - (away % step < 0);
    int64_t rest = 0;
    bool found = false;
    for (int k = 0; k < 2 && !found; ++k) {
      rest = away - (at + k) * step;
      if (std::max(inner_x, rest + inner_y) - std::min<int64_t>(0, rest) <= step) {
        at += k;
        found = true;
      }
    }
    if (!found) return false;
    if (at >= n || -at >= m) return true;
    if (rest >= inner_x || rest + inner_y <= 0) return true;
    away = rest;
  }
  return false;
}

// Whether a tensor holds each element once: each stride goes past all that the dims of smaller strides span.
bool distinct(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;  // strides, sizes
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) dims.push_back({t.stride(i), t.size(i)});
  std::sort(dims.begin(), dims.end());
  int64_t inner = 1;
  for (const auto& [step, n] : dims) {
    if (step < inner) return false;
    inner += (n - 1) * step;
  }
  return true;
}

// Whether two tensors of one shape are the same elements in the same places.
bool same(const Tensor& x, const Tensor& y) {
  for (int64_t i = 0; i < x.dim(); ++i)
    if (x.size(i) > 1 && x.stride(i) != y.stride(i)) return false;
  return x.const_data_ptr() == y.const_data_ptr() && x.scalar_type() == y.scalar_type();
}

// An output holds each element once and overlaps none of `inputs`, but for `own`, the input that it may replace: every element
// of that is read by the thread that writes it, before it does, also where the call has it in another of these places.
void check_output(const Tensor* o, const Tensor* own, std::initializer_list<const Tensor*> inputs) {
  if (o == nullptr) return;
  if (o->numel() != 0 && !distinct(*o)) refuse("an output holds an element twice (an expanded tensor, or strides within one another)");
  for (const Tensor* x : inputs)
    if (x != nullptr && !(x == own && same(*o, *x)) && !apart(*o, *x))
      refuse("an output overlaps an input (it may only be that input itself)");
}

// Nor may it overlap what other threads read, or this one after the output is written.
void check_clear(const Tensor* o, std::initializer_list<const Tensor*> inputs) {
  if (o == nullptr) return;
  for (const Tensor* x : inputs)
    if (x != nullptr && !apart(*o, *x)) refuse("an output overlaps an input that is read beside it");
}

Tensor allocate(const Tensor& like, at::ScalarType dtype) {
  at::AutoDispatchBelowADInplaceOrView below;
  return dtype == like.scalar_type() ? at::empty_like(like) : at::empty_like(like, like.options().dtype(dtype));
}

// A given tensor is written: autograd's saved copies of it are out of date.
void written(const Tensor* t) {
  if (t != nullptr && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

void raise_code(int rc, const char* name) {
  PyObject* r = PyObject_CallFunction(g_check, "is", rc, name);
  Py_XDECREF(r);
  if (r != nullptr) PyErr_SetString(PyExc_RuntimeError, name);
  throw Raised{};
}

PyObject* pair(const Tensor* a, const Tensor* b) {
  PyObject* x = a != nullptr ? THPVariable_Wrap(*a) : Py_NewRef(Py_None);
  PyObject* y = x == nullptr ? nullptr : b != nullptr ? THPVariable_Wrap(*b) : Py_NewRef(Py_None);
  if (y == nullptr) {
    Py_XDECREF(x);
    throw Raised{};
  }
  PyObject* t = PyTuple_New(2);
  if (t == nullptr) {
    Py_DECREF(x);
    Py_DECREF(y);
    throw Raised{};
  }
  PyTuple_SET_ITEM(t, 0, x);
  PyTuple_SET_ITEM(t, 1, y);
  return t;
}

// Runs `body`, turning what it throws into Python errors.
template <typename F>
PyObject* guarded(F body) {
  try {
    return body();
  } catch (const Refuse& r) {
    PyErr_SetString(PyExc_ValueError, r.what.c_str());
  } catch (const Recorded&) {
    PyErr_SetString(PyExc_RuntimeError, "this operator has no backward pass: call it under torch.no_grad()");
  } catch (const Tangent&) {
    PyErr_SetString(PyExc_RuntimeError, "this operator has no forward-mode derivative: give it the primal of a dual tensor");
  } catch (const Raised&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// ------------------------------------------------------------------------------ rotate_qk

// rotate_qk(query, key, rotary, query_norm, key_norm, positions, first_token, out_dtype, q_out, k_out)
PyObject* rotate_qk(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 10) refuse("rotate_qk takes 10 arguments");
    const Tensor& query = given(args[0], "query");
    const Tensor* key = tensor(args[1], "key");
    recap_rotate_qk_args p;
    std::memset(&p, 0, sizeof(p));
    const auto heads_of = [](const Tensor& t, const char* what) {
      if (t.dim() != 4 || (t.stride(3) != 1 && t.size(3) > 1))
        refuse(std::string(what) + " must be [batch, heads, sequence, dim] with dim contiguous");
    };
    heads_of(query, "query");
    const int64_t b = query.size(0), hq = query.size(1), s = query.size(2), d = query.size(3);
    int64_t hk = 0;
    const at::Device device = query.device();
    if (d % 8 || d < 8 || d > 256 || hq < 1) refuse("dim must be a multiple of 8 up to 256, and heads positive");
    if (key != nullptr) {
      heads_of(*key, "key");
      hk = key->size(1);
      if (key->size(0) != b || key->size(2) != s || key->size(3) != d) refuse("query and key differ in batch, sequence or dim");
      if (key->scalar_type() != query.scalar_type() || key->device() != device) refuse("query and key differ in dtype or device");
      if (hk < 1) refuse("key has no heads");
    }
    if (b * s > 0x7fffffff || std::max(hq, hk) > 0x7fffffff - 31) refuse("more than 2^31 - 1 tokens or 2^31 - 32 heads");
    no_gradient(&query);
    no_gradient(key);
    p.in_type = type_of(query.scalar_type(), "query");
    const Tensor* q_given = tensor(args[8], "out");
    const Tensor* k_given = tensor(args[9], "out");
    at::ScalarType out_dtype = dtype_or(args[7], q_given != nullptr ? q_given->scalar_type() : query.scalar_type());
    if (out_dtype != query.scalar_type() && out_dtype != at::kBFloat16) refuse("the output has the inputs' dtype or bfloat16");
    p.out_type = type_of(out_dtype, "out");

    NormParams qn, kn;
    if (args[3] != Py_None || args[4] != Py_None) {
      if (args[3] == Py_None || (key != nullptr && args[4] == Py_None)) refuse("query and key are both normalised or neither");
      qn.read(args[3], d, hq * d, device);
      if (key != nullptr) kn.read(args[4], d, hk * d, device);
      if (key != nullptr && kn.code != qn.code) refuse("the query's and the key's norm differ in kind");
      if (qn.code == RECAP_NORM_RMS_ACROSS && std::max(hq, hk) > (d <= 64 ? 256 : d <= 128 ? 128 : 64))
        refuse("too many heads of " + std::to_string(d) + " dims for a norm across heads");
      const bool q_has = qn.weight || qn.bias, k_has = kn.weight || kn.bias;
      if (q_has && k_has && qn.type != kn.type) refuse("the norms' weights differ in type");
      p.norm = qn.code;
      p.weight_type = k_has ? kn.type : qn.type;
      p.q_weight = qn.weight, p.q_bias = qn.bias, p.k_weight = kn.weight, p.k_bias = kn.bias;
      p.q_eps = qn.eps, p.k_eps = kn.eps;
    }

    const recap_rotary* rotary = nullptr;
    const Tensor* positions = tensor(args[5], "positions");
    p.first_token = integer(args[6]);
    if (args[2] != Py_None) {
      const Attribute spec(args[2], s_spec, kNotARotary);  // (address, head dim, sequence tokens of the grid or -1)
      if (!PyTuple_Check(spec.o) || PyTuple_GET_SIZE(spec.o) != 3) refuse(kNotARotary);
      rotary = reinterpret_cast<const recap_rotary*>(integer(PyTuple_GET_ITEM(spec.o, 0)));
      const int64_t head_dim = integer(PyTuple_GET_ITEM(spec.o, 1)), tokens = integer(PyTuple_GET_ITEM(spec.o, 2));
      if (head_dim != d) refuse("rotary positions of " + std::to_string(head_dim) + " dims on heads of " + std::to_string(d));
      if (tokens >= 0) {
        if (positions != nullptr) refuse("positions are given by the rotary's grid");
        if (p.first_token < 0 || p.first_token > tokens - s)
          refuse("tokens " + std::to_string(p.first_token) + ".." + std::to_string(p.first_token + s) +
                 " outside the sequence of " + std::to_string(tokens));
      } else {
        if (p.first_token != 0) refuse("first_token belongs to a grid");
        if (positions == nullptr) refuse("a rotary without a grid needs positions");
        const at::ScalarType t = positions->scalar_type();
        if (t != at::kInt && t != at::kLong) refuse("positions must be int32 or int64");
        const int64_t nd = positions->dim();
        if ((nd != 2 && nd != 3) || (nd == 3 && positions->size(0) != 1 && positions->size(0) != b) ||
            positions->size(nd - 2) != s || positions->size(nd - 1) != rotary->axes)
          refuse("positions must be [batch or 1, sequence, axes]");
        if (positions->device() != device) refuse("positions are on " + positions->device().str() + ", the rows on " + device.str());
        p.position_bits = t == at::kLong ? 64 : 32;
        p.position_strides[0] = nd == 3 && positions->size(0) > 1 ? positions->stride(0) : 0;
        p.position_strides[1] = positions->stride(nd - 2);
        p.position_strides[2] = positions->stride(nd - 1);
        p.positions = positions->const_data_ptr();
      }
    } else if (positions != nullptr || p.first_token != 0) {
      refuse("positions and first_token need a rotary");
    }

    Tensor q_new, k_new;
    if (q_given != nullptr) {
      if (key != nullptr && k_given == nullptr) refuse("out must match query and key, dim contiguous");
      for (const auto& [o, x] : {std::pair(q_given, &query), std::pair(key != nullptr ? k_given : nullptr, key)}) {
        if (o == nullptr) continue;
        if (o->sizes() != x->sizes() || o->device() != device || o->stride(3) != 1)
          refuse("out must match query and key, dim contiguous");
        if (o->scalar_type() != out_dtype) refuse("out differs in dtype");
        no_gradient(o);
      }
      const Tensor* k_to = key != nullptr ? k_given : nullptr;
      check_output(q_given, &query, {&query});
      check_output(k_to, key, {key});
      // query and key are turned by different blocks
      check_clear(q_given, {key, k_to, qn.tensors[0], qn.tensors[1], kn.tensors[0], kn.tensors[1], positions});
      check_clear(k_to, {&query, qn.tensors[0], qn.tensors[1], kn.tensors[0], kn.tensors[1], positions});
    } else if (k_given != nullptr) {
      refuse("out must match query and key, dim contiguous");
    }
    if (b != 0 && s != 0) {
      aligned(&query, "query");
      aligned(key, "key");
      aligned(q_given, "the query's out");
      if (key != nullptr) aligned(k_given, "the key's out");
      for (const NormParams* n : {&qn, &kn}) n->check_aligned();
    }
    if (!query.is_cuda()) refuse("rotate_qk runs on CUDA tensors only");
    const c10::cuda::CUDAGuard current(device);
    if (q_given == nullptr) {
      q_new = allocate(query, out_dtype);
      if (key != nullptr) k_new = allocate(*key, out_dtype);
    }
    const Tensor& q_out = q_given != nullptr ? *q_given : q_new;
    const Tensor* k_out = key == nullptr ? nullptr : q_given != nullptr ? k_given : &k_new;
    if (b != 0 && s != 0) {
      p.q = query.const_data_ptr();
      p.q_out = q_out.data_ptr();
      for (int i = 0; i < 3; ++i) {
        p.strides[i] = query.stride(i);
        p.strides[6 + i] = q_out.stride(i);
      }
      if (key != nullptr) {
        p.k = key->const_data_ptr();
        p.k_out = k_out->data_ptr();
        for (int i = 0; i < 3; ++i) {
          p.strides[3 + i] = key->stride(i);
          p.strides[9 + i] = k_out->stride(i);
        }
      }
      p.batch = static_cast<int32_t>(b);
      p.q_heads = static_cast<int32_t>(hq);
      p.k_heads = static_cast<int32_t>(hk);
      p.S = static_cast<int32_t>(s);
      p.D = static_cast<int32_t>(d);
      const int rc = g_rotate(&p, rotary, c10::cuda::getCurrentCUDAStream(device.index()).stream());
      if (rc != RECAP_OK) raise_code(rc, "recap_rotate_qk");
      written(q_given);
      if (key != nullptr) written(k_given);
    }
    return pair(&q_out, k_out);
  });
}

// ------------------------------------------------------------------------------ norm_rows

// norm_rows(name, x, branch, gate, branch_norm, norm, scale, shift, x_out, h_out, h_dtype) -> (sum, norm); the name is
// "gated_residual", with a branch, or "modulated_norm", without
PyObject* norm_rows(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 11) refuse("norm_rows takes 11 arguments");
    const Tensor& x = given(args[1], "rows");
    const bool with_branch = PyUnicode_CompareWithASCIIString(args[0], "gated_residual") == 0;
    const Tensor* branch = with_branch ? &given(args[2], "branch") : nullptr;
    recap_norm_rows_args p;
    std::memset(&p, 0, sizeof(p));
    const int64_t nd = x.dim();
    if (nd != 2 && nd != 3) refuse("rows are [batch, tokens, channels] or [tokens, channels]");
    const int64_t c = x.size(nd - 1), s = x.size(nd - 2), b = nd == 3 ? x.size(0) : 1;
    if (c % 8 || c < 8 || c > 16384) refuse("channels must be a multiple of 8 up to 16384");
    if (b * s > 0x7fffffff) refuse("more than 2^31 - 1 tokens");
    const at::Device device = x.device();
    const Tensor* x_given = tensor(args[8], "out");
    const Tensor* h_given = tensor(args[9], "out");
    const bool with_norm = args[5] != Py_None;
    if (!with_norm && !with_branch) refuse("a norm is needed");
    if (!with_norm && (args[6] != Py_None || args[7] != Py_None)) refuse("scale and shift belong to a norm");
    if (!with_norm && h_given != nullptr) refuse("out of a norm that is not asked for");
    const at::ScalarType h_dtype =
        with_branch ? branch->scalar_type() : dtype_or(args[10], h_given != nullptr ? h_given->scalar_type() : x.scalar_type());
    p.x_type = type_of(x.scalar_type(), "rows");
    p.h_type = type_of(h_dtype, with_branch ? "branch" : "the norm's output");
    if (p.h_type != p.x_type && p.x_type != RECAP_TYPE_F32) refuse("only float32 rows have a norm or a branch of another type");
    const auto rows = [&](const Tensor& t, const char* what, int64_t* strides) {
      if (t.sizes() != x.sizes())
        refuse(std::string(what) + " has shape " + shape_text(t.sizes()) + ", expected " + shape_text(x.sizes()));
      if (t.device() != device) refuse(std::string(what) + " is on " + t.device().str() + ", the rows on " + device.str());
      if (t.stride(nd - 1) != 1) refuse(std::string(what) + " needs contiguous channels");
      no_gradient(&t);
      strides[0] = nd == 3 ? t.stride(0) : 0;
      strides[1] = t.stride(nd - 2);
    };
    rows(x, "rows", p.strides);
    if (with_branch) rows(*branch, "branch", p.strides + 2);

    const Tensor* mods[3] = {tensor(args[6], "scale"), tensor(args[7], "shift"), tensor(args[3], "gate")};
    const char* names[3] = {"scale", "shift", "gate"};
    const void** to[3] = {&p.scale, &p.shift, &p.gate};
    bool typed = false;
    for (int i = 0; i < 3; ++i) {
      const Tensor* t = mods[i];
      if (t == nullptr) continue;
      if (t->device() != device) refuse(std::string(names[i]) + " is on " + t->device().str() + ", the rows on " + device.str());
      no_gradient(t);
      const int type = type_of(t->scalar_type(), "modulations");
      if (typed && type != p.mod_type) refuse("scale, shift and gate differ in type");
      p.mod_type = type;
      typed = true;
      const int64_t md = t->dim();
      if (md < 1 || t->size(md - 1) != c || t->stride(md - 1) != 1)
        refuse(std::string(names[i]) + " needs " + std::to_string(c) + " contiguous channels");
      // one vector, or the rows' dims with size 1 where it is shared
      if (md > 1) {
        const int64_t ms = md == nd ? t->size(nd - 2) : 0, mb = md == nd && nd == 3 ? t->size(0) : 1;
        if (md != nd || (ms != 1 && ms != s) || (mb != 1 && mb != b))
          refuse(std::string(names[i]) + " has shape " + shape_text(t->sizes()) + ", which does not spread over " +
                 shape_text(x.sizes()));
        p.mod_strides[2 * i] = nd == 3 && mb > 1 ? t->stride(0) : 0;
        p.mod_strides[2 * i + 1] = ms > 1 ? t->stride(nd - 2) : 0;
      }
      *to[i] = t->const_data_ptr();
    }

    NormParams n, bn;
    if (with_norm) n.read(args[5], c, c, device);
    if (args[4] != Py_None) bn.read(args[4], c, c, device);
    if (n.code == RECAP_NORM_RMS_ACROSS || bn.code == RECAP_NORM_RMS_ACROSS) refuse("a norm across heads belongs to rotate_qk");
    p.norm = n.code, p.weight = n.weight, p.bias = n.bias, p.weight_type = n.type, p.eps = n.eps;
    p.branch_norm = bn.code, p.branch_weight = bn.weight, p.branch_bias = bn.bias, p.branch_weight_type = bn.type;
    p.branch_eps = bn.eps;

    if (x_given != nullptr || h_given != nullptr) {
      int64_t ignored[2];
      if (x_given != nullptr) {
        if (x_given->scalar_type() != x.scalar_type()) refuse("the sum has the residual's dtype");
        rows(*x_given, "out", ignored);
      }
      if (h_given != nullptr) {
        if (h_given->scalar_type() != h_dtype) refuse("the norm's out differs in dtype");
        rows(*h_given, "out", ignored);
      }
      check_output(x_given, &x, {&x, branch, mods[2]});
      check_output(h_given, with_branch ? branch : &x, {&x, branch, mods[0], mods[1], mods[2]});
      // the sum is stored before the norm's modulations are read
      check_clear(x_given, {h_given, mods[0], mods[1], n.tensors[0], n.tensors[1], bn.tensors[0], bn.tensors[1]});
      check_clear(h_given, {n.tensors[0], n.tensors[1], bn.tensors[0], bn.tensors[1]});
    }
    if (b != 0 && s != 0) {
      aligned(&x, with_branch ? "residual" : "x");
      aligned(branch, "branch");
      for (int i = 0; i < 3; ++i) aligned(mods[i], names[i]);
      if (with_branch) aligned(x_given, "the sum's out");
      aligned(h_given, "the norm's out");
      for (const NormParams* params : {&n, &bn}) params->check_aligned();
    }
    if (!x.is_cuda()) refuse(std::string(PyUnicode_AsUTF8(args[0])) + " runs on CUDA tensors only");
    const c10::cuda::CUDAGuard current(device);
    Tensor x_new, h_new;
    const Tensor *x_out = nullptr, *h_out = nullptr;
    const auto place = [&](const Tensor& t, int64_t* strides) {
      strides[0] = nd == 3 ? t.stride(0) : 0;
      strides[1] = t.stride(nd - 2);
      return t.data_ptr();
    };
    if (with_branch) {
      if (x_given == nullptr) x_new = allocate(x, x.scalar_type());
      x_out = x_given != nullptr ? x_given : &x_new;
      p.branch = branch->const_data_ptr();
      p.x_out = place(*x_out, p.strides + 4);
    }
    if (with_norm) {
      if (h_given == nullptr) h_new = allocate(with_branch ? *branch : x, h_dtype);
      h_out = h_given != nullptr ? h_given : &h_new;
      p.h = place(*h_out, p.strides + 6);
    }
    if (b != 0 && s != 0) {
      p.x = x.const_data_ptr();
      p.batch = static_cast<int32_t>(b);
      p.S = static_cast<int32_t>(s);
      p.C = static_cast<int32_t>(c);
      const int rc = g_norm(&p, c10::cuda::getCurrentCUDAStream(device.index()).stream());
      if (rc != RECAP_OK) raise_code(rc, "recap_norm_rows");
      if (with_branch) written(x_given);
      written(h_given);
    }
    return pair(x_out, h_out);
  });
}

// apart(x, y): the overlap test of the outputs.
PyObject* py_apart(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 2) refuse("apart takes 2 tensors");
    return PyBool_FromLong(apart(given(args[0], "x"), given(args[1], "y")));
  });
}

// bind(recap_rotate_qk, recap_norm_rows, check): the library's entry points by address.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    if (n_args != 3) refuse("bind takes 3 arguments");
    g_rotate = reinterpret_cast<RotateFn>(integer(args[0]));
    g_norm = reinterpret_cast<NormFn>(integer(args[1]));
    Py_XDECREF(g_check);
    g_check = Py_NewRef(args[2]);
    return Py_NewRef(Py_None);
  });
}

PyMethodDef methods[] = {
    {"rotate_qk", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(rotate_qk)), METH_FASTCALL, nullptr},
    {"norm_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(norm_rows)), METH_FASTCALL, nullptr},
    {"apart", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_apart)), METH_FASTCALL, nullptr},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native(void) {
  s_code = PyUnicode_InternFromString("code");
  s_eps = PyUnicode_InternFromString("eps");
  s_weight = PyUnicode_InternFromString("weight");
  s_bias = PyUnicode_InternFromString("bias");
  s_spec = PyUnicode_InternFromString("_spec");
  return PyModule_Create(&module);
}
