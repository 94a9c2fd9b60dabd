/*
 * torch_adamw.cpp -- torch binding of the AdamW entry points of the C ABI.
 *
 * Lists of tensors come in as Python sequences and are read in place (no list
 * of handles is built); every check of shape, type, layout and device is made
 * here, on the host, before anything is launched.  A call of any number of
 * tensors is one binding call.  Work runs on the current torch stream of the
 * tensors' device; temporaries come from torch's caching allocator.
 *
 * With hundreds of small tensors this reading is what bounds a call (1800
 * tensors in an 8-bit step of 300 parameters), so it is one pass over all lists
 * that works on the tensor implementations, and a tensor with the dispatch keys,
 * type and device of the one before it is taken without further questions.
 */
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cmath>
#include <cstdint>
#include <optional>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "cubicsplat_b200.h"

namespace py = pybind11;
using at::Tensor;

namespace {

[[noreturn]] void bad(const std::string& what) { throw py::value_error(what); }

void check(int status, const char* what) {
  if (status != CS_OK)
    throw std::runtime_error(std::string(what) + " failed (status " + std::to_string(status) + ")");
}

using Impl = c10::TensorImpl;

// A sequence of tensors, read without copies while `seq` lives.
struct TensorList {
  PyObject* fast;
  PyObject** items;
  Py_ssize_t n;
  const char* name;
  bool lazy = false;             // takes tensors whose sign is still to be applied
  PyTypeObject* kind = nullptr;  // Python type of the last tensor
  c10::DispatchKeySet keys;      // of the last tensor that passed all questions
  caffe2::TypeMeta type;
  int64_t bytes = 0;  // of an element
  TensorList(const py::handle& seq, const char* what) : name(what) {
    fast = THPVariable_Check(seq.ptr()) ? nullptr : PySequence_Fast(seq.ptr(), "");
    if (!fast) {
      PyErr_Clear();
      bad(std::string(what) + " must be a sequence of tensors");
    }
    n = PySequence_Fast_GET_SIZE(fast);
    items = PySequence_Fast_ITEMS(fast);
  }
  TensorList(const TensorList&) = delete;
  TensorList& operator=(const TensorList&) = delete;
  ~TensorList() { Py_XDECREF(fast); }
  py::object kept() const { return py::reinterpret_borrow<py::object>(fast); }
  std::string at(Py_ssize_t i) const { return std::string(name) + "[" + std::to_string(i) + "]"; }
  const Tensor& operator[](Py_ssize_t i) const {
    if (!THPVariable_Check(items[i])) bad(at(i) + " must be a tensor");
    return THPVariable_Unpack(items[i]);
  }
  // The tensor's implementation: dense, on `dev`, of one of the types that
  // `takes` accepts (it names them otherwise).
  template <class Takes>
  Impl* get(Py_ssize_t i, const at::Device& dev, const Takes& takes) {
    PyObject* o = items[i];
    if (__builtin_expect(Py_TYPE(o) != kind, 0)) {
      (*this)[i];
      kind = Py_TYPE(o);
    }
    Impl* x = THPVariable_Unpack(o).unsafeGetTensorImpl();
    if (__builtin_expect(x->key_set() == keys && x->dtype() == type && x->device() == dev, 1))
      return x;
    question(x, i, dev, takes(x->dtype().toScalarType()));
    return x;
  }
  __attribute__((noinline)) void question(Impl* x, Py_ssize_t i, const at::Device& dev,
                                          const char* want) {
    if (x->layout() != at::kStrided) bad(at(i) + " must be a dense tensor");
    if (!x->is_cuda()) bad(at(i) + " must be a CUDA tensor");
    if (x->device() != dev)
      bad(at(i) + " must be on " + dev.str() + ", got " + x->device().str());
    if (want)
      bad(at(i) + " must be " + want + ", got " + c10::toString(x->dtype().toScalarType()));
    if (!x->has_storage()) bad(at(i) + " must have a storage of its own");
    if (!lazy && x->is_neg()) bad(at(i) + " must not be a lazily negated view");
    keys = x->key_set();
    type = x->dtype();
    bytes = (int64_t)type.itemsize();
  }
  // The memory of a tensor that get() returned: its storage's, unless that is
  // still shared copy-on-write (it has a context other than its memory then) and
  // has to be made its own first, or there is none, which is an error.
  void* data(Impl* x) const {
    const at::DataPtr& p =
        x->unsafe_storage().unsafeGetStorageImpl()->_mutable_data_ptr_no_checks();
    if (__builtin_expect(p.get() && p.get() == p.get_context(), 1))
      return static_cast<char*>(p.get()) + x->storage_offset() * bytes;
    return x->mutable_data();
  }
};

const char* takes_float(at::ScalarType t) {
  return t == at::kFloat || t == at::kBFloat16 || t == at::kHalf
             ? nullptr
             : "float32, bfloat16 or float16";
}
const char* takes_float32(at::ScalarType t) { return t == at::kFloat ? nullptr : "Float"; }
const char* takes_byte(at::ScalarType t) { return t == at::kByte ? nullptr : "Byte"; }
const char* takes_long(at::ScalarType t) { return t == at::kLong ? nullptr : "Long"; }

void same_length(const TensorList& a, const TensorList& b) {
  if (a.n != b.n)
    bad(std::string(b.name) + " must have as many tensors as " + a.name + " (" +
        std::to_string(a.n) + "), got " + std::to_string(b.n));
}

int dtype_code(const Impl* x) {
  const at::ScalarType t = x->dtype().toScalarType();
  return t == at::kFloat ? CS_F32 : t == at::kBFloat16 ? CS_BF16 : CS_F16;
}

// The device of a list's first tensor, which has to be a CUDA tensor.
at::Device device_of(TensorList& l) {
  const Tensor& t = l[0];
  if (t.layout() != at::kStrided) bad(l.at(0) + " must be a dense tensor");
  if (!t.is_cuda()) bad(l.at(0) + " must be a CUDA tensor");
  return t.device();
}

bool same_shape(const Impl* a, const Impl* b) {
  const auto x = a->sizes(), y = b->sizes();
  if (x.size() != y.size()) return false;
  for (size_t i = 0; i < x.size(); ++i)
    if (x[i] != y[i]) return false;
  return true;
}

// Both tensors keep the same element at the same place of their storage;
// `contiguous` says whether b is contiguous.
bool same_layout(const Impl* a, const Impl* b, bool contiguous) {
  return (contiguous && a->is_contiguous()) || a->strides() == b->strides();
}

void check_like(const Impl* x, const Impl* p, bool contiguous, const TensorList& l,
                Py_ssize_t i) {
  if (!same_shape(x, p) || !same_layout(x, p, contiguous))
    bad(l.at(i) + " must have its parameter's shape and strides");
}

int64_t scale_count(int64_t numel) { return (numel + CS_ADAMW8_BLOCK - 1) / CS_ADAMW8_BLOCK; }

void check_scales(const Impl* x, int64_t count, const TensorList& l, Py_ssize_t i) {
  if (!x->is_contiguous() || x->numel() != count)
    bad(l.at(i) + " must be " + std::to_string(count) +
        " contiguous uint8 scales (one per started block of " + std::to_string(CS_ADAMW8_BLOCK) +
        " elements)");
}

// Written buffers of a call, to refuse one that is given twice.
struct Written {
  std::vector<const void*> slots;
  size_t mask;
  explicit Written(size_t n) {
    size_t cap = 16;
    while (cap < 2 * n) cap *= 2;
    slots.assign(cap, nullptr);
    mask = cap - 1;
  }
  void add(const void* p, const TensorList& l, Py_ssize_t i) {
    if (!p) return;
    size_t h = (reinterpret_cast<uintptr_t>(p) >> 2) * size_t(0x9E3779B97F4A7C15ull);
    h ^= h >> 32;
    for (h &= mask; slots[h]; h = (h + 1) & mask)
      if (slots[h] == p) bad(l.at(i) + " is given twice: no written tensor may be shared");
    slots[h] = p;
  }
};

// The memory of one value of type T on `dev` (`want` says what it has to be).
template <class T>
T* device_value(const Tensor& t, const at::Device& dev, const std::string& name,
                const char* want) {
  if (t.layout() != at::kStrided || !t.is_cuda() || t.device() != dev ||
      t.scalar_type() != c10::CppTypeToScalarType<T>::value || t.numel() != 1)
    bad(name + " must be " + want + " on " + dev.str());
  if (t.is_neg()) bad(name + " must not be a lazily negated view");
  return t.data_ptr<T>();
}

// A float32 device scalar, or NULL for None.
const float* device_scalar(const std::optional<Tensor>& t, const at::Device& dev,
                           const char* name) {
  return t ? device_value<float>(*t, dev, name, "one float32 value") : nullptr;
}

void* stream_of(const at::Device& dev) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

bool is_scalar_tensor(const py::handle& h) { return THPVariable_Check(h.ptr()); }

struct Groups {
  std::vector<cs_adamw_group> g;
  std::vector<int64_t> ends;     // one past each group's last tensor
  std::vector<int64_t*> counters;  // device step counters, or empty
  std::vector<Impl*> changed;      // their tensors
};

// groups: (tensors, lr, beta1, beta2, eps, weight_decay, step) each; lr a float
// or a device scalar, step an int or an int64 device counter (all or none).
Groups read_groups(const py::list& list, Py_ssize_t tensors, const at::Device& dev) {
  Groups r;
  const size_t n = list.size();
  if (n < 1 || n > CS_ADAMW_MAX_GROUPS)
    bad("a step takes 1 to " + std::to_string(CS_ADAMW_MAX_GROUPS) + " groups");
  int64_t end = 0;
  for (size_t i = 0; i < n; ++i) {
    const py::tuple t = list[i];
    cs_adamw_group g{};
    end += t[0].cast<int64_t>();
    r.ends.push_back(end);
    const py::handle lr = t[1];
    if (is_scalar_tensor(lr))
      g.lr_device = device_scalar(THPVariable_Unpack(lr.ptr()), dev, "lr");
    else
      g.lr = lr.cast<double>();
    g.beta1 = t[2].cast<double>();
    g.beta2 = t[3].cast<double>();
    g.eps = t[4].cast<double>();
    g.weight_decay = t[5].cast<double>();
    if (!(g.lr >= 0.0)) bad("Invalid learning rate: " + std::to_string(g.lr));
    if (!(g.eps >= 0.0)) bad("Invalid epsilon value: " + std::to_string(g.eps));
    if (!(g.beta1 >= 0.0 && g.beta1 < 1.0))
      bad("Invalid beta parameter at index 0: " + std::to_string(g.beta1));
    if (!(g.beta2 >= 0.0 && g.beta2 < 1.0))
      bad("Invalid beta parameter at index 1: " + std::to_string(g.beta2));
    if (!(g.weight_decay >= 0.0))
      bad("Invalid weight_decay value: " + std::to_string(g.weight_decay));
    const py::handle step = t[6];
    if (is_scalar_tensor(step)) {
      const Tensor& s = THPVariable_Unpack(step.ptr());
      r.counters.push_back(device_value<int64_t>(s, dev, "step", "an int or one int64 value"));
      r.changed.push_back(s.unsafeGetTensorImpl());
    } else {
      g.step = step.cast<int64_t>();
      if (g.step < 1) bad("step must be >= 1, got " + std::to_string(g.step));
    }
    r.g.push_back(g);
  }
  if (!r.counters.empty() && r.counters.size() != n)
    bad("either every group counts its steps on the device or none does");
  for (size_t i = 0; i < r.counters.size(); ++i)
    for (size_t j = 0; j < i; ++j)
      if (r.counters[i] == r.counters[j]) bad("groups must not share a device step counter");
  if (end != tensors) bad("the groups must hold every tensor of the call");
  return r;
}

// Device coefficients of counted groups: the tensor keeps them alive until the
// step is enqueued (the allocator then reuses the memory in stream order).
std::optional<Tensor> advance(const Groups& r, uint32_t seed, const at::Device& dev) {
  if (r.counters.empty()) return std::nullopt;
  Tensor coef = at::empty({4 * (int64_t)r.g.size()}, at::TensorOptions().dtype(at::kFloat).device(dev));
  check(cs_adamw_advance(r.counters.data(), r.g.data(), (int32_t)r.g.size(), seed,
                         static_cast<float*>(coef.data_ptr()), stream_of(dev)),
        "cs_adamw_advance");
  return coef;
}

// Device step counters of every tensor of a call, where the call has them.
struct Counters {
  std::optional<TensorList> list;
  std::vector<int64_t*> at;
  Counters(const py::handle& seq, const TensorList& params, const Groups& r) {
    if (seq.is_none()) return;
    if (!r.counters.empty()) bad("steps are counted by group or by tensor, not by both");
    list.emplace(seq, "steps");
    same_length(params, *list);
    at.reserve(params.n);
  }
  size_t size() const { return list ? (size_t)list->n : 0; }
  void read(Py_ssize_t i, const at::Device& dev, std::vector<Impl*>& changed, Written& written) {
    if (!list) return;
    Impl* x = list->get(i, dev, takes_long);
    if (x->numel() != 1) bad(list->at(i) + " must be one value");
    changed.push_back(x);
    at.push_back(static_cast<int64_t*>(list->data(x)));
    written.add(at.back(), *list, i);
  }
};

// Tensors that a call has written: their versions go up once it is enqueued, so
// that a graph which saved them notices.
void bump_versions(const std::vector<Impl*>& changed) {
  for (Impl* x : changed)
    if (!x->is_inference()) x->bump_version();
}

// A parameter and its gradient; a gradient of another layout is copied.
// Returns whether the parameter is contiguous.
bool read_param(TensorList& params, TensorList& grads, Py_ssize_t i, const at::Device& dev,
                cs_adamw_tensor& s, Impl*& p, std::vector<Tensor>& copies,
                std::vector<Impl*>& changed, Written& written) {
  p = params.get(i, dev, takes_float);
  const bool contiguous = p->is_contiguous();
  if (!contiguous && !p->is_non_overlapping_and_dense())
    bad(params.at(i) + " must be non-overlapping and dense");
  Impl* g = grads.get(i, dev, takes_float);
  if (g->dtype() != p->dtype() || !same_shape(g, p))
    bad(grads.at(i) + " must have its parameter's shape and type");
  s.dtype = dtype_code(p);
  s.numel = p->numel();
  if (!s.numel) return contiguous;
  changed.push_back(p);
  s.param = params.data(p);
  if (same_layout(g, p, contiguous) && !g->is_neg()) {
    s.grad = grads.data(g);
  } else {
    at::NoGradGuard no_grad;
    copies.push_back(at::empty_like(params[i]).copy_(grads[i]));
    s.grad = copies.back().data_ptr();
  }
  written.add(s.param, params, i);
  return contiguous;
}

void set_groups(const Groups& r, std::vector<cs_adamw_tensor>& t) {
  size_t g = 0;
  for (size_t i = 0; i < t.size(); ++i) {
    while ((int64_t)i >= r.ends[g]) ++g;
    t[i].group = (int32_t)g;
  }
}

// A step that has been read and checked and is not yet enqueued.  It keeps the
// lists it was read from: an iterator's tensors have no other owner.
struct Step {
  std::array<py::object, 7> lists;
  at::Device dev = at::kCPU;
  int bits;
  Groups r;
  std::vector<cs_adamw_tensor> t;
  std::vector<Tensor> copies;
  std::vector<int64_t*> counters;  // one of each tensor, or empty
  std::vector<Impl*> changed;
  const float* scale;
  uint32_t seed = 0;
  int32_t first_place = 0;

  void enqueue() const {
    if (t.empty()) return;
    c10::cuda::CUDAGuard guard(dev);
    const auto count = (int32_t)t.size(), groups = (int32_t)r.g.size();
    if (!counters.empty()) {
      const Tensor work =
          at::empty({4 * (int64_t)count}, at::TensorOptions().dtype(at::kFloat).device(dev));
      auto* w = static_cast<float*>(work.data_ptr());
      if (bits == 8)
        check(cs_adamw8_step_counted(t.data(), count, r.g.data(), groups, counters.data(), w, seed,
                                     first_place, scale, stream_of(dev)),
              "cs_adamw8_step_counted");
      else
        check(cs_adamw_step_counted(t.data(), count, r.g.data(), groups, counters.data(), w, scale,
                                    stream_of(dev)),
              "cs_adamw_step_counted");
    } else {
      const std::optional<Tensor> coef = advance(r, seed, dev);
      const float* c = coef ? static_cast<const float*>(coef->data_ptr()) : nullptr;
      if (bits == 8)
        check(cs_adamw8_step_at(t.data(), count, r.g.data(), groups, c, seed, first_place, scale,
                                stream_of(dev)),
              "cs_adamw8_step_at");
      else
        check(cs_adamw_step(t.data(), count, r.g.data(), groups, c, scale, stream_of(dev)),
              "cs_adamw_step");
    }
    bump_versions(changed);
  }
};

Step read_step(const py::handle& params_, const py::handle& grads_, const py::handle& exp_avgs_,
               const py::handle& exp_avg_sqs_, const py::list& groups,
               const std::optional<Tensor>& grad_scale, const py::handle& steps) {
  Step step;
  step.bits = 32;
  TensorList params(params_, "params"), grads(grads_, "grads"), m(exp_avgs_, "exp_avgs"),
      v(exp_avg_sqs_, "exp_avg_sqs");
  for (const TensorList* l : {&grads, &m, &v}) same_length(params, *l);
  grads.lazy = true;
  if (params.n == 0) return step;
  step.r = read_groups(groups, params.n, params[0].device());
  const at::Device dev = step.dev = device_of(params);
  step.scale = device_scalar(grad_scale, dev, "grad_scale");
  step.t.resize(params.n, cs_adamw_tensor{});
  step.changed = step.r.changed;
  Counters counters(steps, params, step.r);
  step.changed.reserve(step.changed.size() + counters.size() + 3 * params.n);
  Written written(counters.size() + 3 * params.n);
  for (Py_ssize_t i = 0; i < params.n; ++i) {
    cs_adamw_tensor& s = step.t[i];
    Impl* p;
    const bool contiguous =
        read_param(params, grads, i, dev, s, p, step.copies, step.changed, written);
    Impl* mi = m.get(i, dev, takes_float32);
    Impl* vi = v.get(i, dev, takes_float32);
    check_like(mi, p, contiguous, m, i);
    check_like(vi, p, contiguous, v, i);
    counters.read(i, dev, step.changed, written);
    if (!s.numel) continue;
    step.changed.push_back(mi);
    step.changed.push_back(vi);
    written.add(s.exp_avg = m.data(mi), m, i);
    written.add(s.exp_avg_sq = v.data(vi), v, i);
  }
  set_groups(step.r, step.t);
  step.counters = std::move(counters.at);
  py::object* kept = step.lists.data();
  for (const TensorList* l : {&params, &grads, &m, &v}) *kept++ = l->kept();
  if (counters.list) *kept = counters.list->kept();
  return step;
}

Step read_step8(const py::handle& params_, const py::handle& grads_, const py::handle& exp_avgs_,
                const py::handle& m_scales_, const py::handle& exp_avg_sqs_,
                const py::handle& v_scales_, const py::list& groups, uint32_t seed,
                const std::optional<Tensor>& grad_scale, int32_t first_place,
                const py::handle& steps) {
  Step step;
  step.bits = 8;
  step.seed = seed;
  step.first_place = first_place;
  TensorList params(params_, "params"), grads(grads_, "grads"), m(exp_avgs_, "exp_avgs"),
      ms(m_scales_, "exp_avg_scales"), v(exp_avg_sqs_, "exp_avg_sqs"),
      vs(v_scales_, "exp_avg_sq_scales");
  for (const TensorList* l : {&grads, &m, &ms, &v, &vs}) same_length(params, *l);
  grads.lazy = true;
  if (params.n == 0) return step;
  step.r = read_groups(groups, params.n, params[0].device());
  const at::Device dev = step.dev = device_of(params);
  step.scale = device_scalar(grad_scale, dev, "grad_scale");
  step.t.resize(params.n, cs_adamw_tensor{});
  step.changed = step.r.changed;
  Counters counters(steps, params, step.r);
  step.changed.reserve(step.changed.size() + counters.size() + 5 * params.n);
  Written written(counters.size() + 5 * params.n);
  for (Py_ssize_t i = 0; i < params.n; ++i) {
    cs_adamw_tensor& s = step.t[i];
    Impl* p;
    const bool contiguous =
        read_param(params, grads, i, dev, s, p, step.copies, step.changed, written);
    Impl* mi = m.get(i, dev, takes_byte);
    Impl* vi = v.get(i, dev, takes_byte);
    check_like(mi, p, contiguous, m, i);
    check_like(vi, p, contiguous, v, i);
    Impl* msi = ms.get(i, dev, takes_byte);
    Impl* vsi = vs.get(i, dev, takes_byte);
    check_scales(msi, scale_count(s.numel), ms, i);
    check_scales(vsi, scale_count(s.numel), vs, i);
    counters.read(i, dev, step.changed, written);
    if (!s.numel) continue;
    for (Impl* x : {mi, vi, msi, vsi}) step.changed.push_back(x);
    written.add(s.exp_avg = m.data(mi), m, i);
    written.add(s.exp_avg_sq = v.data(vi), v, i);
    written.add(s.exp_avg_scales = static_cast<uint8_t*>(ms.data(msi)), ms, i);
    written.add(s.exp_avg_sq_scales = static_cast<uint8_t*>(vs.data(vsi)), vs, i);
  }
  set_groups(step.r, step.t);
  step.counters = std::move(counters.at);
  py::object* kept = step.lists.data();
  for (const TensorList* l : {&params, &grads, &m, &v, &ms, &vs}) *kept++ = l->kept();
  if (counters.list) *kept = counters.list->kept();
  return step;
}

void adamw_step(const py::object& params, const py::object& grads, const py::object& exp_avgs,
                const py::object& exp_avg_sqs, const py::list& groups,
                const std::optional<Tensor>& grad_scale) {
  read_step(params, grads, exp_avgs, exp_avg_sqs, groups, grad_scale, py::none()).enqueue();
}

void adamw8_step(const py::object& params, const py::object& grads, const py::object& exp_avgs,
                 const py::object& m_scales, const py::object& exp_avg_sqs,
                 const py::object& v_scales, const py::list& groups, uint32_t seed,
                 const std::optional<Tensor>& grad_scale) {
  read_step8(params, grads, exp_avgs, m_scales, exp_avg_sqs, v_scales, groups, seed, grad_scale, 0,
             py::none())
      .enqueue();
}

// The calls of one optimiser step: (params, grads, exp_avgs, exp_avg_sqs, groups,
// steps) each, with 8-bit moments (..., groups, steps, exp_avg_scales,
// exp_avg_sq_scales, seed, first place); steps is None or the tensors' device
// counters.  All of them are read and checked before the first is enqueued.
void adamw_steps(const py::list& calls, const std::optional<Tensor>& grad_scale) {
  std::vector<Step> all;
  all.reserve(calls.size());
  for (const py::handle& call : calls) {
    const py::tuple c = py::reinterpret_borrow<py::tuple>(call);
    if (c.size() == 6)
      all.push_back(read_step(c[0], c[1], c[2], c[3], c[4], grad_scale, c[5]));
    else
      all.push_back(read_step8(c[0], c[1], c[2], c[6], c[3], c[7], c[4], c[8].cast<uint32_t>(),
                               grad_scale, c[9].cast<int32_t>(), c[5]));
  }
  for (const Step& s : all) s.enqueue();
}

void adamw8_moments(const py::object& exp_avgs_, const py::object& m_scales_,
                    const py::object& exp_avg_sqs_, const py::object& v_scales_,
                    const py::object& out_m_, const py::object& out_v_) {
  TensorList m(exp_avgs_, "exp_avgs"), ms(m_scales_, "exp_avg_scales"),
      v(exp_avg_sqs_, "exp_avg_sqs"), vs(v_scales_, "exp_avg_sq_scales"), om(out_m_, "out[0]"),
      ov(out_v_, "out[1]");
  for (const TensorList* l : {&ms, &v, &vs, &om, &ov}) same_length(m, *l);
  if (m.n == 0) return;
  const at::Device dev = device_of(m);
  c10::cuda::CUDAGuard guard(dev);
  std::vector<cs_adamw_tensor> t(m.n, cs_adamw_tensor{});
  std::vector<Impl*> changed;
  changed.reserve(2 * m.n);
  Written written(2 * m.n);
  for (Py_ssize_t i = 0; i < m.n; ++i) {
    cs_adamw_tensor& s = t[i];
    Impl* c = m.get(i, dev, takes_byte);
    const bool contiguous = c->is_contiguous();
    if (!contiguous && !c->is_non_overlapping_and_dense())
      bad(m.at(i) + " must be non-overlapping and dense");
    Impl* vi = v.get(i, dev, takes_byte);
    Impl* omi = om.get(i, dev, takes_float32);
    Impl* ovi = ov.get(i, dev, takes_float32);
    check_like(vi, c, contiguous, v, i);
    check_like(omi, c, contiguous, om, i);
    check_like(ovi, c, contiguous, ov, i);
    Impl* msi = ms.get(i, dev, takes_byte);
    Impl* vsi = vs.get(i, dev, takes_byte);
    s.numel = c->numel();
    s.dtype = CS_F32;
    check_scales(msi, scale_count(s.numel), ms, i);
    check_scales(vsi, scale_count(s.numel), vs, i);
    if (!s.numel) continue;
    s.exp_avg = m.data(c);
    s.exp_avg_sq = v.data(vi);
    s.exp_avg_scales = static_cast<uint8_t*>(ms.data(msi));
    s.exp_avg_sq_scales = static_cast<uint8_t*>(vs.data(vsi));
    changed.push_back(omi);
    changed.push_back(ovi);
    written.add(s.param = om.data(omi), om, i);
    written.add(s.grad = ov.data(ovi), ov, i);
  }
  check(cs_adamw8_moments(t.data(), (int32_t)t.size(), stream_of(dev)), "cs_adamw8_moments");
  bump_versions(changed);
}

std::tuple<Tensor, Tensor> grad_norm(const py::object& grads_, double max_norm, double eps) {
  TensorList grads(grads_, "grads");
  if (grads.n == 0) bad("grads must not be empty");
  grads.lazy = true;  // the norm of -x is that of x
  if (!(max_norm >= 0.0)) bad("Invalid max_norm: " + std::to_string(max_norm));
  if (!(eps >= 0.0)) bad("Invalid epsilon value: " + std::to_string(eps));
  const at::Device dev = device_of(grads);
  c10::cuda::CUDAGuard guard(dev);
  at::NoGradGuard no_grad;
  std::vector<cs_grad_tensor> t(grads.n, cs_grad_tensor{});
  std::vector<Tensor> copies;
  for (Py_ssize_t i = 0; i < grads.n; ++i) {
    Impl* g = grads.get(i, dev, takes_float);
    t[i].dtype = dtype_code(g);
    t[i].numel = g->numel();
    if (!t[i].numel) continue;
    if (g->is_contiguous() || g->is_non_overlapping_and_dense()) {
      t[i].data = grads.data(g);
    } else {
      copies.push_back(grads[i].contiguous());
      t[i].data = copies.back().data_ptr();
    }
  }
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
  Tensor norm = at::empty({}, f32), scale = at::empty({}, f32);
  const size_t bytes = cs_grad_norm_workspace_size(t.data(), (int32_t)t.size());
  Tensor ws;
  if (bytes) ws = at::empty({(int64_t)bytes}, f32.dtype(at::kByte));
  check(cs_grad_norm(t.data(), (int32_t)t.size(), max_norm, eps,
                     static_cast<float*>(norm.data_ptr()), static_cast<float*>(scale.data_ptr()),
                     bytes ? ws.data_ptr() : nullptr, stream_of(dev)),
        "cs_grad_norm");
  return {norm, scale};
}

}  // namespace

void bind_adamw(py::module_& m) {
  m.attr("ADAMW8_BLOCK") = CS_ADAMW8_BLOCK;
  m.attr("ADAMW_MAX_GROUPS") = CS_ADAMW_MAX_GROUPS;
  m.def("adamw_step", &adamw_step);
  m.def("adamw8_step", &adamw8_step);
  m.def("adamw_steps", &adamw_steps);
  m.def("adamw8_moments", &adamw8_moments);
  m.def("grad_norm", &grad_norm);
}
