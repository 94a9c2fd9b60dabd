/*
 * torch_adamw.cpp -- torch binding of the AdamW entry points of the C ABI.
 *
 * Lists of tensors come in as Python sequences and are read in place (no list
 * of handles is built); every check of shape, type, layout and device is made
 * here, on the host, before anything is launched.  A call of any number of
 * tensors is one binding call.  Work runs on the current torch stream of the
 * tensors' device; temporaries come from torch's caching allocator.
 */
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

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

// A sequence of tensors, read without copies while `seq` lives.
struct TensorList {
  PyObject* fast;
  Py_ssize_t n;
  const char* name;
  TensorList(const py::handle& seq, const char* what) : name(what) {
    fast = THPVariable_Check(seq.ptr()) ? nullptr : PySequence_Fast(seq.ptr(), "");
    if (!fast) {
      PyErr_Clear();
      bad(std::string(what) + " must be a sequence of tensors");
    }
    n = PySequence_Fast_GET_SIZE(fast);
  }
  TensorList(const TensorList&) = delete;
  TensorList& operator=(const TensorList&) = delete;
  ~TensorList() { Py_XDECREF(fast); }
  std::string at(Py_ssize_t i) const { return std::string(name) + "[" + std::to_string(i) + "]"; }
  const Tensor& operator[](Py_ssize_t i) const {
    PyObject* o = PySequence_Fast_GET_ITEM(fast, i);
    if (!THPVariable_Check(o)) bad(at(i) + " must be a tensor");
    return THPVariable_Unpack(o);
  }
};

void same_length(const TensorList& a, const TensorList& b) {
  if (a.n != b.n)
    bad(std::string(b.name) + " must have as many tensors as " + a.name + " (" +
        std::to_string(a.n) + "), got " + std::to_string(b.n));
}

int dtype_code(const Tensor& t, const TensorList& l, Py_ssize_t i) {
  switch (t.scalar_type()) {
    case at::kFloat: return CS_F32;
    case at::kBFloat16: return CS_BF16;
    case at::kHalf: return CS_F16;
    default: bad(l.at(i) + " must be float32, bfloat16 or float16");
  }
}

void on_device(const Tensor& t, const at::Device& dev, const TensorList& l, Py_ssize_t i) {
  if (t.layout() != at::kStrided) bad(l.at(i) + " must be a dense tensor");
  if (!t.is_cuda()) bad(l.at(i) + " must be a CUDA tensor");
  if (t.device() != dev) bad(l.at(i) + " must be on " + dev.str() + ", got " + t.device().str());
}

// Both tensors keep the same element at the same place of their storage.
bool same_layout(const Tensor& a, const Tensor& b) {
  return a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous());
}

void like_param(const Tensor& t, const Tensor& p, at::ScalarType type, const TensorList& l,
                Py_ssize_t i) {
  on_device(t, p.device(), l, i);
  if (t.scalar_type() != type)
    bad(l.at(i) + " must be " + std::string(c10::toString(type)) + ", got " +
        c10::toString(t.scalar_type()));
  if (t.sizes() != p.sizes() || !same_layout(t, p))
    bad(l.at(i) + " must have its parameter's shape and strides");
}

int64_t scale_count(int64_t numel) { return (numel + CS_ADAMW8_BLOCK - 1) / CS_ADAMW8_BLOCK; }

void check_scales(const Tensor& t, int64_t numel, const at::Device& dev, const TensorList& l,
                  Py_ssize_t i) {
  on_device(t, dev, l, i);
  if (t.scalar_type() != at::kByte || !t.is_contiguous() || t.numel() != scale_count(numel))
    bad(l.at(i) + " must be " + std::to_string(scale_count(numel)) +
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

// A 0-d (or one-element) float32 device scalar, or NULL for None.
const float* device_scalar(const std::optional<Tensor>& t, const at::Device& dev,
                           const char* name) {
  if (!t) return nullptr;
  if (!t->is_cuda() || t->device() != dev || t->scalar_type() != at::kFloat || t->numel() != 1)
    bad(std::string(name) + " must be one float32 value on " + dev.str());
  return static_cast<const float*>(t->data_ptr());
}

void* stream_of(const at::Device& dev) {
  return static_cast<void*>(c10::cuda::getCurrentCUDAStream(dev.index()).stream());
}

bool is_scalar_tensor(const py::handle& h) { return THPVariable_Check(h.ptr()); }

struct Groups {
  std::vector<cs_adamw_group> g;
  std::vector<int64_t> ends;     // one past each group's last tensor
  std::vector<int64_t*> counters;  // device step counters, or empty
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
      if (!s.is_cuda() || s.device() != dev || s.scalar_type() != at::kLong || s.numel() != 1)
        bad("step must be an int or one int64 value on " + dev.str());
      r.counters.push_back(s.data_ptr<int64_t>());
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

void written_param(const Tensor& p) {
  if (!p.is_inference()) p.unsafeGetTensorImpl()->bump_version();
}

// Parameters and gradients of a call; a gradient of another layout is copied.
void read_params(const TensorList& params, const TensorList& grads,
                 std::vector<cs_adamw_tensor>& out, std::vector<Tensor>& copies,
                 const at::Device& dev, Written& written) {
  for (Py_ssize_t i = 0; i < params.n; ++i) {
    const Tensor& p = params[i];
    const Tensor& g = grads[i];
    on_device(p, dev, params, i);
    cs_adamw_tensor& s = out[i];
    s.dtype = dtype_code(p, params, i);
    if (!p.is_non_overlapping_and_dense())
      bad(params.at(i) + " must be non-overlapping and dense");
    on_device(g, dev, grads, i);
    if (g.scalar_type() != p.scalar_type() || g.sizes() != p.sizes())
      bad(grads.at(i) + " must have its parameter's shape and type");
    s.numel = p.numel();
    s.param = s.numel ? p.data_ptr() : nullptr;
    if (same_layout(g, p) && !g.is_neg()) {
      s.grad = s.numel ? g.data_ptr() : nullptr;
    } else {
      copies.push_back(at::empty_like(p).copy_(g));
      s.grad = s.numel ? copies.back().data_ptr() : nullptr;
    }
    written.add(s.param, params, i);
  }
}

void set_groups(const Groups& r, std::vector<cs_adamw_tensor>& t) {
  size_t g = 0;
  for (size_t i = 0; i < t.size(); ++i) {
    while ((int64_t)i >= r.ends[g]) ++g;
    t[i].group = (int32_t)g;
  }
}

void adamw_step(const py::object& params_, const py::object& grads_, const py::object& exp_avgs_,
                const py::object& exp_avg_sqs_, const py::list& groups,
                const std::optional<Tensor>& grad_scale) {
  const TensorList params(params_, "params"), grads(grads_, "grads"), m(exp_avgs_, "exp_avgs"),
      v(exp_avg_sqs_, "exp_avg_sqs");
  same_length(params, grads);
  same_length(params, m);
  same_length(params, v);
  if (params.n == 0) return;
  const at::Device dev = params[0].device();
  const Groups r = read_groups(groups, params.n, dev);
  on_device(params[0], dev, params, 0);
  c10::cuda::CUDAGuard guard(dev);
  at::NoGradGuard no_grad;
  std::vector<cs_adamw_tensor> t(params.n, cs_adamw_tensor{});
  std::vector<Tensor> copies;
  Written written(3 * params.n);
  const float* scale = device_scalar(grad_scale, dev, "grad_scale");
  read_params(params, grads, t, copies, dev, written);
  for (Py_ssize_t i = 0; i < params.n; ++i) {
    like_param(m[i], params[i], at::kFloat, m, i);
    like_param(v[i], params[i], at::kFloat, v, i);
    if (!t[i].numel) continue;
    t[i].exp_avg = m[i].data_ptr();
    t[i].exp_avg_sq = v[i].data_ptr();
    written.add(t[i].exp_avg, m, i);
    written.add(t[i].exp_avg_sq, v, i);
  }
  set_groups(r, t);
  const std::optional<Tensor> coef = advance(r, 0, dev);
  check(cs_adamw_step(t.data(), (int32_t)t.size(), r.g.data(), (int32_t)r.g.size(),
                      coef ? static_cast<const float*>(coef->data_ptr()) : nullptr, scale,
                      stream_of(dev)),
        "cs_adamw_step");
  for (Py_ssize_t i = 0; i < params.n; ++i) written_param(params[i]);
}

void adamw8_step(const py::object& params_, const py::object& grads_, const py::object& exp_avgs_,
                 const py::object& m_scales_, const py::object& exp_avg_sqs_,
                 const py::object& v_scales_, const py::list& groups, uint32_t seed,
                 const std::optional<Tensor>& grad_scale) {
  const TensorList params(params_, "params"), grads(grads_, "grads"), m(exp_avgs_, "exp_avgs"),
      ms(m_scales_, "exp_avg_scales"), v(exp_avg_sqs_, "exp_avg_sqs"),
      vs(v_scales_, "exp_avg_sq_scales");
  for (const TensorList* l : {&grads, &m, &ms, &v, &vs}) same_length(params, *l);
  if (params.n == 0) return;
  const at::Device dev = params[0].device();
  const Groups r = read_groups(groups, params.n, dev);
  on_device(params[0], dev, params, 0);
  c10::cuda::CUDAGuard guard(dev);
  at::NoGradGuard no_grad;
  std::vector<cs_adamw_tensor> t(params.n, cs_adamw_tensor{});
  std::vector<Tensor> copies;
  Written written(5 * params.n);
  const float* scale = device_scalar(grad_scale, dev, "grad_scale");
  read_params(params, grads, t, copies, dev, written);
  for (Py_ssize_t i = 0; i < params.n; ++i) {
    like_param(m[i], params[i], at::kByte, m, i);
    like_param(v[i], params[i], at::kByte, v, i);
    check_scales(ms[i], t[i].numel, dev, ms, i);
    check_scales(vs[i], t[i].numel, dev, vs, i);
    if (!t[i].numel) continue;
    t[i].exp_avg = m[i].data_ptr();
    t[i].exp_avg_sq = v[i].data_ptr();
    t[i].exp_avg_scales = static_cast<uint8_t*>(ms[i].data_ptr());
    t[i].exp_avg_sq_scales = static_cast<uint8_t*>(vs[i].data_ptr());
    written.add(t[i].exp_avg, m, i);
    written.add(t[i].exp_avg_sq, v, i);
    written.add(t[i].exp_avg_scales, ms, i);
    written.add(t[i].exp_avg_sq_scales, vs, i);
  }
  set_groups(r, t);
  const std::optional<Tensor> coef = advance(r, seed, dev);
  check(cs_adamw8_step(t.data(), (int32_t)t.size(), r.g.data(), (int32_t)r.g.size(),
                       coef ? static_cast<const float*>(coef->data_ptr()) : nullptr, seed, scale,
                       stream_of(dev)),
        "cs_adamw8_step");
  for (Py_ssize_t i = 0; i < params.n; ++i) written_param(params[i]);
}

void adamw8_moments(const py::object& exp_avgs_, const py::object& m_scales_,
                    const py::object& exp_avg_sqs_, const py::object& v_scales_,
                    const py::object& out_m_, const py::object& out_v_) {
  const TensorList m(exp_avgs_, "exp_avgs"), ms(m_scales_, "exp_avg_scales"),
      v(exp_avg_sqs_, "exp_avg_sqs"), vs(v_scales_, "exp_avg_sq_scales"), om(out_m_, "out[0]"),
      ov(out_v_, "out[1]");
  for (const TensorList* l : {&ms, &v, &vs, &om, &ov}) same_length(m, *l);
  if (m.n == 0) return;
  const at::Device dev = m[0].device();
  on_device(m[0], dev, m, 0);
  c10::cuda::CUDAGuard guard(dev);
  std::vector<cs_adamw_tensor> t(m.n, cs_adamw_tensor{});
  Written written(2 * m.n);
  for (Py_ssize_t i = 0; i < m.n; ++i) {
    const Tensor& c = m[i];
    on_device(c, dev, m, i);
    if (c.scalar_type() != at::kByte || !c.is_non_overlapping_and_dense())
      bad(m.at(i) + " must be non-overlapping, dense uint8 codes");
    like_param(v[i], c, at::kByte, v, i);
    like_param(om[i], c, at::kFloat, om, i);
    like_param(ov[i], c, at::kFloat, ov, i);
    check_scales(ms[i], c.numel(), dev, ms, i);
    check_scales(vs[i], c.numel(), dev, vs, i);
    t[i].numel = c.numel();
    t[i].dtype = CS_F32;
    if (!t[i].numel) continue;
    t[i].param = om[i].data_ptr();
    t[i].grad = ov[i].data_ptr();
    t[i].exp_avg = c.data_ptr();
    t[i].exp_avg_sq = v[i].data_ptr();
    t[i].exp_avg_scales = static_cast<uint8_t*>(ms[i].data_ptr());
    t[i].exp_avg_sq_scales = static_cast<uint8_t*>(vs[i].data_ptr());
    written.add(t[i].param, om, i);
    written.add(t[i].grad, ov, i);
  }
  check(cs_adamw8_moments(t.data(), (int32_t)t.size(), stream_of(dev)), "cs_adamw8_moments");
  for (Py_ssize_t i = 0; i < m.n; ++i) {
    written_param(om[i]);
    written_param(ov[i]);
  }
}

std::tuple<Tensor, Tensor> grad_norm(const py::object& grads_, double max_norm, double eps) {
  const TensorList grads(grads_, "grads");
  if (grads.n == 0) bad("grads must not be empty");
  if (!(max_norm >= 0.0)) bad("Invalid max_norm: " + std::to_string(max_norm));
  if (!(eps >= 0.0)) bad("Invalid epsilon value: " + std::to_string(eps));
  const at::Device dev = grads[0].device();
  on_device(grads[0], dev, grads, 0);
  c10::cuda::CUDAGuard guard(dev);
  at::NoGradGuard no_grad;
  std::vector<cs_grad_tensor> t(grads.n, cs_grad_tensor{});
  std::vector<Tensor> copies;
  for (Py_ssize_t i = 0; i < grads.n; ++i) {
    const Tensor& g = grads[i];
    on_device(g, dev, grads, i);
    t[i].dtype = dtype_code(g, grads, i);
    t[i].numel = g.numel();
    if (!t[i].numel) continue;
    if (g.is_non_overlapping_and_dense()) {
      t[i].data = g.data_ptr();
    } else {
      copies.push_back(g.contiguous());
      t[i].data = copies.back().data_ptr();
    }
  }
  const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
  Tensor norm = at::empty({}, f32), scale = at::empty({}, f32);
  Tensor ws = at::empty({(int64_t)cs_grad_norm_workspace_size((int32_t)grads.n)},
                        f32.dtype(at::kByte));
  check(cs_grad_norm(t.data(), (int32_t)t.size(), max_norm, eps,
                     static_cast<float*>(norm.data_ptr()), static_cast<float*>(scale.data_ptr()),
                     ws.data_ptr(), stream_of(dev)),
        "cs_grad_norm");
  return {norm, scale};
}

}  // namespace

void bind_adamw(py::module_& m) {
  m.attr("ADAMW8_BLOCK") = CS_ADAMW8_BLOCK;
  m.attr("ADAMW_MAX_GROUPS") = CS_ADAMW_MAX_GROUPS;
  m.def("adamw_step", &adamw_step);
  m.def("adamw8_step", &adamw8_step);
  m.def("adamw8_moments", &adamw8_moments);
  m.def("grad_norm", &grad_norm);
}
