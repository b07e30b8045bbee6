// Host side of the operators around the convolutions: root-mean-square norm, log probabilities and the AdamW step, over the C
// ABI of libsphmap.so.  Part of the extension whose module torch_shim.cpp defines.
//
// A tensor is taken as rows (its normalised or classified dimension has stride 1 and the others are one run of equal steps:
// the last dimension of a contiguous tensor, a slice of wider rows, dimension 1 of a channels-last image) or as planes (a
// contiguous tensor, any dimension).  Others are refused.
#include <torch/extension.h>

#include <ATen/TracerMode.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include <algorithm>
#include <mutex>
#include <vector>

#include "sphmap.h"

namespace {

namespace py = pybind11;
using torch::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = c10::optional<Tensor>;

void ok(int status, const char *what) { TORCH_CHECK(status == SPH_OK, what, ": ", sph_status_string(status)); }

void *current_stream() { return (void *)at::cuda::getCurrentCUDAStream().stream(); }

int element_of(const Tensor &t, const char *name) {
  switch (t.scalar_type()) {
    case torch::kFloat: return SPH_F32;
    case torch::kBFloat16: return SPH_BF16;
    case torch::kHalf: return SPH_F16;
    default: TORCH_CHECK(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}

size_t element_bytes(int dtype) { return dtype == SPH_F32 ? 4 : 2; }

void check_device(const Tensor &t, const char *name, const Tensor &like) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor (this build has no CPU path)");
  TORCH_CHECK(t.device() == like.device(), name, " must be on the same device as the input");
}

// How a tensor lies in memory around one of its dimensions.
struct Layout {
  int64_t dim, outer, C, inner, stride;  // stride of rows (inner == 1)
  bool moved;                            // rows with values behind their dimension too: outputs are rows seen through movedim
};

Layout layout_of(const Tensor &t, int64_t dim, const char *name) {
  TORCH_CHECK(t.dim() >= 1, name, " must have at least one dimension");
  TORCH_CHECK(t.layout() == torch::kStrided, name, " must be a dense tensor");
  TORCH_CHECK(dim >= -t.dim() && dim < t.dim(), "dim must be in [", -t.dim(), ", ", t.dim() - 1, "], got ", dim);
  Layout l{dim < 0 ? dim + t.dim() : dim, 1, 0, 1, 0, false};
  l.C = t.size(l.dim);
  TORCH_CHECK(l.C > 0, name, " must have at least one value along dim");
  for (int64_t i = 0; i < t.dim(); i++)
    if (i != l.dim) (i < l.dim ? l.outer : l.inner) *= t.size(i);
  if (l.outer * l.inner == 0) {  // nothing in it: rows
    l.outer = 0, l.inner = 1, l.stride = l.C;
    l.moved = l.dim != t.dim() - 1;
    return l;
  }
  if (t.is_contiguous()) {
    if (l.inner == 1 || l.C == 1) l.outer *= l.inner, l.inner = 1;
    l.stride = l.C;
    return l;
  }
  bool rows = l.C == 1 || t.stride(l.dim) == 1;
  int64_t step = l.C, run = -1;  // the rows' stride (of one row: any), and the one that the next dimension has to have
  for (int64_t i = t.dim() - 1; i >= 0 && rows; i--) {
    if (i == l.dim || t.size(i) == 1) continue;
    if (run < 0) step = t.stride(i);
    else if (t.stride(i) != run) rows = false;
    run = t.stride(i) * t.size(i);
  }
  TORCH_CHECK(rows && step >= l.C, name, " must be contiguous, or rows of one stride with dim of stride 1");
  l.moved = l.inner > 1;
  l.outer *= l.inner, l.inner = 1, l.stride = step;
  return l;
}

std::vector<int64_t> sizes_without(const Tensor &t, int64_t dim) {
  std::vector<int64_t> s = t.sizes().vec();
  s.erase(s.begin() + dim);
  return s;
}
// A dense tensor of the layout's order with n values along its dimension.  (Made with its strides, not as a view, which autograd
// would not let be written in place.)
Tensor like_layout(const Tensor &t, const Layout &l, int64_t n, torch::ScalarType type) {
  std::vector<int64_t> s = t.sizes().vec(), strides(s.size(), 1);
  const auto options = t.options().dtype(type).memory_format(c10::nullopt).requires_grad(false);
  s[l.dim] = n;
  if (!l.moved) return torch::empty(s, options);
  int64_t step = n;
  for (int64_t i = t.dim() - 1; i >= 0; i--)
    if (i != l.dim) strides[i] = step, step *= std::max<int64_t>(s[i], 1);
  return torch::empty_strided(s, strides, options);
}
// Another tensor of the same sizes, dense in that order (copied if it is not).
Tensor in_layout(const Tensor &t, const Layout &l) {
  return l.moved ? t.movedim(l.dim, -1).contiguous().movedim(-1, l.dim) : t.contiguous();
}

// What a node saves goes through whatever hooks are set (to the host and back, say), which may bring it back with other strides;
// the kernels are given nothing that is not what was saved otherwise.
void came_back(bool same) { TORCH_CHECK(same, "a saved tensor's hooks returned another size, dtype or device than was saved"); }
Tensor came_back(const Tensor &t, int64_t numel, torch::ScalarType type, const Tensor &like) {
  came_back(t.defined() && t.numel() == numel && t.scalar_type() == type && t.layout() == torch::kStrided && t.device() == like.device());
  return t.contiguous();
}
// The input (or the sum) of a node: in the layout that it had, or dense in that order.
struct SavedInput {
  SavedVariable saved;
  at::DimVector sizes, strides;
  torch::ScalarType type;
  c10::Device device = c10::kCPU;
  void set(const Tensor &t, bool output) {
    saved = SavedVariable(t, output);
    sizes = at::DimVector(t.sizes()), strides = at::DimVector(t.strides()), type = t.scalar_type(), device = t.device();
  }
  // `l.stride` becomes that of what is returned.
  Tensor unpack(std::shared_ptr<Node> node, Layout &l) const {
    Tensor t = saved.unpack(std::move(node));
    came_back(t.defined() && t.sizes() == at::IntArrayRef(sizes) && t.scalar_type() == type && t.layout() == torch::kStrided && t.device() == device);
    if (t.strides() != at::IntArrayRef(strides)) t = in_layout(t, l), l.stride = l.C;
    return t;
  }
};

bool transformed(std::initializer_list<const Tensor *> ts) {
  if (at::tracer::impl::is_dispatch_enabled() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode))
    return true;
  for (const Tensor *t : ts)
    if (t != nullptr && t->defined() && t->_fw_grad(0).defined()) return true;
  return false;
}
bool wants_grad(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t != nullptr && t->defined() && t->requires_grad()) return true;
  return false;
}
template <class N> std::shared_ptr<N> new_node(const torch::autograd::edge_list &edges) {
  std::shared_ptr<N> n(new N(), torch::autograd::deleteNode);
  n->set_next_edges(torch::autograd::edge_list(edges));
  return n;
}
// Gradients of a backward pass that is to be differentiated itself raise when that happens.
variable_list once(variable_list r) {
  if (!at::GradMode::is_enabled()) return r;
  variable_list some;
  for (const Tensor &t : r)
    if (t.defined()) some.push_back(t.detach().requires_grad_());
  some = (*std::make_shared<torch::autograd::DelayedError>("this operator cannot be differentiated twice", (int64_t)some.size()))(std::move(some));
  size_t k = 0;
  for (Tensor &t : r)
    if (t.defined()) t = some[k++];
  return r;
}

// ---- root-mean-square norm -----------------------------------------------------------------------------------------
struct NormResult {
  Tensor out, sum, scale, rstd;
  Layout layout;
};

NormResult norm_forward(const Tensor &x, const Tensor &weight, const Tensor &residual, double eps, int64_t dim, bool quantized, bool train) {
  const int dtype = element_of(x, "input");
  NormResult r;
  r.layout = layout_of(x, dim, "input");
  const Layout &l = r.layout;
  TORCH_CHECK(eps >= 0 && std::isfinite(eps), "eps must be finite and not negative, got ", eps);
  int64_t r_stride = 0;
  if (weight.defined()) {
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == l.C, "weight must have the size (", l.C, ",) of the normalised dimension");
    TORCH_CHECK(weight.scalar_type() == torch::kFloat || weight.scalar_type() == x.scalar_type(),
                "weight must be float32 or have the input's dtype");
    TORCH_CHECK(weight.is_contiguous(), "weight must be contiguous");
  }
  if (residual.defined()) {
    TORCH_CHECK(residual.sizes() == x.sizes(), "residual must have the input's size");
    TORCH_CHECK(residual.scalar_type() == x.scalar_type(), "residual must have the input's dtype");
    const Layout q = layout_of(residual, dim, "residual");
    TORCH_CHECK(q.inner == l.inner && q.moved == l.moved, "residual must have the input's memory layout");
    r_stride = q.stride;
  }
  check_device(x, "input", x);
  if (weight.defined()) check_device(weight, "weight", x);
  if (residual.defined()) check_device(residual, "residual", x);
  c10::cuda::CUDAGuard guard(x.device());
  r.out = like_layout(x, l, l.C, quantized ? torch::kFloat8_e4m3fn : x.scalar_type());
  if (residual.defined()) r.sum = like_layout(x, l, l.C, x.scalar_type());
  const auto f32 = x.options().dtype(torch::kFloat).memory_format(c10::nullopt).requires_grad(false);
  if (quantized) r.scale = torch::empty(sizes_without(x, l.dim), f32);
  if (train) r.rstd = torch::empty({l.outer * l.inner}, f32);
  ok(sph_rms_norm_forward(x.data_ptr(), residual.defined() ? residual.data_ptr() : nullptr, weight.defined() ? weight.data_ptr() : nullptr,
                          r.sum.defined() ? r.sum.data_ptr() : nullptr, r.out.data_ptr(),
                          quantized ? r.scale.data_ptr<float>() : nullptr, train ? r.rstd.data_ptr<float>() : nullptr, l.outer, l.C,
                          l.inner, l.stride, r_stride, eps, dtype,
                          weight.defined() && weight.scalar_type() == torch::kFloat ? SPH_F32 : dtype, current_stream()),
     "sph_rms_norm_forward");
  return r;
}

struct RmsNormNode : public Node {
  SavedInput s;
  SavedVariable weight, rstd;
  bool added = false;  // s is the sum, an output
  torch::ScalarType weight_type = torch::kFloat;
  Layout layout;
  std::mutex mu;
  std::string name() const override { return "RmsNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mu);
    for (SavedVariable *v : {&s.saved, &weight, &rstd}) v->reset_data();
  }
  variable_list apply(variable_list &&g) override {
    std::lock_guard<std::mutex> lock(mu);
    variable_list r(3);
    {
      at::NoGradGuard no_grad;
      Layout l = layout;
      const Tensor x = s.unpack(added ? shared_from_this() : nullptr, l), rs = came_back(rstd.unpack(), l.outer * l.inner, torch::kFloat, x);
      Tensor w = weight.unpack();
      if (w.defined()) w = came_back(w, l.C, weight_type, x);
      const bool want_x = task_should_compute_output(0) || task_should_compute_output(1), want_w = w.defined() && task_should_compute_output(2);
      Tensor gout = g[0], gsum = added && g.size() > 1 ? g[1] : Tensor();
      if (!gout.defined()) gout = torch::zeros_like(x);
      c10::cuda::CUDAGuard guard(x.device());
      gout = in_layout(gout, l);
      if (gsum.defined()) gsum = in_layout(gsum, l);
      const int dtype = element_of(x, "input");
      Tensor gx, gw, ws;
      if (want_x) gx = like_layout(x, l, l.C, x.scalar_type());
      if (want_w) {
        gw = torch::empty_like(w);
        ws = torch::empty({(int64_t)sph_rms_norm_workspace_bytes(l.outer, l.C, l.inner)}, x.options().dtype(torch::kUInt8).memory_format(c10::nullopt));
      }
      if (want_x || want_w)
        ok(sph_rms_norm_backward(gout.data_ptr(), gsum.defined() ? gsum.data_ptr() : nullptr, x.data_ptr(), w.defined() ? w.data_ptr() : nullptr,
                                 rs.data_ptr<float>(), want_x ? gx.data_ptr() : nullptr, want_w ? gw.data_ptr() : nullptr, l.outer, l.C,
                                 l.inner, l.stride, dtype,
                                 w.defined() && w.scalar_type() == torch::kFloat ? SPH_F32 : dtype, want_w ? ws.data_ptr() : nullptr,
                                 want_w ? (size_t)ws.numel() : 0, current_stream()),
           "sph_rms_norm_backward");
      if (task_should_compute_output(0)) r[0] = gx;
      if (task_should_compute_output(1)) r[1] = gx;
      if (want_w) r[2] = gw;
    }
    return once(std::move(r));
  }
};

// (out,) or (out, sum); nothing where the native node is invisible to what looks at the call.
c10::optional<std::vector<Tensor>> rms_norm(const Tensor &x, const OptTensor &weight, const OptTensor &residual, double eps, int64_t dim,
                                            bool inside) {
  const Tensor w = weight.value_or(Tensor()), res = residual.value_or(Tensor());
  if (!inside && transformed({&x, &w, &res})) return c10::nullopt;
  const bool train = wants_grad({&x, &w, &res});
  NormResult r;
  {
    at::NoGradGuard no_grad;
    r = norm_forward(x, w, res, eps, dim, false, train);
  }
  std::vector<Tensor> out{r.out};
  if (res.defined()) out.push_back(r.sum);
  if (train) {
    auto n = new_node<RmsNormNode>(torch::autograd::collect_next_edges(x, res, w));
    n->layout = r.layout;
    n->added = res.defined();
    torch::autograd::set_history(out, n);
    if (n->added) n->layout.stride = r.layout.C;  // (the sum is dense)
    n->s.set(n->added ? out[1] : x, n->added);
    if (w.defined()) n->weight_type = w.scalar_type();
    n->weight = SavedVariable(w, false);
    n->rstd = SavedVariable(r.rstd, false);
  }
  return out;
}

// (out, scale) or (out, scale, sum), none with a gradient; nothing where what looks at the call would see the allocations alone.
c10::optional<std::vector<Tensor>> rms_norm_quantized(const Tensor &x, const OptTensor &weight, const OptTensor &residual, double eps,
                                                      int64_t dim, bool inside) {
  const Tensor w = weight.value_or(Tensor()), res = residual.value_or(Tensor());
  if (!inside && transformed({&x, &w, &res})) return c10::nullopt;
  at::NoGradGuard no_grad;
  NormResult r = norm_forward(x, w, res, eps, dim, true, false);
  std::vector<Tensor> out{r.out, r.scale};
  if (res.defined()) out.push_back(r.sum);
  return out;
}

// ---- log probabilities -----------------------------------------------------------------------------------------------
struct LogProbsNode : public Node {
  SavedInput x;
  SavedVariable target, stats, entropy, top_index;
  Layout layout;
  int64_t k = 0, ignore_index = 0;
  std::mutex mu;
  std::string name() const override { return "TokenLogProbsBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mu);
    for (SavedVariable *v : {&x.saved, &target, &stats, &entropy, &top_index}) v->reset_data();
  }
  // One value for all (the gradient of a sum or a mean) is taken as such.
  static const float *spread(Tensor &g, int64_t &stride) {
    stride = 1;
    if (!g.defined()) return nullptr;
    bool one = true;
    for (int64_t i = 0; i < g.dim(); i++) one = one && (g.size(i) == 1 || g.stride(i) == 0);
    if (one)
      stride = 0;
    else
      g = g.contiguous();
    return g.data_ptr<float>();
  }
  variable_list apply(variable_list &&g) override {
    std::lock_guard<std::mutex> lock(mu);
    variable_list r(1);
    {
      at::NoGradGuard no_grad;
      if (!task_should_compute_output(0)) return r;
      Layout l = layout;
      const int64_t n = l.outer * l.inner;
      const Tensor in = x.unpack(nullptr, l), t = came_back(target.unpack(), n, torch::kLong, in), s = came_back(stats.unpack(), 2 * n, torch::kFloat, in),
                   e = came_back(entropy.unpack(shared_from_this()), n, torch::kFloat, in);
      Tensor index = top_index.unpack();
      c10::cuda::CUDAGuard guard(in.device());
      r[0] = like_layout(in, l, l.C, in.scalar_type());
      int64_t g_stride, h_stride;
      const float *gp = spread(g[0], g_stride), *hp = spread(g[1], h_stride);
      Tensor gt = k > 0 && g.size() > 2 ? g[2] : Tensor();
      if (gt.defined()) {
        gt = in_layout(gt, l);
        came_back(index.defined() && index.sizes() == gt.sizes() && index.scalar_type() == torch::kLong && index.device() == in.device());
        index = in_layout(index, l);
      }
      ok(sph_token_log_probs_backward(in.data_ptr(), t.data_ptr<int64_t>(), s.data_ptr<float>(), e.data_ptr<float>(),
                                      gt.defined() ? index.data_ptr<int64_t>() : nullptr, gp, g_stride, hp, h_stride,
                                      gt.defined() ? gt.data_ptr<float>() : nullptr, r[0].data_ptr(), l.outer, l.C, l.inner, l.stride, k,
                                      ignore_index, element_of(in, "logits"), current_stream()),
         "sph_token_log_probs_backward");
    }
    return once(std::move(r));
  }
};

// (log_probs, entropy[, top_log_probs, top_indices])
c10::optional<std::vector<Tensor>> token_log_probs(const Tensor &x, const Tensor &target, int64_t dim, int64_t k, int64_t ignore_index,
                                                   bool inside) {
  if (!inside && transformed({&x})) return c10::nullopt;
  const int dtype = element_of(x, "logits");
  const Layout l = layout_of(x, dim, "logits");
  TORCH_CHECK(target.scalar_type() == torch::kLong, "target must be int64, got ", target.scalar_type());
  TORCH_CHECK(target.sizes() == sizes_without(x, l.dim), "target must have the logits' size without dim");
  TORCH_CHECK(target.is_contiguous(), "target must be contiguous");
  TORCH_CHECK(k >= 0 && k <= l.C, "top_k must be in [0, ", l.C, "], got ", k);
  check_device(x, "logits", x);
  check_device(target, "target", x);
  const bool train = wants_grad({&x});
  std::vector<Tensor> out;
  Tensor stats, index;
  {
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(x.device());
    const auto f32 = x.options().dtype(torch::kFloat).memory_format(c10::nullopt).requires_grad(false);
    out = {torch::empty(target.sizes(), f32), torch::empty(target.sizes(), f32)};
    if (k > 0) {
      out.push_back(like_layout(x, l, k, torch::kFloat));
      index = like_layout(x, l, k, torch::kLong);
    }
    if (train) stats = torch::empty({target.numel(), 2}, f32);
    ok(sph_token_log_probs_forward(x.data_ptr(), target.data_ptr<int64_t>(), out[0].data_ptr<float>(), out[1].data_ptr<float>(),
                                   train ? stats.data_ptr<float>() : nullptr, k > 0 ? out[2].data_ptr<float>() : nullptr,
                                   k > 0 ? index.data_ptr<int64_t>() : nullptr, l.outer, l.C, l.inner, l.stride, k, ignore_index, dtype,
                                   current_stream()),
       "sph_token_log_probs_forward");
  }
  if (train) {
    auto n = new_node<LogProbsNode>(torch::autograd::collect_next_edges(x));
    n->layout = l;
    n->k = k;
    n->ignore_index = ignore_index;
    torch::autograd::set_history(out, n);
    n->x.set(x, false);
    n->target = SavedVariable(target, false);
    n->stats = SavedVariable(stats, false);
    n->entropy = SavedVariable(out[1], true);
    n->top_index = SavedVariable(index, false);
  }
  if (k > 0) out.push_back(index);
  return out;
}

// ---- AdamW -----------------------------------------------------------------------------------------------------------
// A Python list or tuple of tensors, or None for no list; read where it is (a network's parameters make hundreds of tensors a
// step, and copying them would take longer than the step).  The caller holds the list and the interpreter's lock.
class TensorList {
 public:
  TensorList(const py::object &o, const char *name) : name_(name) {
    if (o.is_none()) return;
    seq_ = py::reinterpret_steal<py::object>(PySequence_Fast(o.ptr(), "adamw_step takes lists of tensors"));
    if (!seq_) throw py::error_already_set();
    items_ = PySequence_Fast_ITEMS(seq_.ptr());
    size_ = (size_t)PySequence_Fast_GET_SIZE(seq_.ptr());
  }
  explicit operator bool() const { return items_ != nullptr || seq_; }
  size_t size() const { return size_; }
  bool has(size_t i) const { return items_[i] != Py_None; }
  const Tensor &operator[](size_t i) const {
    TORCH_CHECK_TYPE(THPVariable_Check(items_[i]), "adamw_step: every ", name_, " must be a tensor");
    return THPVariable_Unpack(items_[i]);
  }

 private:
  const char *name_;
  py::object seq_;
  PyObject **items_ = nullptr;
  size_t size_ = 0;
};

// Whether a step's tensors lie apart in memory.  Where those of a list lie one behind the other and the lists apart, nothing has to be
// sorted.
struct InOrder {
  struct {
    uintptr_t from = 0, to = 0;
  } list[7];
  bool so = true;
  void next(int k, const void *p, size_t bytes) {
    if (bytes == 0) return;
    auto &l = list[k];
    if (l.from == l.to) l.from = (uintptr_t)p;
    so = so && (uintptr_t)p >= l.to;
    l.to = (uintptr_t)p + bytes;
  }
  bool apart() const {
    for (int i = 1; so && i < 7; i++)
      for (int j = 0; j < i; j++)
        if (list[i].from < list[j].to && list[j].from < list[i].to) return false;
    return so;
  }
};
// Else what lies forwards or backwards, most of a list as a rule, is merged.
class Spans {
 public:
  explicit Spans(size_t most) { all_.reserve(most); }
  template <class P> void list(const std::vector<P> &from, const std::vector<int64_t> &numels, size_t bytes, int64_t per, bool written) {
    const size_t first = all_.size();
    for (size_t i = 0; i < from.size(); i++)
      if (numels[i] > 0) all_.push_back({(uintptr_t)from[i], ((uintptr_t)from[i] + bytes * ((numels[i] + per - 1) / per)) << 1 | written});
    for (auto b = all_.begin() + first; b != all_.end();) {
      auto e = std::is_sorted_until(b, all_.end());
      if (e == b + 1) {
        e = std::is_sorted_until(b, all_.end(), [](const Span &x, const Span &y) { return y < x; });
        std::reverse(b, e);
      }
      ends_.push_back(e - all_.begin());
      b = e;
    }
  }
  // Whether nothing that is written shares memory with anything else.
  bool apart() {
    std::vector<Span> other(all_.size());
    while (ends_.size() > 1) {
      std::vector<size_t> ends;
      size_t at = 0;
      for (size_t k = 0; k < ends_.size(); k += 2) {
        const size_t mid = ends_[k], end = k + 1 < ends_.size() ? ends_[k + 1] : mid;
        std::merge(all_.begin() + at, all_.begin() + mid, all_.begin() + mid, all_.begin() + end, other.begin() + at);
        ends.push_back(at = end);
      }
      all_.swap(other), ends_.swap(ends);
    }
    uintptr_t written = 0, read = 0;  // ends of what came so far
    for (const Span &s : all_) {
      const bool w = s.to_written & 1;
      if (s.from < written || (w && s.from < read)) return false;
      uintptr_t &end = w ? written : read;
      end = std::max(end, s.to_written >> 1);
    }
    return true;
  }

 private:
  struct Span {
    uintptr_t from, to_written;  // (the end, and whether it is written in the lowest bit)
    bool operator<(const Span &o) const { return from < o.from; }
  };
  std::vector<Span> all_;
  std::vector<size_t> ends_;
};

void adamw_step(const py::object &params_list, const py::object &grads_list, const py::object &m_list, const py::object &v_list,
                const py::object &masters_list, const py::object &m_scales_list, const py::object &v_scales_list, double step, double lr,
                double beta1, double beta2, double eps, double weight_decay, double grad_scale, const OptTensor &step_at,
                const OptTensor &lr_at) {
  TORCH_CHECK(!at::tracer::impl::is_dispatch_enabled(), "adamw_step cannot be traced: a trace would hold nothing of it");
  const TensorList params(params_list, "param"), grads(grads_list, "grad"), m(m_list, "exp_avg"), v(v_list, "exp_avg_sq"),
      masters(masters_list, "master"), m_scales(m_scales_list, "exp_avg_scale"), v_scales(v_scales_list, "exp_avg_sq_scale");
  const size_t n = params.size();
  TORCH_CHECK(grads.size() == n && m.size() == n && v.size() == n && (!masters || masters.size() == n) && (!m_scales || m_scales.size() == n) &&
                  (!v_scales || v_scales.size() == n),
              "adamw_step: the lists must have the same length");
  TORCH_CHECK((bool)m_scales == (bool)v_scales, "adamw_step: both moments have scales, or neither");
  TORCH_CHECK(lr >= 0 && std::isfinite(lr) && weight_decay >= 0 && eps >= 0, "adamw_step: lr, weight_decay and eps must not be negative");
  TORCH_CHECK(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "adamw_step: betas must be in [0, 1)");
  TORCH_CHECK(step_at || step >= 1, "adamw_step: step counts from 1");
  TORCH_CHECK(!lr_at || step_at, "adamw_step: lr on the device needs step there too");
  if (n == 0) return;
  const bool eight = (bool)m_scales;
  const auto state = eight ? torch::kFloat8_e4m3fn : torch::kFloat;
  const Tensor &like = params[0];
  struct Group {
    int dtype, grad_dtype;
    bool master;
    std::vector<void *> p, m, v;
    std::vector<const void *> g;
    std::vector<float *> w, ms, vs;
    std::vector<int64_t> n;
  };
  std::vector<Group> groups;
  InOrder order;
  const auto fits = [&](const Tensor &t, const char *name, torch::ScalarType type, int64_t numel) -> void * {
    TORCH_CHECK(t.scalar_type() == type, name, " must be ", type, ", got ", t.scalar_type());
    TORCH_CHECK(t.layout() == torch::kStrided && t.is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(t.numel() == numel, name, " must have ", numel, " values, got ", t.numel());
    return t.unsafeGetTensorImpl()->mutable_data();
  };
  // (sizes and types of all first: these refusals need no device)
  for (size_t i = 0; i < n; i++) {
    const Tensor &p = params[i], &g = grads[i];
    const int dtype = element_of(p, "param"), grad_dtype = element_of(g, "grad");
    const bool master = masters && masters.has(i);
    TORCH_CHECK(grad_dtype == dtype || grad_dtype == SPH_F32, "grad must be float32 or have its param's dtype");
    TORCH_CHECK(!master || dtype != SPH_F32, "a float32 param takes no master");
    const int64_t numel = p.numel(), blocks = (numel + 255) / 256;
    size_t at = 0;
    while (at < groups.size() && !(groups[at].dtype == dtype && groups[at].grad_dtype == grad_dtype && groups[at].master == master)) at++;
    if (at == groups.size()) {
      groups.emplace_back();
      Group &q = groups[at];
      q.dtype = dtype, q.grad_dtype = grad_dtype, q.master = master;
      q.p.reserve(n), q.g.reserve(n), q.m.reserve(n), q.v.reserve(n), q.n.reserve(n);
      if (master) q.w.reserve(n);
      if (eight) q.ms.reserve(n), q.vs.reserve(n);
    }
    Group &q = groups[at];
    q.p.push_back(fits(p, "param", p.scalar_type(), numel));
    q.g.push_back(fits(g, "grad", g.scalar_type(), numel));
    q.m.push_back(fits(m[i], "exp_avg", state, numel));
    q.v.push_back(fits(v[i], "exp_avg_sq", state, numel));
    q.n.push_back(numel);
    const size_t state_bytes = eight ? numel : 4 * numel;
    order.next(0, q.p.back(), element_bytes(dtype) * numel);
    order.next(1, q.g.back(), element_bytes(grad_dtype) * numel);
    order.next(2, q.m.back(), state_bytes);
    order.next(3, q.v.back(), state_bytes);
    if (master) q.w.push_back((float *)fits(masters[i], "master", torch::kFloat, numel)), order.next(4, q.w.back(), 4 * numel);
    if (eight) {
      q.ms.push_back((float *)fits(m_scales[i], "exp_avg_scale", torch::kFloat, blocks));
      q.vs.push_back((float *)fits(v_scales[i], "exp_avg_sq_scale", torch::kFloat, blocks));
      order.next(5, q.ms.back(), 4 * blocks);
      order.next(6, q.vs.back(), 4 * blocks);
    }
  }
  const auto scalar = [&](const OptTensor &t, const char *name) -> const float * {
    if (!t) return nullptr;
    TORCH_CHECK(t->scalar_type() == torch::kFloat && t->numel() == 1, name, " must be one float32 value");
    check_device(*t, name, like);
    return t->data_ptr<float>();
  };
  const float *step_p = scalar(step_at, "step"), *lr_p = scalar(lr_at, "lr");
  const c10::Device device = like.device();
  const TensorList *lists[] = {&params, &grads, &m, &v, &masters, &m_scales, &v_scales};
  if (!order.apart()) {
    Spans spans(7 * n);
    for (const Group &q : groups) {
      const size_t state_bytes = eight ? 1 : 4;
      spans.list(q.p, q.n, element_bytes(q.dtype), 1, true);
      spans.list(q.g, q.n, element_bytes(q.grad_dtype), 1, false);
      spans.list(q.m, q.n, state_bytes, 1, true);
      spans.list(q.v, q.n, state_bytes, 1, true);
      spans.list(q.w, q.n, 4, 1, true);
      spans.list(q.ms, q.n, 4, 256, true);
      spans.list(q.vs, q.n, 4, 256, true);
    }
    TORCH_CHECK(spans.apart(), "adamw_step: a tensor that is written appears twice, or overlaps another");
  }
  for (const TensorList *list : lists)
    for (size_t i = 0; *list && i < n; i++)
      if (list->has(i)) {
        const Tensor &t = (*list)[i];
        TORCH_CHECK(t.is_cuda() && t.device() == device, "every tensor of adamw_step must be a CUDA tensor of one device (this build has no CPU path)");
      }
  c10::cuda::CUDAGuard guard(device);
  for (Group &q : groups)
    ok(sph_adamw_step((int64_t)q.n.size(), q.p.data(), q.g.data(), q.master ? q.w.data() : nullptr, q.m.data(), q.v.data(),
                      eight ? q.ms.data() : nullptr, eight ? q.vs.data() : nullptr, q.n.data(), q.dtype, q.grad_dtype, eight ? 8 : 32, lr,
                      beta1, beta2, eps, weight_decay, grad_scale, step, lr_p, step_p, current_stream()),
       "sph_adamw_step");
  // written behind autograd's back: whoever saved one of these tensors has to notice
  for (const TensorList *list : lists)
    for (size_t i = 0; list != &grads && *list && i < n; i++)
      if (list->has(i) && !(*list)[i].is_inference()) (*list)[i].unsafeGetTensorImpl()->bump_version();
}

}  // namespace

void bind_network_ops(pybind11::module_ &m) {
  m.def("rms_norm_op", &rms_norm, py::arg("x"), py::arg("weight"), py::arg("residual"), py::arg("eps"), py::arg("dim"),
        py::arg("inside") = false);
  m.def("rms_norm_quantized", &rms_norm_quantized, py::arg("x"), py::arg("weight"), py::arg("residual"), py::arg("eps"), py::arg("dim"),
        py::arg("inside") = false);
  m.def("token_log_probs_op", &token_log_probs, py::arg("x"), py::arg("target"), py::arg("dim"), py::arg("top_k"),
        py::arg("ignore_index"), py::arg("inside") = false);
  m.def("adamw_step", &adamw_step, py::arg("params"), py::arg("grads"), py::arg("exp_avgs"), py::arg("exp_avg_sqs"), py::arg("masters"),
        py::arg("exp_avg_scales"), py::arg("exp_avg_sq_scales"), py::arg("step"), py::arg("lr"), py::arg("beta1"), py::arg("beta2"),
        py::arg("eps"), py::arg("weight_decay"), py::arg("grad_scale"), py::arg("step_at"), py::arg("lr_at"));
}
