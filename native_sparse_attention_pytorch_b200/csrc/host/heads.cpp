// Rotation of queries and keys by their positions, with or without their norm: the call, and the autograd node around it.

#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <algorithm>
#include <initializer_list>

#include "nsa_host.h"

namespace nsa_host {

namespace {

struct Rotation {
  Tensor steps, positions;       // int64 [rotary_dim / 2]; [n] or [batch, n], or undefined
  int64_t rotary_dim = 0, offset = 0;
  bool half = false, norm = false;
  double magnitude = 1, eps = 0;
};

void require(bool ok, const std::string& what) {
  if (!ok) throw Error("heads: " + what);
}

// The last axis next to itself; the kernels take any other strides
Tensor dense_rows(const Tensor& t) { return t.size(3) == 1 || t.stride(3) == 1 ? t : t.contiguous(); }

// A view that PyTorch negates when it is read (the imaginary part of a conjugate) as values that lie in memory; its gradient passes
Tensor plain(const Tensor& t) { return t.defined() && t.is_neg() ? t.resolve_neg() : t; }

void check_rows(const Tensor& t, const char* name, const Tensor& like, const Rotation& r) {
  require_cuda(t);
  require(t.dim() == 4, std::string(name) + " must be [batch, heads, seq, dim_head]");
  dtype_code(t);
  require(t.device() == like.device() && t.scalar_type() == like.scalar_type(), "queries and keys must share device and type");
  require(t.size(0) == like.size(0) && t.size(2) == like.size(2) && t.size(3) == like.size(3),
          "queries and keys must share batch, seq and dim_head");
  require(r.rotary_dim <= t.size(3), "dim_head is smaller than the rotary dimension");
}

// [d] or [heads, d], of x's type or fp32; both parts' alike
void check_weight(const Tensor& w, const Tensor& x, const char* name) {
  require_cuda(w);
  require(w.device() == x.device(), std::string(name) + " must be on the device of the tensor it belongs to");
  require((w.dim() == 1 && w.size(0) == x.size(3)) || (w.dim() == 2 && w.size(0) == x.size(1) && w.size(1) == x.size(3)),
          std::string(name) + " must be [dim_head] or [heads, dim_head]");
  require(w.scalar_type() == x.scalar_type() || w.scalar_type() == at::kFloat, std::string(name) + " must be of the tensor's type or float32");
}

nsa_heads_args head_args(const Rotation& r, const Tensor& like) {
  nsa_heads_args a = {};
  a.batch = like.size(0); a.seq = like.size(2); a.dim_head = like.size(3);
  a.rotary_dim = r.rotary_dim; a.half = r.half; a.norm = r.norm; a.dtype = dtype_code(like);
  a.magnitude = r.magnitude; a.eps = r.eps; a.offset = r.offset;
  a.steps = reinterpret_cast<const uint64_t*>(r.steps.data_ptr());
  if (r.positions.defined()) {
    a.positions = r.positions.data_ptr();
    a.pos_stride_b = r.positions.dim() == 2 ? r.positions.stride(0) : 0;
    a.pos_i64 = r.positions.scalar_type() == at::kLong;
  }
  return a;
}

// Do strided tensors meet in memory?  Addresses are base + sum index_k step_k, so they do if their bases' difference is a sum of
// e_k step_k with every e_k between the bounds that the sizes set; axes are tried from the widest step down, each over the few numbers
// that leave what the narrower ones can reach.  (ATen's own test answers for dense tensors alone, and neither some heads of a
// projection nor some rows of a cache are dense.)
struct Axis { int64_t step, lo, hi; };      // bytes

class Sums {
 public:
  void add(int64_t step, int64_t lo, int64_t hi) {
    if (step != 0 && lo != hi) axes_.push_back({step, lo, hi});
  }
  // Is there such a sum?  Also true where that is not found out within so many tries
  bool reach(int64_t target) {
    std::sort(axes_.begin(), axes_.end(), [](const Axis& a, const Axis& b) { return a.step > b.step; });
    least_.assign(axes_.size() + 1, 0);
    most_.assign(axes_.size() + 1, 0);
    for (size_t k = axes_.size(); k-- > 0;) {
      least_[k] = least_[k + 1] + axes_[k].lo * axes_[k].step;
      most_[k] = most_[k + 1] + axes_[k].hi * axes_[k].step;
    }
    tries_ = 1 << 16;
    return from(0, target);
  }

 private:
  static int64_t floor_of(int64_t x, int64_t y) { return x / y - (x % y < 0); }
  bool from(size_t k, int64_t target) {
    if (target < least_[k] || target > most_[k]) return false;
    if (k == axes_.size() || --tries_ < 0) return true;
    const Axis& a = axes_[k];
    const int64_t lo = std::max(a.lo, -floor_of(most_[k + 1] - target, a.step)), hi = std::min(a.hi, floor_of(target - least_[k + 1], a.step));
    for (int64_t e = lo; e <= hi; ++e)
      if (from(k + 1, target - e * a.step)) return true;
    return false;
  }
  std::vector<Axis> axes_;
  std::vector<int64_t> least_, most_;
  int tries_ = 0;
};

bool meet(const Tensor& a, const Tensor& b) {
  if (!a.defined() || !b.defined() || a.numel() == 0 || b.numel() == 0) return false;
  Sums sums;
  for (int64_t k = 0; k < a.dim(); ++k) sums.add(a.stride(k) * a.element_size(), 0, a.size(k) - 1);
  for (int64_t k = 0; k < b.dim(); ++k) sums.add(b.stride(k) * b.element_size(), -(b.size(k) - 1), 0);
  sums.add(1, -(int64_t)(b.element_size() - 1), a.element_size() - 1);
  return sums.reach(reinterpret_cast<intptr_t>(b.data_ptr()) - reinterpret_cast<intptr_t>(a.data_ptr()));
}

// Do two elements of a tensor share memory?  Then their indices' first difference, along some axis, is positive for one of them
bool meets_itself(const Tensor& t) {
  if (t.numel() == 0) return false;
  for (int64_t k = 0; k < t.dim(); ++k) {
    if (t.size(k) <= 1) continue;
    if (t.stride(k) == 0) return true;
    Sums sums;
    sums.add(t.stride(k) * t.element_size(), 0, t.size(k) - 2);
    for (int64_t i = k + 1; i < t.dim(); ++i) sums.add(t.stride(i) * t.element_size(), -(t.size(i) - 1), t.size(i) - 1);
    sums.add(1, -(int64_t)(t.element_size() - 1), t.element_size() - 1);
    if (sums.reach(-t.stride(k) * (int64_t)t.element_size())) return true;
  }
  return false;
}

bool same_place(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.sizes() != b.sizes()) return false;
  for (int64_t k = 0; k < a.dim(); ++k)
    if (a.size(k) > 1 && a.stride(k) != b.stride(k)) return false;
  return true;
}

// A thread reads its part of a row before it writes it, so an output may be the tensor that it belongs to, and nothing else that is read
void check_output(const Tensor& out, const Tensor& own, const Tensor& other, const Tensor& other_out, std::initializer_list<Tensor> read) {
  require(!meets_itself(out), "an output must not be broadcast, nor overlap itself");
  require(same_place(out, own) || !meet(out, own), "an output may be the tensor itself, but must not overlap it otherwise");
  require(!meet(out, other) && !meet(out, other_out), "an output of one of the tensors must not overlap the other's");
  for (const Tensor& t : read) require(!meet(out, t), "an output must not overlap the weights, the positions or the frequencies");
  require(!at::GradMode::is_enabled() || !out.requires_grad(), "an output that wants gradients itself cannot be given");
}

// Shapes that do not fit the C structs' 32 bits
void check_sizes(const Tensor& t) {
  for (int64_t s : t.sizes()) require(s <= 0x7fffffff, "a size is above 2^31");
}

void set_weight(nsa_heads_args& a, int part, const Tensor& w, const Tensor& x) {
  a.part[part].weight = w.data_ptr();
  a.weight_per_head = w.dim() == 2;
  a.weight_f32 = w.scalar_type() == at::kFloat && x.scalar_type() != at::kFloat;
}

// Uninitialised tensor of these sizes whose dimensions lie in memory in the order that the strides say
Tensor empty_in_order(at::IntArrayRef sizes, at::IntArrayRef strides, const at::TensorOptions& options) {
  std::vector<int64_t> order = {0, 1, 2, 3}, in_order(4), back(4);
  std::stable_sort(order.begin(), order.end() - 1, [&](int64_t a, int64_t b) { return strides[a] > strides[b]; });
  for (int64_t i = 0; i < 4; ++i) {
    in_order[i] = sizes[order[i]];
    back[order[i]] = i;
  }
  return at::empty(in_order, options).permute(back);
}

// dx in the memory order of x, dw as w
struct Gradients {
  Tensor dx[2], dw[2];
};

struct RotatedHeadsBackward : torch::autograd::Node {
  Rotation r;
  torch::autograd::SavedVariable x[2], w[2];     // with norm
  torch::autograd::SavedVariable positions;      // kept as a saved tensor, so that one overwritten before the backward pass is refused
  // what the gradients look like (without norm nothing of the inputs is kept)
  at::TensorOptions options;
  std::vector<int64_t> sizes[2], strides[2];
  bool by_positions = false;

  void release_variables() override {
    for (auto* t : {&x[0], &x[1], &w[0], &w[1], &positions}) t->reset_data();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    torch::autograd::variable_list out(4);
    Tensor dy[2] = {grads[0], grads.size() > 1 ? grads[1] : Tensor()};     // without keys there is one result
    if (!dy[0].defined() && !dy[1].defined()) return out;
    try {
      const at::NoGradGuard no_grad;
      Tensor xs[2], ws[2];
      for (int i = 0; i < 2; ++i) {
        if (sizes[i].empty() || !r.norm) continue;
        xs[i] = x[i].unpack(getptr());
        ws[i] = w[i].unpack(getptr());
      }
      Rotation turn = r;
      if (by_positions) turn.positions = positions.unpack(getptr());
      Gradients g = heads_backward(turn, xs, ws, dy);
      for (int i = 0; i < 2; ++i) {
        if (task_should_compute_output(i)) out[i] = g.dx[i];
        if (r.norm && task_should_compute_output(2 + i)) out[2 + i] = g.dw[i];
      }
    } catch (const Error& e) {
      raise_python_error(e.what());
    }
    if (at::GradMode::is_enabled()) {   // create_graph: the gradients are there, their own gradients are not
      for (auto& t : out)
        if (t.defined()) t.set_requires_grad(true);
      torch::autograd::DelayedError fail("trying to differentiate twice the native backward of the rotation of heads", 4);
      return fail.apply(std::move(out));
    }
    return out;
  }

  Gradients heads_backward(const Rotation& r, const Tensor* x, const Tensor* w, const Tensor* dy) const;
};

// A tensor whose result gets no gradient has none itself
Gradients RotatedHeadsBackward::heads_backward(const Rotation& r, const Tensor* x, const Tensor* w, const Tensor* dy) const {
  const c10::cuda::CUDAGuard guard(options.device());
  Gradients g;
  Tensor rows[2];
  nsa_heads_args a = {};
  bool begun = false;
  for (int i = 0; i < 2; ++i) {
    if (sizes[i].empty() || !dy[i].defined()) continue;
    g.dx[i] = empty_in_order(sizes[i], strides[i], options);
    rows[i] = dense_rows(plain(dy[i]));
    if (!begun) a = head_args(r, g.dx[i]);
    begun = true;
    a.part[i].heads = g.dx[i].size(1);
    a.part[i].out = t4(g.dx[i]);
    a.part[i].dy = t4(rows[i]);
    if (r.norm) {
      a.part[i].x = t4(x[i]);
      set_weight(a, i, w[i], x[i]);
      // (a tensor without heads is not there for the kernels)
      g.dw[i] = x[i].size(1) > 0 ? at::empty(w[i].sizes(), w[i].options()) : at::zeros(w[i].sizes(), w[i].options());
      a.part[i].dweight = g.dw[i].data_ptr();
    }
  }
  Tensor ws;
  if (r.norm) {
    ws = at::empty({nsa_heads_workspace_bytes(&a)}, options.dtype(at::kByte));
    a.workspace = ws.data_ptr();
    a.workspace_bytes = ws.numel();
  }
  check(nsa_heads_bwd(&a, c10::cuda::getCurrentCUDAStream(options.device().index()).stream()));
  return g;
}

}  // namespace

// -> the rotated queries and keys
static std::vector<OptTensor> rotate_heads(Tensor q, OptTensor k_, OptTensor wq, OptTensor wk, Tensor steps, int64_t rotary_dim, bool half,
                                           double magnitude, OptTensor positions, int64_t offset, bool norm, double eps,
                                           OptTensor out_q, OptTensor out_k) {
  Rotation r;
  r.steps = steps; r.rotary_dim = rotary_dim; r.half = half; r.magnitude = magnitude; r.offset = offset; r.norm = norm; r.eps = eps;
  q = plain(q);
  Tensor x[2] = {q, plain(k_.value_or(Tensor()))}, w[2] = {plain(wq.value_or(Tensor())), plain(wk.value_or(Tensor()))};
  Tensor given[2] = {out_q.value_or(Tensor()), out_k.value_or(Tensor())};
  bool wanted = false;
  require_cuda(q);
  require(q.dim() == 4, "queries must be [batch, heads, seq, dim_head]");
  require(steps.device() == q.device(), "the frequencies are on another device");
  for (int i = 0; i < 2; ++i) {
    if (!x[i].defined()) {
      require(!w[i].defined() && !given[i].defined(), "a weight or an output of keys without keys");
      continue;
    }
    check_rows(x[i], i ? "keys" : "queries", q, r);
    check_sizes(x[i]);
    wanted = wanted || x[i].requires_grad();
    if (norm) {
      require(w[i].defined(), "the norm needs a weight for each of the tensors");
      check_weight(w[i], x[i], i ? "the keys' weight" : "the queries' weight");
      require(i == 0 || (w[0].dim() == w[1].dim() && w[0].scalar_type() == w[1].scalar_type()), "both weights must be of one form and type");
      wanted = wanted || w[i].requires_grad();
    }
    if (given[i].defined())
      require(given[i].device() == x[i].device() && given[i].scalar_type() == x[i].scalar_type() && given[i].sizes() == x[i].sizes() &&
                  (x[i].size(3) == 1 || given[i].stride(3) == 1) && !given[i].is_neg(),
              "an output must have the tensor's device, type and shape, a contiguous last axis, and not be negated");
  }
  for (int i = 0; i < 2; ++i)
    if (given[i].defined()) check_output(given[i], x[i], x[1 - i], given[1 - i], {w[0], w[1], positions.value_or(Tensor()), steps});
  wanted = wanted && at::GradMode::is_enabled();
  require(!wanted || (!given[0].defined() && !given[1].defined()), "outputs cannot be given where gradients are wanted");
  if (positions.has_value() && positions->defined()) {
    Tensor p = *positions;
    require_cuda(p);
    require(p.device() == q.device(), "positions are on another device");
    require(p.scalar_type() == at::kLong || p.scalar_type() == at::kInt, "positions must be int64 or int32");
    require((p.dim() == 1 || (p.dim() == 2 && (p.size(0) == q.size(0) || p.size(0) == 1))) && p.size(-1) == q.size(2),
            "positions must be [seq], or [batch, seq]");
    if (p.dim() == 2 && p.size(0) == 1) p = p[0];
    if (p.size(-1) > 1 && p.stride(-1) != 1) p = p.contiguous();
    r.positions = p;
  }

  const c10::cuda::CUDAGuard guard(q.device());
  Tensor y[2], seen[2], weight[2];
  {
    const at::NoGradGuard no_grad;
    nsa_heads_args a = head_args(r, q);
    for (int i = 0; i < 2; ++i) {
      if (!x[i].defined()) continue;
      seen[i] = dense_rows(x[i]);
      y[i] = given[i].defined() ? given[i] : at::empty(x[i].sizes(), x[i].options());
      a.part[i].heads = x[i].size(1);
      a.part[i].x = t4(seen[i]);
      a.part[i].out = t4(y[i]);
      if (norm) {
        weight[i] = w[i].contiguous();
        set_weight(a, i, weight[i], x[i]);
      }
    }
    check(nsa_heads_fwd(&a, stream_of(q)));
    for (const Tensor& t : given)        // as any write in place: whoever saved these for a backward pass learns of it
      if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  if (wanted) {
    using torch::autograd::SavedVariable;
    auto node = std::shared_ptr<RotatedHeadsBackward>(new RotatedHeadsBackward, torch::autograd::deleteNode);
    auto edge = [](const Tensor& t) { return t.defined() ? torch::autograd::impl::gradient_edge(t) : torch::autograd::Edge(); };
    node->set_next_edges({edge(x[0]), edge(x[1]), edge(w[0]), edge(w[1])});
    node->r = r;
    node->r.positions = Tensor();
    node->by_positions = r.positions.defined();
    if (node->by_positions) node->positions = SavedVariable(r.positions.is_inference() ? r.positions.clone() : r.positions, false);
    node->options = q.options();
    for (int i = 0; i < 2; ++i) {
      if (!x[i].defined()) continue;
      node->sizes[i] = x[i].sizes().vec();
      node->strides[i] = x[i].strides().vec();
      if (norm) {
        node->x[i] = SavedVariable(seen[i], false);
        node->w[i] = SavedVariable(weight[i], false);
      }
    }
    std::vector<Tensor> results;
    for (const Tensor& t : y)
      if (t.defined()) results.push_back(t);
    torch::autograd::set_history(results, node);
  }
  return {y[0], y[1].defined() ? OptTensor(y[1]) : OptTensor()};
}

void bind_heads(pybind11::module_& m) {
  m.def("rotate_heads", &rotate_heads, pybind11::call_guard<pybind11::gil_scoped_release>());
  // what outputs are checked by, on any tensors
  m.def("tensors_meet", &meet);
  m.def("tensor_meets_itself", &meets_itself);
}

}  // namespace nsa_host
