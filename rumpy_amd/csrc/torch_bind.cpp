// torch binding of the row operators (residual_norm.hip, distill.hip): checks of arguments, allocation of outputs and workspaces, launches and autograd
// nodes in C++.  A call is then bound by its launches: with the nodes in Python a training pass of two short kernels spent 95 - 190 us of host time in
// two threads (the autograd engine runs a node in a thread of its own), several times what the GPU needed.
// The kernels stay behind the C ABI: their addresses come from the loaded library (bind), so this file links to torch alone and is plain C++.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/rumpy_amd.h"

namespace {
using at::Tensor;
using std::optional;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

// ---- entry points of the kernel library
struct Entries {
  decltype(&rumpy_residual_norm_fwd) norm_fwd = nullptr;
  decltype(&rumpy_residual_norm_bwd) norm_bwd = nullptr;
  decltype(&rumpy_residual_norm_partial_floats) norm_partial = nullptr;
  decltype(&rumpy_top_logits) top = nullptr;
  decltype(&rumpy_top_logits_work_bytes) top_work = nullptr;
  decltype(&rumpy_distill_fwd) distill_fwd = nullptr;
  decltype(&rumpy_distill_bwd) distill_bwd = nullptr;
  decltype(&rumpy_distill_partial_floats) distill_partial = nullptr;
  decltype(&rumpy_last_error) last_error = nullptr;
} lib;

void bind(const std::map<std::string, uint64_t>& at) {
  auto set = [&](auto& fn, const char* name) { fn = reinterpret_cast<std::decay_t<decltype(fn)>>(at.at(name)); };
  set(lib.norm_fwd, "rumpy_residual_norm_fwd");
  set(lib.norm_bwd, "rumpy_residual_norm_bwd");
  set(lib.norm_partial, "rumpy_residual_norm_partial_floats");
  set(lib.top, "rumpy_top_logits");
  set(lib.top_work, "rumpy_top_logits_work_bytes");
  set(lib.distill_fwd, "rumpy_distill_fwd");
  set(lib.distill_bwd, "rumpy_distill_bwd");
  set(lib.distill_partial, "rumpy_distill_partial_floats");
  set(lib.last_error, "rumpy_last_error");
}

// one launch on the current stream of the tensors' own device (the caller holds the device guard)
template <typename Fn, typename Args> void launch(const char* name, Fn fn, const Args& args, const at::Device& dev) {
  const int rc = fn(&args, c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream());
  TORCH_CHECK(rc == 0, "rumpy_amd ", name, " failed (", rc, "): ", lib.last_error());
}

// ---- tensors
constexpr int64_t MAX_CHANNELS = 8192, MAX_TOP = 256, MAX_COLUMNS = int64_t(1) << 30;

int fmt_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return RUMPY_FMT_F32;
    case at::kBFloat16: return RUMPY_FMT_BF16;
    case at::kHalf: return RUMPY_FMT_F16;
    default: return -1;
  }
}
std::string name_of(const Tensor& t) { return c10::getDtypeNames(t.scalar_type()).first; }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
const float* fptr(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
void* out_ptr(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
float* out_fptr(const Tensor& t) { return static_cast<float*>(out_ptr(t)); }
Tensor or_none(const optional<Tensor>& t) { return t ? *t : Tensor(); }

// rows of contiguous channels at one stride; copied only where they do not lie so
struct Rows {
  Tensor t;
  int64_t ld = 0;
  Rows() = default;
  explicit Rows(const Tensor& from) : t(from) {
    if (!t.defined()) return;
    const int64_t d = t.dim();
    ld = t.size(-1);
    if (t.is_contiguous()) return;
    if (t.stride(-1) == 1) {
      // the dimensions in front are one when each step is the whole of the next (dimensions of one entry have no step)
      int64_t step = -1, whole = 1;
      bool one = true;
      for (int64_t i = d - 2; i >= 0; --i) {
        if (t.size(i) == 1) continue;
        if (step < 0) step = t.stride(i);
        else one = one && t.stride(i) == step * whole;
        whole *= t.size(i);
      }
      if (one) { if (step >= 0) ld = step; return; }
    }
    t = t.contiguous();
  }
};
Tensor new_like(const Tensor& t) { return at::empty(t.sizes(), t.options()); }
Tensor new_floats(at::IntArrayRef shape, const Tensor& beside) { return at::empty(shape, beside.options().dtype(at::kFloat)); }

bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts) if (t->defined() && t->requires_grad()) return true;
  return false;
}
void no_forward_mode(const char* name, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts) TORCH_CHECK(!torch::autograd::isFwGradDefined(*t), "rumpy_amd: ", name, " has no forward-mode derivative");
}
void need_gpu(const char* name, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "rumpy_amd: ", name, " runs on an MI355X through the HIP extension; there is no CPU path");
}
// (grad mode is on in a backward pass under create_graph=True alone)
void once_differentiable(const char* name) { TORCH_CHECK(!at::GradMode::is_enabled(), "rumpy_amd: ", name, " has no second derivative"); }

// ================================================================================================================ residual_norm
struct NormCfg { int post, pre, gate_mode; int64_t group_rows; float scale, eps; };
constexpr int GATE_NONE = 0, GATE_GROUP = 1, GATE_FULL = 2;

Tensor plain_gate(const Tensor& gate, int mode) { return gate.defined() && mode != GATE_FULL ? gate.contiguous() : gate; }

void norm_forward(const Tensor& x, const Tensor& branch, const Tensor& gate, const Tensor& pw, const Tensor& pb, const Tensor& w, const Tensor& b, const NormCfg& cfg,
                  bool keep, Tensor& y, Tensor& h, Tensor& stats) {
  const int64_t c = x.size(-1), rows = x.numel() / c;
  const Tensor& tb = branch.defined() ? branch : x;
  if (branch.defined()) y = new_like(x);
  if (cfg.pre) h = new_like(tb);
  if (keep) stats = new_floats({rows, 4}, x);
  if (rows == 0) return;
  const c10::DeviceGuard guard(x.device());
  const Rows rx(x), rt(branch), rg(cfg.gate_mode == GATE_FULL ? gate : Tensor());
  const Tensor g = cfg.gate_mode == GATE_FULL ? rg.t : plain_gate(gate, cfg.gate_mode);
  rumpy_residual_norm_args a{};
  a.x = ptr(rx.t); a.t = ptr(rt.t); a.gate = ptr(g);
  a.post_w = fptr(pw); a.post_b = fptr(pb); a.pre_w = fptr(w); a.pre_b = fptr(b);
  a.y = out_ptr(y); a.h = out_ptr(h); a.stats = out_fptr(stats);
  a.rows = rows; a.group_rows = cfg.group_rows; a.ldx = rx.ld; a.ldt = rt.ld; a.ldg = rg.ld;
  a.C = (int32_t)c; a.x_fmt = fmt_of(x); a.t_fmt = fmt_of(tb); a.gate_mode = cfg.gate_mode; a.post = cfg.post; a.pre = cfg.pre;
  a.scale = cfg.scale; a.eps = cfg.eps;
  launch("rumpy_residual_norm_fwd", lib.norm_fwd, a, x.device());
}

struct ResidualNormBackward : public torch::autograd::Node {
  NormCfg cfg;
  bool has_y = false, has_h = false;
  SavedVariable x_, branch_, gate_, pw_, pb_, w_;
  Tensor stats_;
  std::string name() const override { return "ResidualNormBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    x_.reset_data(); branch_.reset_data(); gate_.reset_data(); pw_.reset_data(); pb_.reset_data(); w_.reset_data();
    stats_.reset();
  }
  // edges: x, branch, gate, post weight, post bias, pre weight, pre bias
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);          // (backward passes of one graph in several threads)
    once_differentiable("residual_norm");
    const Tensor dy = has_y ? grads[0] : Tensor(), dh = has_h ? grads[has_y ? 1 : 0] : Tensor();
    variable_list out(7);
    if (!dy.defined() && !dh.defined()) return out;
    const Tensor x = x_.unpack(), branch = branch_.unpack(), gate = gate_.unpack(), pw = pw_.unpack(), pb = pb_.unpack(), w = w_.unpack();
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    const int64_t c = x.size(-1), rows = x.numel() / c;
    const Tensor& tb = branch.defined() ? branch : x;
    if (task_should_compute_output(0)) out[0] = new_like(x);
    if (task_should_compute_output(1)) out[1] = new_like(branch);
    if (task_should_compute_output(2)) out[2] = new_like(gate);
    // (where nothing arrives through the norm in front, its parameters have no gradient)
    for (int i = 3; i < (dh.defined() ? 7 : 5); ++i) if (task_should_compute_output(i)) out[i] = new_floats({c}, x);
    if (rows == 0) {
      for (Tensor& t : out) if (t.defined()) t.zero_();
      return out;
    }
    const Rows rx(x), rt(branch), rdy(dy), rdh(dh), rg(cfg.gate_mode == GATE_FULL ? gate : Tensor());
    const Tensor g = cfg.gate_mode == GATE_FULL ? rg.t : plain_gate(gate, cfg.gate_mode);
    const Tensor partial = new_floats({lib.norm_partial(rows, cfg.group_rows, (int32_t)c, cfg.gate_mode)}, x);
    rumpy_residual_norm_bwd_args a{};
    a.dy = ptr(rdy.t); a.dh = ptr(rdh.t); a.x = ptr(rx.t); a.t = ptr(rt.t); a.gate = ptr(g);
    a.post_w = fptr(pw); a.post_b = fptr(pb); a.pre_w = fptr(w); a.stats = fptr(stats_);
    a.dx = out_ptr(out[0]); a.dt = out_ptr(out[1]); a.dgate = out_ptr(out[2]);
    a.d_post_w = out_fptr(out[3]); a.d_post_b = out_fptr(out[4]); a.d_pre_w = out_fptr(out[5]); a.d_pre_b = out_fptr(out[6]);
    a.partial = out_fptr(partial);
    a.rows = rows; a.group_rows = cfg.group_rows; a.lddy = rdy.ld; a.lddh = rdh.ld; a.ldx = rx.ld; a.ldt = rt.ld; a.ldg = rg.ld;
    a.C = (int32_t)c; a.x_fmt = fmt_of(x); a.t_fmt = fmt_of(tb); a.gate_mode = cfg.gate_mode; a.post = cfg.post; a.pre = cfg.pre; a.scale = cfg.scale;
    launch("rumpy_residual_norm_bwd", lib.norm_bwd, a, x.device());
    return out;
  }
};

int norm_kind(const optional<std::string>& k) {
  if (!k) return 0;
  if (*k == "layer") return 1;
  if (*k == "rms") return 2;
  TORCH_CHECK_VALUE(false, "rumpy_amd: residual_norm knows the norms 'layer' and 'rms', not '", *k, "'");
}
Tensor norm_param(const optional<Tensor>& p, const char* name, int kind, int64_t c, const at::Device& dev) {
  if (!p) return Tensor();
  TORCH_CHECK_VALUE(kind, "rumpy_amd: residual_norm has ", name, " but no norm it belongs to");
  TORCH_CHECK_VALUE(p->dim() == 1 && p->size(0) == c && p->scalar_type() == at::kFloat && p->device() == dev, "rumpy_amd: residual_norm takes ", name,
                    " as float32 [", c, "] beside its input, not ", name_of(*p), " ", p->sizes());
  return p->is_contiguous() ? *p : p->contiguous();
}

std::pair<Tensor, optional<Tensor>> residual_norm(const Tensor& x, const optional<Tensor>& branch_, const optional<Tensor>& gate_, double scale,
                                                  const optional<std::string>& post_norm, const optional<Tensor>& post_weight, const optional<Tensor>& post_bias,
                                                  const optional<std::string>& pre_norm, const optional<Tensor>& pre_weight, const optional<Tensor>& pre_bias,
                                                  double eps) {
  NormCfg cfg{norm_kind(post_norm), norm_kind(pre_norm), GATE_NONE, 0, (float)scale, (float)eps};
  TORCH_CHECK_VALUE(eps >= 1e-30 && eps < 1e30, "rumpy_amd: residual_norm takes an eps above zero, not ", eps);
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= MAX_CHANNELS, "rumpy_amd: residual_norm takes [..., C] with 1 <= C <= ", MAX_CHANNELS, ", not ",
                    x.sizes());
  const Tensor branch = or_none(branch_), gate = or_none(gate_);
  const int64_t c = x.size(-1), rows = x.numel() / c;
  if (!branch.defined()) {
    TORCH_CHECK_VALUE(!gate.defined() && !cfg.post && cfg.pre, "rumpy_amd: residual_norm without a branch is the norm in front alone");
    TORCH_CHECK(fmt_of(x) >= 0, "rumpy_amd: residual_norm takes float32, bfloat16 or float16, not ", name_of(x));
  } else {
    TORCH_CHECK_VALUE(branch.sizes() == x.sizes() && branch.device() == x.device(), "rumpy_amd: residual_norm takes a branch like x, ", x.sizes(), ", not ",
                      branch.sizes());
    TORCH_CHECK(fmt_of(x) >= 0 && fmt_of(branch) >= 0 && (x.scalar_type() == branch.scalar_type() || x.scalar_type() == at::kFloat),
                "rumpy_amd: residual_norm takes x and branch in one of float32, bfloat16, float16, or x in float32 beside a 16-bit branch, not ", name_of(x),
                " and ", name_of(branch));
    if (gate.defined()) {
      TORCH_CHECK_VALUE(gate.device() == x.device(), "rumpy_amd: residual_norm takes a gate beside x");
      const bool f32 = gate.scalar_type() == at::kFloat;
      if (f32 && gate.dim() == 1 && gate.size(0) == c) {
        cfg.gate_mode = GATE_GROUP;
        cfg.group_rows = std::max<int64_t>(rows, 1);
      } else if (gate.sizes() == x.sizes() && gate.scalar_type() == branch.scalar_type()) {
        cfg.gate_mode = GATE_FULL;
      } else if (f32 && x.dim() >= 2 && gate.dim() == 2 && gate.size(0) == x.size(0) && gate.size(1) == c) {
        cfg.gate_mode = GATE_GROUP;
        cfg.group_rows = std::max<int64_t>(rows / std::max<int64_t>(x.size(0), 1), 1);
      } else {
        TORCH_CHECK_VALUE(false, "rumpy_amd: residual_norm takes a gate as float32 [C], float32 [", x.size(0), ", C] or like the branch, not ", name_of(gate), " ",
                          gate.sizes());
      }
    }
  }
  const Tensor pw = norm_param(post_weight, "post_weight", cfg.post, c, x.device()), pb = norm_param(post_bias, "post_bias", cfg.post, c, x.device());
  const Tensor w = norm_param(pre_weight, "pre_weight", cfg.pre, c, x.device()), b = norm_param(pre_bias, "pre_bias", cfg.pre, c, x.device());
  need_gpu("residual_norm", x);
  no_forward_mode("residual_norm", {&x, &branch, &gate, &pw, &pb, &w, &b});
  const bool grad = wants_grad({&x, &branch, &gate, &pw, &pb, &w, &b});
  Tensor y, h, stats;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    norm_forward(x, branch, gate, pw, pb, w, b, cfg, grad, y, h, stats);
  }
  if (grad) {
    auto node = std::shared_ptr<ResidualNormBackward>(new ResidualNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, branch, gate, pw, pb, w, b));
    node->cfg = cfg;
    node->has_y = y.defined();
    node->has_h = h.defined();
    node->x_ = SavedVariable(x, false);
    node->branch_ = SavedVariable(branch, false);
    node->gate_ = SavedVariable(gate, false);
    node->pw_ = SavedVariable(pw, false);
    node->pb_ = SavedVariable(pb, false);
    node->w_ = SavedVariable(w, false);
    node->stats_ = stats;
    if (y.defined()) torch::autograd::set_history(y, node);
    if (h.defined()) torch::autograd::set_history(h, node);
  }
  return {branch.defined() ? y : x, h.defined() ? optional<Tensor>(h) : std::nullopt};
}

// ================================================================================================================ distillation
double check_logits(const char* name, const Tensor& logits, double temperature) {
  TORCH_CHECK(fmt_of(logits) >= 0, "rumpy_amd: ", name, " takes float32, bfloat16 or float16 logits, not ", name_of(logits));
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= MAX_COLUMNS, "rumpy_amd: ", name, " takes [..., V] logits with V >= 1, not ",
                    logits.sizes());
  TORCH_CHECK_VALUE(temperature > 1e-30 && temperature < 1e30, "rumpy_amd: ", name, " takes a temperature above zero, not ", temperature);
  return temperature;
}

std::tuple<Tensor, Tensor, Tensor> top_logits(const Tensor& logits, int64_t k, double temperature) {
  const double tau = check_logits("top_logits", logits, temperature);
  const int64_t v = logits.size(-1), rows = logits.numel() / v;
  TORCH_CHECK_VALUE(k >= 1 && k <= std::min(v, MAX_TOP), "rumpy_amd: top_logits takes 1 <= k <= ", MAX_TOP, " of rows of ", v, " logits, not ", k);
  need_gpu("top_logits", logits);
  const at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(logits.device());
  auto shape = logits.sizes().vec();
  shape.back() = k;
  const Tensor values = at::empty(shape, logits.options()), indices = at::empty(shape, logits.options().dtype(at::kLong));
  const Tensor tail = new_floats(logits.sizes().slice(0, logits.dim() - 1), logits);
  if (rows) {
    const Rows z(logits);
    const int64_t bytes = lib.top_work(rows, (int32_t)v, (int32_t)k);
    const Tensor work = bytes ? new_floats({(bytes + 3) / 4}, logits) : Tensor();
    rumpy_top_logits_args a{};
    a.logits = ptr(z.t); a.values = out_ptr(values); a.indices = out_ptr(indices); a.tail = out_fptr(tail); a.work = out_ptr(work);
    a.rows = rows; a.ld = z.ld; a.V = (int32_t)v; a.k = (int32_t)k; a.fmt = fmt_of(logits); a.tau = tau;
    launch("rumpy_top_logits", lib.top, a, logits.device());
  }
  return {values, indices, tail};
}

enum Reduction { NONE, SUM, MEAN };

// what both directions give to the kernels; state: [rows, 8], the reduction's factor, the workspace of rows that are cut, the rows' losses
rumpy_distill_args distill_args(const Rows& z, int64_t v, const Tensor& values, const Tensor& indices, const Tensor& tail, const Tensor& weight, const Tensor& state,
                                Reduction reduction, double tau) {
  const int64_t rows = z.t.numel() / v;
  rumpy_distill_args a{};
  a.logits = ptr(z.t); a.top_values = ptr(values); a.top_indices = ptr(indices); a.tail = fptr(tail); a.row_weight = fptr(weight);
  a.state = out_fptr(state); a.factor = a.state + 8 * rows;
  const int64_t pf = lib.distill_partial(rows, (int32_t)v);
  a.partial = pf ? a.factor + 1 : nullptr;
  a.row_loss = a.factor + 1 + pf;
  a.rows = rows; a.ld = z.ld; a.V = (int32_t)v; a.k = (int32_t)values.size(-1); a.fmt = fmt_of(z.t); a.value_fmt = fmt_of(values);
  a.index64 = indices.scalar_type() == at::kLong; a.mean = reduction == MEAN; a.tau = tau;
  return a;
}

struct DistillBackward : public torch::autograd::Node {
  Reduction reduction;
  double tau;
  SavedVariable logits_, values_, indices_, tail_, weight_;
  Tensor state_;
  std::string name() const override { return "DistillBackward"; }
  void release_variables() override {
    const std::lock_guard<std::mutex> lock(mutex_);
    logits_.reset_data(); values_.reset_data(); indices_.reset_data(); tail_.reset_data(); weight_.reset_data();
    state_.reset();
  }
  variable_list apply(variable_list&& grads) override {
    const std::lock_guard<std::mutex> lock(mutex_);
    once_differentiable("distill_loss");
    if (!grads[0].defined() || !task_should_compute_output(0)) return {Tensor()};
    const Tensor logits = logits_.unpack(), values = values_.unpack(), indices = indices_.unpack(), tail = tail_.unpack(), weight = weight_.unpack();
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(logits.device());
    const Tensor g = grads[0].contiguous(), dl = new_like(logits);
    if (logits.numel()) {
      const Rows z(logits);
      rumpy_distill_args a = distill_args(z, logits.size(-1), values, indices, tail, weight, state_, reduction, tau);
      a.gout = fptr(g);
      a.dlogits = out_ptr(dl);
      a.loss = reduction == NONE ? nullptr : a.row_loss;          // (says that g is the gradient of one number; nothing but dlogits is written)
      launch("rumpy_distill_bwd", lib.distill_bwd, a, logits.device());
    }
    return {dl};
  }
};

Tensor distill_loss(const Tensor& logits, const Tensor& top_values, const Tensor& top_indices, const optional<Tensor>& tail_, double temperature,
                    const optional<Tensor>& weight_, const std::string& reduction_) {
  const double tau = check_logits("distill_loss", logits, temperature);
  TORCH_CHECK_VALUE(reduction_ == "mean" || reduction_ == "sum" || reduction_ == "none", "rumpy_amd: distill_loss reduces by 'mean', 'sum' or 'none', not '", reduction_, "'");
  const Reduction reduction = reduction_ == "mean" ? MEAN : reduction_ == "sum" ? SUM : NONE;
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(top_values.sizes() == top_indices.sizes() && top_values.dim() == logits.dim() && top_values.sizes().slice(0, logits.dim() - 1) == lead &&
                        top_values.size(-1) >= 1 && top_values.size(-1) <= MAX_TOP,
                    "rumpy_amd: distill_loss takes top logits and indices ", lead, " + [k] with k <= ", MAX_TOP, ", not ", top_values.sizes(), " and ", top_indices.sizes());
  TORCH_CHECK(fmt_of(top_values) >= 0 && (top_indices.scalar_type() == at::kLong || top_indices.scalar_type() == at::kInt),
              "rumpy_amd: distill_loss takes float32, bfloat16 or float16 top logits with int64 or int32 indices, not ", name_of(top_values), " and ",
              name_of(top_indices));
  TORCH_CHECK_VALUE(!tail_ || tail_->sizes() == lead, "rumpy_amd: distill_loss takes tail ", lead, ", not ", tail_->sizes());
  TORCH_CHECK_VALUE(!weight_ || weight_->sizes() == lead, "rumpy_amd: distill_loss takes row_weight ", lead, ", not ", weight_->sizes());
  Tensor values = top_values, indices = top_indices, tail = or_none(tail_), weight = or_none(weight_);
  for (const Tensor* t : {&values, &indices, &tail, &weight})
    TORCH_CHECK_VALUE(!t->defined() || t->device() == logits.device(), "rumpy_amd: distill_loss takes its tensors on one device, ", logits.device(), ", not ", t->device());
  need_gpu("distill_loss", logits);
  no_forward_mode("distill_loss", {&logits, &values, &tail, &weight});
  const bool grad = wants_grad({&logits});
  Tensor loss, state;
  {
    const at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(logits.device());
    values = values.contiguous();
    indices = indices.contiguous();
    if (tail.defined()) tail = tail.to(at::kFloat).contiguous();
    if (weight.defined()) weight = weight.to(at::kFloat).contiguous();
    const Rows z(logits);
    const int64_t v = logits.size(-1), rows = logits.numel() / v;
    state = new_floats({rows * 9 + 1 + lib.distill_partial(rows, (int32_t)v)}, logits);
    loss = new_floats(reduction == NONE ? lead : at::IntArrayRef{}, logits);
    rumpy_distill_args a = distill_args(z, v, values, indices, tail, weight, state, reduction, tau);
    if (reduction == NONE) a.row_loss = out_fptr(loss);
    else a.loss = out_fptr(loss);
    if (rows || a.loss) launch("rumpy_distill_fwd", lib.distill_fwd, a, logits.device());
  }
  if (grad) {
    auto node = std::shared_ptr<DistillBackward>(new DistillBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->reduction = reduction;
    node->tau = tau;
    node->logits_ = SavedVariable(logits, false);
    node->values_ = SavedVariable(values, false);
    node->indices_ = SavedVariable(indices, false);
    node->tail_ = SavedVariable(tail, false);
    node->weight_ = SavedVariable(weight, false);
    node->state_ = state;
    torch::autograd::set_history(loss, node);
  }
  return loss;
}
}  // namespace

PYBIND11_MODULE(_torch_bind, m) {
  namespace py = pybind11;
  m.def("bind", &bind);
  m.def("residual_norm", &residual_norm, py::arg("x"), py::arg("branch"), py::arg("gate"), py::arg("scale"), py::arg("post_norm"), py::arg("post_weight"),
        py::arg("post_bias"), py::arg("pre_norm"), py::arg("pre_weight"), py::arg("pre_bias"), py::arg("eps"), py::call_guard<py::gil_scoped_release>());
  m.def("top_logits", &top_logits, py::arg("logits"), py::arg("k"), py::arg("temperature"),
        py::call_guard<py::gil_scoped_release>());
  m.def("distill_loss", &distill_loss, py::arg("logits"), py::arg("top_values"), py::arg("top_indices"), py::arg("tail"), py::arg("temperature"), py::arg("row_weight"),
        py::arg("reduction"), py::call_guard<py::gil_scoped_release>());
}
