// PyTorch front end of the block-norm operators of libfln_b200 (fln_norm_gate_add_norm_*,
// fln_qk_norm_rotary_*): argument checks, allocation, autograd nodes, operator registrations.
// Like fln_torch_shim.cpp it does no arithmetic; errors are RuntimeErrors, unsupported dtypes
// NotImplementedErrors, and there is no CPU path.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/autograd.h>
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "fln_b200.h"
#include "fln_torch_blocks.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

int dtype_code(const Tensor& t, const char* op) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return FLN_F32;
    case at::kBFloat16:
      return FLN_BF16;
    case at::kHalf:
      return FLN_F16;
    default:
      TORCH_CHECK_NOT_IMPLEMENTED(false, "\"", op, "\" not implemented for '", toString(t.scalar_type()), "'");
  }
  return -1;
}

void check_status(int st, const char* what) {
  TORCH_CHECK(st == FLN_OK, what, ": ", fln_status_string(st), " (status ", st, ")");
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
OptTensor opt(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

Tensor new_cuda(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& on_device_of) {
  return Tensor(at::detail::empty_cuda(sizes, dtype, on_device_of.device(), std::nullopt));
}
Tensor new_like(const Tensor& x) { return new_cuda(x.sizes(), x.scalar_type(), x); }

struct DeviceOf {
  std::optional<c10::cuda::CUDAGuard> guard;
  explicit DeviceOf(const Tensor& x) {
    if (c10::cuda::current_device() != x.device().index()) guard.emplace(x.device());
  }
};
void* stream_of(const Tensor& x) { return at::cuda::getCurrentCUDAStream(x.get_device()).stream(); }

void check_kind(int64_t kind) {
  TORCH_CHECK(kind == FLN_LAYERNORM || kind == FLN_RMSNORM || kind == FLN_NO_NORM,
              "norm must be 'layernorm', 'rmsnorm' or 'none'");
}
// same device and type as x
void check_beside(const Tensor& t, const Tensor& x, const char* name) {
  TORCH_CHECK(t.device().is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.device() == x.device(), name, " and input must be on the same device");
  TORCH_CHECK(t.scalar_type() == x.scalar_type(), name, " and input must have the same dtype");
}

// ---------------------------------------------------------------------------------------
// norm -> gate -> residual add -> norm
// ---------------------------------------------------------------------------------------
// how a parameter lies next to input [.., H]: one vector, one vector per entry of the first
// dimension, or an element each
enum class Spread { kVector, kGroup, kElement };
Spread spread_of(const Tensor& t, const Tensor& x, const char* name, bool allow_element) {
  const int64_t h = x.size(-1);
  TORCH_CHECK(t.dim() >= 1 && t.size(-1) == h, name, " size must match hidden dimension");
  if (t.numel() == h && (t.dim() == 1 || std::all_of(t.sizes().begin(), t.sizes().end() - 1, [](int64_t n) { return n == 1; })))
    return Spread::kVector;
  if (allow_element && t.sizes() == x.sizes()) return Spread::kElement;
  bool group = x.dim() >= 2 && t.dim() >= 2 && t.dim() <= x.dim() && t.size(0) == x.size(0);
  for (int64_t i = 1; group && i + 1 < t.dim(); ++i) group = t.size(i) == 1;
  TORCH_CHECK(group, name, " of shape ", t.sizes(), " does not fit input of shape ", x.sizes(),
              ": expected [hidden], [input.shape[0], hidden]", allow_element ? " or the shape of input" : "");
  return Spread::kGroup;
}

struct NgaConf {
  int64_t post_kind, kind, act;
  double ba, ra, woff, eps1, eps2;
};

// Validated, contiguous tensors of a call; `keep` owns what the argument block points to.
struct NgaCall {
  fln_nga_args a{};
  std::vector<Tensor> keep;
  Tensor x;
  const void* hold(const Tensor& t) {
    keep.push_back(t.contiguous());
    return keep.back().data_ptr();
  }
};
NgaCall nga_call(const Tensor& input, const OptTensor& residual, const OptTensor& gate, const OptTensor& w1,
                 const OptTensor& b1, const OptTensor& w2, const OptTensor& b2, const NgaConf& c) {
  NgaCall k;
  TORCH_CHECK(input.device().is_cuda(), "input must be a CUDA tensor");
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) > 0, "input must have a last dimension to normalize over");
  check_kind(c.post_kind);
  check_kind(c.kind);
  TORCH_CHECK(c.act >= FLN_GATE_ACT_NONE && c.act <= FLN_GATE_ACT_TANH,
              "gate_activation must be 'none', 'sigmoid', 'silu' or 'tanh'");
  k.a.dtype = dtype_code(input, "norm_gate_add_norm");
  k.x = input.contiguous();
  k.a.x = k.x.data_ptr();
  k.a.cols = input.size(-1);
  k.a.rows = input.numel() / k.a.cols;
  k.a.group_rows = input.dim() >= 2 && input.size(0) > 0 ? k.a.rows / input.size(0) : k.a.rows;
  if (k.a.group_rows == 0) k.a.group_rows = 1;
  k.a.post_kind = (int)c.post_kind;
  k.a.kind = (int)c.kind;
  k.a.gate_act = (int)c.act;
  k.a.branch_scale = (float)c.ba;
  k.a.residual_scale = (float)c.ra;
  k.a.weight_offset = (float)c.woff;
  k.a.post_eps = (float)c.eps1;
  k.a.eps = (float)c.eps2;
  if (has(residual)) {
    check_beside(*residual, input, "residual");
    TORCH_CHECK(residual->sizes() == input.sizes(), "residual shape must match input shape");
    k.a.residual = k.hold(*residual);
  }
  if (has(gate)) {
    check_beside(*gate, input, "gate");
    const Spread s = spread_of(*gate, input, "gate", true);
    k.a.gate_mode = s == Spread::kVector ? FLN_GATE_VECTOR : (s == Spread::kGroup ? FLN_GATE_GROUP : FLN_GATE_ELEMENT);
    k.a.gate = k.hold(*gate);
  }
  TORCH_CHECK(c.post_kind != FLN_NO_NORM || (!has(w1) && !has(b1)), "post_weight / post_bias without post_norm");
  TORCH_CHECK(c.kind != FLN_NO_NORM || (!has(w2) && !has(b2)), "weight / bias without norm");
  auto vec = [&](const OptTensor& t, const char* name) -> const void* {
    if (!has(t)) return nullptr;
    check_beside(*t, input, name);
    TORCH_CHECK(t->dim() == 1, name, " must be 1D");
    TORCH_CHECK(t->size(0) == k.a.cols, name, " size must match hidden dimension");
    return k.hold(*t);
  };
  k.a.post_weight = vec(w1, "post_weight");
  k.a.post_bias = vec(b1, "post_bias");
  int grouped = -1;
  auto affine = [&](const OptTensor& t, const char* name) -> const void* {
    if (!has(t)) return nullptr;
    check_beside(*t, input, name);
    const int g = spread_of(*t, input, name, false) == Spread::kGroup ? 1 : 0;
    TORCH_CHECK(grouped < 0 || grouped == g, "weight and bias must both be [hidden] or both [input.shape[0], hidden]");
    grouped = g;
    return k.hold(*t);
  };
  k.a.weight = affine(w2, "weight");
  k.a.bias = affine(b2, "bias");
  k.a.affine_grouped = grouped > 0 ? 1 : 0;
  return k;
}

struct NgaOut {
  Tensor y, sum, mean1, rstd1, mean2, rstd2;
};
NgaOut nga_forward(const Tensor& input, const OptTensor& residual, const OptTensor& gate, const OptTensor& w1,
                   const OptTensor& b1, const OptTensor& w2, const OptTensor& b2, const NgaConf& c, bool stats) {
  NgaCall k = nga_call(input, residual, gate, w1, b1, w2, b2, c);
  DeviceOf guard(input);
  NgaOut o;
  if (c.kind != FLN_NO_NORM) o.y = new_like(input);
  o.sum = new_like(input);
  auto stat = [&](bool want) { return want ? new_cuda({k.a.rows}, at::kFloat, input) : Tensor(); };
  auto p = [](const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; };
  o.mean1 = stat(stats && c.post_kind == FLN_LAYERNORM);
  o.rstd1 = stat(stats && c.post_kind != FLN_NO_NORM);
  o.mean2 = stat(stats && c.kind == FLN_LAYERNORM);
  o.rstd2 = stat(stats && c.kind != FLN_NO_NORM);
  check_status(fln_norm_gate_add_norm_forward(&k.a, o.y.defined() ? o.y.data_ptr() : nullptr, o.sum.data_ptr(),
                                              p(o.mean1), p(o.rstd1), p(o.mean2), p(o.rstd2), stream_of(input)),
               "norm_gate_add_norm");
  return o;
}

// which gradients: input, residual, gate, post_weight, post_bias, weight, bias
using NgaNeed = std::array<bool, 7>;
std::array<Tensor, 7> nga_backward(const OptTensor& dy_o, const OptTensor& dsum_o, const Tensor& input,
                                   const OptTensor& residual, const OptTensor& gate, const OptTensor& w1, const OptTensor& b1,
                                   const OptTensor& w2, const OptTensor& b2, const OptTensor& mean1,
                                   const OptTensor& rstd1, const OptTensor& mean2, const OptTensor& rstd2,
                                   const NgaConf& c, NgaNeed need) {
  NgaCall k = nga_call(input, residual, gate, w1, b1, w2, b2, c);
  DeviceOf guard(input);
  auto like = [&](const OptTensor& t, const char* name) -> const void* {
    if (!has(t)) return nullptr;
    check_beside(*t, input, name);
    TORCH_CHECK(t->sizes() == input.sizes(), name, " shape must match input shape");
    return k.hold(*t);
  };
  auto stat = [&](const OptTensor& t, const char* name) -> const float* {
    if (!has(t)) return nullptr;
    TORCH_CHECK(t->device() == input.device() && t->scalar_type() == at::kFloat && t->numel() == k.a.rows, name,
                " must be float32 with one entry per row, on the device of input");
    return reinterpret_cast<const float*>(k.hold(*t));
  };
  const void* dy = like(dy_o, "grad of y");
  const void* dsum = like(dsum_o, "grad of sum");
  if (!has(dy_o)) need[5] = need[6] = false;  // sum does not depend on weight and bias
  std::array<Tensor, 7> g;
  auto want = [&](int i, bool present, const OptTensor& t) {
    if (need[i] && present) g[i] = new_cuda(t->sizes(), input.scalar_type(), input);
  };
  want(0, true, input);
  want(1, true, input);  // (asked for only where there was one; without a second norm it is not kept)
  want(2, has(gate), gate);
  want(3, has(w1), w1);
  want(4, has(b1), b1);
  want(5, has(w2), w2);
  want(6, has(b2), b2);
  if (k.a.rows == 0) {  // sums over no rows
    for (Tensor& t : g)
      if (t.defined()) t.zero_();
    return g;
  }
  Tensor ws;
  size_t bytes = 0;
  const bool sums = (g[2].defined() && k.a.gate_mode != FLN_GATE_ELEMENT) || g[3].defined() || g[4].defined() ||
                    g[5].defined() || g[6].defined();
  if (sums) {
    bytes = fln_norm_gate_add_norm_workspace_bytes(&k.a);
    if (bytes > 0) ws = new_cuda({(int64_t)bytes}, at::kByte, input);
  }
  auto p = [](const Tensor& t) -> void* { return t.defined() ? t.data_ptr() : nullptr; };
  check_status(fln_norm_gate_add_norm_backward(&k.a, stat(mean1, "post_mean"), stat(rstd1, "post_rstd"),
                                               stat(mean2, "mean"), stat(rstd2, "rstd"), dy, dsum, p(g[0]), p(g[1]),
                                               p(g[2]), p(g[3]), p(g[4]), p(g[5]), p(g[6]), p(ws), bytes,
                                               stream_of(input)),
               "norm_gate_add_norm_backward");
  return g;
}

void refuse_double_backward(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " has no second derivative: call backward without create_graph=True");
}

// The autograd nodes are written against torch's Node directly: a node made by
// torch::autograd::Function keeps its constants in a dictionary and its tensors in lists, some
// 20 us per step on the host, more than the kernels take at small sizes.
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
SavedVariable saved(const OptTensor& t) { return has(t) ? SavedVariable(*t, false) : SavedVariable(); }
OptTensor unpacked(const SavedVariable& v) {
  Tensor t = v.unpack();
  return t.defined() ? OptTensor(t) : std::nullopt;
}
Tensor or_undefined(const OptTensor& t) { return has(t) ? *t : Tensor(); }
// (a dual tensor need not require grad, and no_grad leaves forward mode on: asked before anything else)
void refuse_forward_mode(std::initializer_list<const OptTensor*> ts, const char* what) {
  for (const OptTensor* t : ts)
    TORCH_CHECK(!has(*t) || !torch::autograd::isFwGradDefined(*t), what, " has no forward-mode derivative");
}
template <typename N>
std::shared_ptr<N> make_node(torch::autograd::edge_list&& edges) {
  auto n = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
  n->set_next_edges(std::move(edges));
  return n;
}

// gradients of input, residual, gate, post_weight, post_bias, weight, bias from those of (y, sum),
// or of (sum) when there is no second norm
struct NgaNode : public torch::autograd::Node {
  SavedVariable in[7], stat[4];
  NgaConf c{};
  std::string name() const override { return "NormGateAddNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& v : in) v.reset_data();
    for (auto& v : stat) v.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    refuse_double_backward("fused_norm_gate_add_norm");
    const Tensor dy = c.kind == FLN_NO_NORM ? Tensor() : grads[0];
    const Tensor ds = c.kind == FLN_NO_NORM ? grads[0] : grads[1];
    variable_list out(7);
    if (!dy.defined() && !ds.defined()) return out;
    NgaNeed need;
    for (size_t j = 0; j < 7; ++j) need[j] = task_should_compute_output(j);
    auto g = nga_backward(opt(dy), opt(ds), *unpacked(in[0]), unpacked(in[1]), unpacked(in[2]), unpacked(in[3]),
                          unpacked(in[4]), unpacked(in[5]), unpacked(in[6]), unpacked(stat[0]), unpacked(stat[1]),
                          unpacked(stat[2]), unpacked(stat[3]), c, need);
    for (size_t j = 0; j < 7; ++j) out[j] = g[j];
    return out;
  }
};

bool wants_grad(std::initializer_list<const OptTensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const OptTensor* t : ts)
    if (has(*t) && (*t)->requires_grad()) return true;
  return false;
}

// eager entry: (y or None, sum)
std::tuple<OptTensor, Tensor> norm_gate_add_norm(const Tensor& input, const OptTensor& residual, const OptTensor& gate,
                                                 const OptTensor& w1, const OptTensor& b1, const OptTensor& w2,
                                                 const OptTensor& b2, int64_t post_kind, int64_t kind, int64_t act,
                                                 double ba, double ra, double woff, double eps1, double eps2) {
  const OptTensor in = input;
  refuse_forward_mode({&in, &residual, &gate, &w1, &b1, &w2, &b2}, "fused_norm_gate_add_norm");
  if (!wants_grad({&in, &residual, &gate, &w1, &b1, &w2, &b2})) {
    NgaOut o = nga_forward(input, residual, gate, w1, b1, w2, b2, {post_kind, kind, act, ba, ra, woff, eps1, eps2}, false);
    return {opt(o.y), o.sum};
  }
  const NgaConf c{post_kind, kind, act, ba, ra, woff, eps1, eps2};
  NgaOut o;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    o = nga_forward(input, residual, gate, w1, b1, w2, b2, c, true);
  }
  auto n = make_node<NgaNode>(torch::autograd::collect_next_edges(input, or_undefined(residual), or_undefined(gate),
                                                                  or_undefined(w1), or_undefined(b1), or_undefined(w2),
                                                                  or_undefined(b2)));
  const OptTensor* ts[7] = {&in, &residual, &gate, &w1, &b1, &w2, &b2};
  for (int i = 0; i < 7; ++i)
    if (i != 1 || kind != FLN_NO_NORM) n->in[i] = saved(*ts[i]);
  const Tensor* st[4] = {&o.mean1, &o.rstd1, &o.mean2, &o.rstd2};
  for (int i = 0; i < 4; ++i) n->stat[i] = saved(opt(*st[i]));
  n->c = c;
  if (kind != FLN_NO_NORM) torch::autograd::set_history(o.y, n);
  torch::autograd::set_history(o.sum, n);
  return {opt(o.y), o.sum};
}

// operator forms (torch.compile): absent tensors are empty ones
Tensor or_empty(const Tensor& t, const Tensor& like) { return t.defined() ? t : new_cuda({0}, like.scalar_type(), like); }
Tensor or_empty_stat(const Tensor& t, const Tensor& like) { return t.defined() ? t : new_cuda({0}, at::kFloat, like); }
OptTensor none_if_empty(const Tensor& t, const Tensor& x) {
  return t.defined() && (t.numel() > 0 || x.numel() == 0) ? OptTensor(t) : std::nullopt;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> nga_fwd_op(
    const Tensor& input, const OptTensor& residual, const OptTensor& gate, const OptTensor& w1, const OptTensor& b1,
    const OptTensor& w2, const OptTensor& b2, int64_t post_kind, int64_t kind, int64_t act, double ba, double ra,
    double woff, double eps1, double eps2) {
  NgaOut o = nga_forward(input, residual, gate, w1, b1, w2, b2, {post_kind, kind, act, ba, ra, woff, eps1, eps2}, true);
  return {or_empty(o.y, input),          o.sum, or_empty_stat(o.mean1, input), or_empty_stat(o.rstd1, input),
          or_empty_stat(o.mean2, input), or_empty_stat(o.rstd2, input)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> nga_bwd_op(
    const OptTensor& dy, const OptTensor& dsum, const Tensor& input, const OptTensor& residual, const OptTensor& gate,
    const OptTensor& w1, const OptTensor& b1, const OptTensor& w2, const OptTensor& b2, const Tensor& mean1,
    const Tensor& rstd1, const Tensor& mean2, const Tensor& rstd2, int64_t post_kind, int64_t kind, int64_t act,
    double ba, double ra, double woff, double eps1, double eps2, std::array<bool, 7> need) {
  auto g = nga_backward(dy, dsum, input, residual, gate, w1, b1, w2, b2, none_if_empty(mean1, input),
                        none_if_empty(rstd1, input), none_if_empty(mean2, input), none_if_empty(rstd2, input),
                        {post_kind, kind, act, ba, ra, woff, eps1, eps2}, need);
  return {or_empty(g[0], input), or_empty(g[1], input), or_empty(g[2], input), or_empty(g[3], input),
          or_empty(g[4], input), or_empty(g[5], input), or_empty(g[6], input)};
}

// ---------------------------------------------------------------------------------------
// head norm -> rotary positions
// ---------------------------------------------------------------------------------------
struct RotConf {
  int64_t pairs, axes, layout, kind;
  double eps, woff, mag;
};

// One stride for dimensions [from, to) of t taken as one, or nothing if they do not fold.
std::optional<int64_t> fold(const Tensor& t, int64_t from, int64_t to) {
  int64_t stride = 0, next = -1;
  for (int64_t i = to - 1; i >= from; --i) {
    if (t.size(i) == 1) continue;
    if (next < 0) stride = t.stride(i);
    else if (t.stride(i) != next) return std::nullopt;
    next = t.stride(i) * t.size(i);
  }
  return stride;
}

// [.., heads, dim] seen as [batch, seq, heads, dim]: batch all leading dimensions but the last
struct Heads {
  Tensor keep;
  int64_t batch_s = 0, seq_s = 0, head_s = 0, heads = 0;
};
bool heads_view(const Tensor& t, Heads* h) {
  const int64_t nd = t.dim();
  if (t.numel() == 0) {  // nothing to step over
    h->keep = t;
    h->heads = t.size(nd - 2);
    return true;
  }
  if (t.size(-1) > 1 && t.stride(-1) != 1) return false;
  auto b = fold(t, 0, nd > 2 ? nd - 3 : 0);
  if (!b) return false;
  h->keep = t;
  h->batch_s = *b;
  h->seq_s = nd >= 3 ? t.stride(nd - 3) : 0;
  h->head_s = t.stride(nd - 2);
  h->heads = t.size(nd - 2);
  return true;
}
Heads heads_of(const Tensor& t) {
  Heads h;
  if (!heads_view(t, &h)) heads_view(t.contiguous(), &h);
  return h;
}

struct RotCall {
  fln_rotary_args a{};
  std::vector<Tensor> keep;
};

RotCall rot_call(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& turns, const Tensor& axis,
                 const std::array<OptTensor, 4>& wb, const RotConf& c) {
  RotCall r;
  TORCH_CHECK(q.device().is_cuda(), "q must be a CUDA tensor");
  TORCH_CHECK(q.dim() >= 2, "q must be [.., heads, head_dim]");
  check_kind(c.kind);
  r.a.dtype = dtype_code(q, "qk_norm_rotary");
  const int64_t nd = q.dim(), dim = q.size(-1);
  const auto lead = q.sizes().slice(0, nd - 2);
  if (has(k)) {
    check_beside(*k, q, "k");
    TORCH_CHECK(k->dim() == nd && k->size(-1) == dim && k->sizes().slice(0, nd - 2) == lead,
                "q and k must agree in all dimensions but the number of heads");
  }
  TORCH_CHECK(dim > 0 && c.pairs >= 0 && 2 * c.pairs <= dim, "the rotary plan rotates ", 2 * c.pairs,
              " elements, more than head_dim ", dim);
  TORCH_CHECK(dim <= 512, "head_dim must be at most 512");
  r.a.seq = nd >= 3 ? q.size(nd - 3) : 1;
  r.a.batch = 1;
  for (int64_t i = 0; i + 3 < nd; ++i) r.a.batch *= q.size(i);
  TORCH_CHECK(r.a.batch * r.a.seq <= 0x7fffffff, "too many tokens");
  r.a.head_dim = (int)dim;
  r.a.pairs = (int)c.pairs;
  r.a.layout = (int)c.layout;
  r.a.kind = (int)c.kind;
  r.a.eps = (float)c.eps;
  r.a.weight_offset = (float)c.woff;
  r.a.magnitude = (float)c.mag;
  TORCH_CHECK(positions.device() == q.device() && turns.device() == q.device() && axis.device() == q.device(),
              "positions, the rotary plan and q must be on the same device");
  TORCH_CHECK(positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt, "positions must be int32 or int64");
  TORCH_CHECK(turns.scalar_type() == at::kLong && axis.scalar_type() == at::kByte && turns.numel() == c.pairs &&
                  axis.numel() == c.pairs && turns.is_contiguous() && axis.is_contiguous(),
              "bad rotary plan");
  // [axes, *lead], [axes, last of lead] for all of the batch, or without the axes where there is one
  Tensor pos = positions;
  const bool plain = c.axes == 1 && (pos.sizes() == lead || (pos.dim() == 1 && lead.size() > 1 && pos.size(0) == lead.back()));
  if (plain) pos = pos.unsqueeze(0);
  TORCH_CHECK(pos.dim() >= 1 && pos.size(0) == c.axes, "positions must have ", c.axes, " axes in front, got shape ",
              positions.sizes());
  std::vector<int64_t> full{c.axes};
  full.insert(full.end(), lead.begin(), lead.end());
  if (pos.sizes() != at::IntArrayRef(full)) {
    TORCH_CHECK(pos.dim() == 2 && lead.size() > 1 && pos.size(1) == lead.back(), "positions of shape ", positions.sizes(),
                " do not fit tokens of shape ", lead);
    for (size_t i = 1; i < lead.size(); ++i) pos = pos.unsqueeze(1);
    pos = pos.expand(full);
  }
  const int64_t pd = pos.dim();
  auto pb = fold(pos, 1, pd > 1 ? pd - 1 : 1);
  if (!pb) {
    pos = pos.contiguous();
    pb = fold(pos, 1, pd > 1 ? pd - 1 : 1);
  }
  r.a.pos_axis = pos.stride(0);
  r.a.pos_batch = *pb;
  r.a.pos_seq = pd > 1 ? pos.stride(pd - 1) : 0;
  r.a.pos64 = pos.scalar_type() == at::kLong ? 1 : 0;
  r.a.positions = pos.data_ptr();
  r.keep.push_back(pos);
  r.a.turns = reinterpret_cast<const uint64_t*>(turns.data_ptr<int64_t>());
  r.a.axis = axis.data_ptr<uint8_t>();
  const char* names[4] = {"q_weight", "k_weight", "q_bias", "k_bias"};
  for (int i = 0; i < 4; ++i) {
    if (!has(wb[i])) continue;
    TORCH_CHECK(c.kind != FLN_NO_NORM, names[i], " without a norm");
    TORCH_CHECK(has(k) || (i & 1) == 0, names[i], " without k");
    check_beside(*wb[i], q, names[i]);
    TORCH_CHECK(wb[i]->dim() == 1 && wb[i]->size(0) == dim, names[i], " must be [head_dim]");
    r.keep.push_back(wb[i]->contiguous());
    (i < 2 ? r.a.t[i & 1].weight : r.a.t[i & 1].bias) = r.keep.back().data_ptr();
  }
  return r;
}

void set_in(fln_rotary_tensor& t, const Heads& h) {
  t.in = h.keep.data_ptr();
  t.in_batch = h.batch_s;
  t.in_seq = h.seq_s;
  t.in_head = h.head_s;
  t.heads = (int)h.heads;
}
void set_out(fln_rotary_tensor& t, const Heads& h) {
  t.out = h.keep.data_ptr();
  t.out_batch = h.batch_s;
  t.out_seq = h.seq_s;
  t.out_head = h.head_s;
}

// ---- what may be written in place ------------------------------------------------------
int64_t span(const Tensor& t, const std::vector<int64_t>& dims) {
  int64_t n = 1;
  for (int64_t d : dims) n += (t.size(d) - 1) * t.stride(d);
  return n;
}
// no element of t lies on another: sorted by stride, every dimension steps over all smaller ones
bool elements_apart(const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> d;
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1) d.emplace_back(t.stride(i), t.size(i));
  std::sort(d.begin(), d.end());
  int64_t covered = 1;
  for (auto& e : d) {
    if (e.first < covered) return false;
    covered = (e.second - 1) * e.first + covered;
  }
  return true;
}
// q and k hold no element in common: their ranges are apart, or become so when the outermost
// dimensions, which both step through alike, are taken off (views of one packed projection).  What
// is left of both together has to fit between two steps of every dimension that was taken off.
bool tensors_apart(const Tensor& q, const Tensor& k) {
  if (q.numel() == 0 || k.numel() == 0 || !q.is_alias_of(k)) return true;
  const int64_t off = k.storage_offset() - q.storage_offset();
  std::vector<int64_t> dims;
  for (int64_t i = 0; i < q.dim(); ++i) dims.push_back(i);
  int64_t window = INT64_MAX;  // the step of the dimension taken off last
  while (true) {
    const int64_t sq = span(q, dims), sk = span(k, dims);
    const int64_t lo = std::min<int64_t>(0, off), hi = std::max(sq, off + sk);
    if (hi - lo > window) return false;
    if (off >= sq || off + sk <= 0) return true;
    int64_t best = -1;
    for (int64_t d : dims)
      if (q.size(d) > 1 && (best < 0 || q.stride(d) > q.stride(best))) best = d;
    if (best < 0 || q.size(best) != k.size(best) || q.stride(best) != k.stride(best)) return false;
    window = q.stride(best);
    dims.erase(std::find(dims.begin(), dims.end(), best));
  }
}

void check_in_place(const Tensor& q, const OptTensor& k, Heads* views) {
  const Tensor* in[2] = {&q, has(k) ? &*k : nullptr};
  for (int i = 0; i < 2; ++i) {
    if (in[i] == nullptr) continue;
    TORCH_CHECK(in[i]->dim() >= 2, "q and k must be [.., heads, head_dim]");
    TORCH_CHECK(heads_view(*in[i], &views[i]) && elements_apart(*in[i]),
                "in place, q and k need a contiguous last dimension, leading dimensions that fold, and no element twice");
  }
  TORCH_CHECK(in[1] == nullptr || (k->dim() == q.dim() && tensors_apart(q, *k)), "in place, q and k must not overlap");
}

// (q', k'); k' undefined without k
std::pair<Tensor, Tensor> rot_forward(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& turns,
                                      const Tensor& axis, const std::array<OptTensor, 4>& wb, const RotConf& c, bool in_place) {
  RotCall r = rot_call(q, k, positions, turns, axis, wb, c);
  DeviceOf guard(q);
  Tensor out[2];
  const Tensor* in[2] = {&q, has(k) ? &*k : nullptr};
  Heads keep[4];
  if (in_place) check_in_place(q, k, keep);
  for (int i = 0; i < 2; ++i) {
    if (in[i] == nullptr) continue;
    if (!in_place) {
      keep[i] = heads_of(*in[i]);
      out[i] = new_like(*in[i]);
      keep[2 + i] = heads_of(out[i]);
    } else {
      out[i] = *in[i];
      keep[2 + i] = keep[i];
    }
    set_in(r.a.t[i], keep[i]);
    set_out(r.a.t[i], keep[2 + i]);
  }
  check_status(fln_qk_norm_rotary_forward(&r.a, stream_of(q)), "qk_norm_rotary");
  if (in_place)
    for (int i = 0; i < 2; ++i)
      if (in[i] != nullptr && !in[i]->is_inference()) torch::autograd::impl::bump_version(*in[i]);
  return {out[0], out[1]};
}

// gradients of q, k, q_weight, k_weight, q_bias, k_bias
std::array<Tensor, 6> rot_backward(const OptTensor& dq, const OptTensor& dk, const Tensor& q, const OptTensor& k,
                                   const Tensor& positions, const Tensor& turns, const Tensor& axis,
                                   const std::array<OptTensor, 4>& wb, const RotConf& c, const std::array<bool, 6>& need) {
  RotCall r = rot_call(q, k, positions, turns, axis, wb, c);
  DeviceOf guard(q);
  std::array<Tensor, 6> g;
  const Tensor* in[2] = {&q, has(k) ? &*k : nullptr};
  const OptTensor* go[2] = {&dq, &dk};
  Heads keep[4];
  void *dx[2] = {nullptr, nullptr}, *dw[2] = {nullptr, nullptr}, *db[2] = {nullptr, nullptr};
  bool sums = false;
  for (int i = 0; i < 2; ++i) {
    if (in[i] == nullptr || !has(*go[i])) continue;  // nothing arrives: no gradients for this tensor
    check_beside(**go[i], q, "grad");
    TORCH_CHECK((*go[i])->sizes() == in[i]->sizes(), "grad shape must match the input shape");
    keep[i] = heads_of(*in[i]);
    keep[2 + i] = heads_of(**go[i]);
    set_in(r.a.t[i], keep[i]);
    set_out(r.a.t[i], keep[2 + i]);
    if (need[i]) dx[i] = (g[i] = new_like(*in[i])).data_ptr();
    if (need[2 + i] && has(wb[i])) dw[i] = (g[2 + i] = new_like(*wb[i])).data_ptr();
    if (need[4 + i] && has(wb[2 + i])) db[i] = (g[4 + i] = new_like(*wb[2 + i])).data_ptr();
    sums = sums || dw[i] != nullptr || db[i] != nullptr;
  }
  Tensor ws;
  size_t bytes = 0;
  if (sums) {
    bytes = fln_qk_norm_rotary_workspace_bytes(&r.a);
    if (bytes > 0) ws = new_cuda({(int64_t)bytes}, at::kByte, q);
  }
  check_status(fln_qk_norm_rotary_backward(&r.a, dx, dw, db, ws.defined() ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
               "qk_norm_rotary_backward");
  return g;
}

// gradients of q, k, q_weight, k_weight, q_bias, k_bias
struct RotNode : public torch::autograd::Node {
  SavedVariable in[9];  // q, k, positions, turns, axis, weights, biases
  RotConf c{};
  std::string name() const override { return "QKNormRotaryBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& v : in) v.reset_data();
  }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    refuse_double_backward("fused_qk_norm_rotary");
    std::array<bool, 6> need;
    for (size_t j = 0; j < 6; ++j) need[j] = task_should_compute_output(j);
    auto g = rot_backward(opt(grads[0]), grads.size() > 1 ? opt(grads[1]) : std::nullopt, *unpacked(in[0]),
                          unpacked(in[1]), *unpacked(in[2]), *unpacked(in[3]), *unpacked(in[4]),
                          {unpacked(in[5]), unpacked(in[6]), unpacked(in[7]), unpacked(in[8])}, c, need);
    variable_list out(6);
    for (size_t j = 0; j < 6; ++j) out[j] = g[j];
    return out;
  }
};

std::tuple<Tensor, OptTensor> qk_norm_rotary(const Tensor& q, const OptTensor& k, const Tensor& positions,
                                             const Tensor& turns, const Tensor& axis, const OptTensor& qw,
                                             const OptTensor& kw, const OptTensor& qb, const OptTensor& kb, int64_t pairs,
                                             int64_t axes, int64_t layout, int64_t kind, double eps, double woff,
                                             double mag, bool in_place) {
  const OptTensor qo = q;
  refuse_forward_mode({&qo, &k, &qw, &kw, &qb, &kb}, "fused_qk_norm_rotary");
  const bool grad = wants_grad({&qo, &k, &qw, &kw, &qb, &kb});
  TORCH_CHECK(!(in_place && grad), "the in-place form records no gradient: use it under torch.no_grad()");
  if (!grad) {
    auto o = rot_forward(q, k, positions, turns, axis, {qw, kw, qb, kb}, {pairs, axes, layout, kind, eps, woff, mag}, in_place);
    return {o.first, opt(o.second)};
  }
  const RotConf c{pairs, axes, layout, kind, eps, woff, mag};
  std::pair<Tensor, Tensor> o;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    o = rot_forward(q, k, positions, turns, axis, {qw, kw, qb, kb}, c, false);
  }
  auto n = make_node<RotNode>(torch::autograd::collect_next_edges(q, or_undefined(k), or_undefined(qw), or_undefined(kw),
                                                                  or_undefined(qb), or_undefined(kb)));
  const OptTensor pos = positions, tu = turns, ax = axis;
  const OptTensor* ts[9] = {&qo, &k, &pos, &tu, &ax, &qw, &kw, &qb, &kb};
  for (int i = 0; i < 9; ++i) n->in[i] = saved(*ts[i]);
  n->c = c;
  torch::autograd::set_history(o.first, n);
  if (has(k)) torch::autograd::set_history(o.second, n);
  return {o.first, opt(o.second)};
}

std::tuple<Tensor, Tensor> rot_fwd_op(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& turns,
                                      const Tensor& axis, const OptTensor& qw, const OptTensor& kw, const OptTensor& qb,
                                      const OptTensor& kb, int64_t pairs, int64_t axes, int64_t layout, int64_t kind,
                                      double eps, double woff, double mag) {
  auto o = rot_forward(q, k, positions, turns, axis, {qw, kw, qb, kb}, {pairs, axes, layout, kind, eps, woff, mag}, false);
  return {o.first, or_empty(o.second, q)};
}
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> rot_bwd_op(
    const OptTensor& dq, const OptTensor& dk, const Tensor& q, const OptTensor& k, const Tensor& positions,
    const Tensor& turns, const Tensor& axis, const OptTensor& qw, const OptTensor& kw, const OptTensor& qb,
    const OptTensor& kb, int64_t pairs, int64_t axes, int64_t layout, int64_t kind, double eps, double woff, double mag,
    std::array<bool, 6> need) {
  auto g = rot_backward(dq, dk, q, k, positions, turns, axis, {qw, kw, qb, kb}, {pairs, axes, layout, kind, eps, woff, mag}, need);
  return {or_empty(g[0], q), or_empty(g[1], q), or_empty(g[2], q), or_empty(g[3], q), or_empty(g[4], q), or_empty(g[5], q)};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(fused_layernorm, m) {
  m.def("norm_gate_add_norm_fwd(Tensor input, Tensor? residual, Tensor? gate, Tensor? post_weight, Tensor? post_bias, Tensor? weight, Tensor? bias, int post_kind, int kind, int gate_act, float branch_scale, float residual_scale, float weight_offset, float post_eps, float eps) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("norm_gate_add_norm_bwd(Tensor? grad_y, Tensor? grad_sum, Tensor input, Tensor? residual, Tensor? gate, Tensor? post_weight, Tensor? post_bias, Tensor? weight, Tensor? bias, Tensor post_mean, Tensor post_rstd, Tensor mean, Tensor rstd, int post_kind, int kind, int gate_act, float branch_scale, float residual_scale, float weight_offset, float post_eps, float eps, bool[7] need) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("qk_norm_rotary_fwd(Tensor q, Tensor? k, Tensor positions, Tensor turns, Tensor axis, Tensor? q_weight, Tensor? k_weight, Tensor? q_bias, Tensor? k_bias, int pairs, int axes, int layout, int kind, float eps, float weight_offset, float magnitude) -> (Tensor, Tensor)");
  m.def("qk_norm_rotary_bwd(Tensor? grad_q, Tensor? grad_k, Tensor q, Tensor? k, Tensor positions, Tensor turns, Tensor axis, Tensor? q_weight, Tensor? k_weight, Tensor? q_bias, Tensor? k_bias, int pairs, int axes, int layout, int kind, float eps, float weight_offset, float magnitude, bool[6] need) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(fused_layernorm, CUDA, m) {
  m.impl("norm_gate_add_norm_fwd", &nga_fwd_op);
  m.impl("norm_gate_add_norm_bwd", &nga_bwd_op);
  m.impl("qk_norm_rotary_fwd", &rot_fwd_op);
  m.impl("qk_norm_rotary_bwd", &rot_bwd_op);
}

void fln_bind_blocks(pybind11::module& m) {
  namespace py = pybind11;
  m.def("norm_gate_add_norm", &norm_gate_add_norm,
        "(y or None, sum): norm -> gate -> residual add -> norm, recording one C++ autograd node where a gradient is "
        "wanted",
        py::arg("input"), py::arg("residual"), py::arg("gate"), py::arg("post_weight"), py::arg("post_bias"),
        py::arg("weight"), py::arg("bias"), py::arg("post_kind"), py::arg("kind"), py::arg("gate_act"),
        py::arg("branch_scale"), py::arg("residual_scale"), py::arg("weight_offset"), py::arg("post_eps"),
        py::arg("eps"));
  m.def("qk_norm_rotary", &qk_norm_rotary,
        "(q', k' or None): norm of every head, then the rotation of its position; in_place writes into q and k",
        py::arg("q"), py::arg("k"), py::arg("positions"), py::arg("turns"), py::arg("axis"), py::arg("q_weight"),
        py::arg("k_weight"), py::arg("q_bias"), py::arg("k_bias"), py::arg("pairs"), py::arg("axes"), py::arg("layout"),
        py::arg("kind"), py::arg("eps"), py::arg("weight_offset"), py::arg("magnitude"), py::arg("in_place"));
  m.def("check_rotary_in_place",
        [](const Tensor& q, const OptTensor& k) {
          Heads views[2];
          check_in_place(q, k, views);
        },
        "raises if qk_norm_rotary could not write over these q and k (of any device)", py::arg("q"), py::arg("k"));
}
