// Autograd nodes of the batch-independent layers (group norm, client-keyed dropout, rotary positions): allocation, layout and
// launch in C++, both passes.  A backward pass in Python runs in the autograd engine's own thread, where the interpreter's
// objects come from the other core's cache: 40 to 90 us a layer on top of the kernels, against 5 here.
//
// Arguments are checked by the Python functions of ops/layers.py; this file sees fp32, bf16 or fp16 tensors of one GPU.  The
// kernels are reached through the addresses of their C entry points, which ops/_hip.py hands over: no second library.
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <cmath>
#include <memory>
#include <vector>

#include "layers_abi.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

// entry points of libblades_hip (see the sources for the arguments)
struct {
  decltype(&blades_group_norm_plan_size) gn_plan_size;
  decltype(&blades_group_norm_plan) gn_plan;
  decltype(&blades_group_norm_forward) gn_fwd;
  decltype(&blades_group_norm_backward) gn_bwd;
  decltype(&blades_client_dropout_plan_size) dropout_plan_size;
  decltype(&blades_client_dropout) dropout;
  decltype(&blades_rope_plan_size) rope_plan_size;
  decltype(&blades_rope_plan) rope_plan;
  decltype(&blades_rope_axes) rope;
} lib;

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2; }

// Gradients and what hooks unpack can be tensors without memory (wrapper subclasses, batches of gradients under a transform):
// those raise, in front of any launch.
void check_memory(const Tensor& t) {
  TORCH_CHECK(t.has_storage() && (t.numel() == 0 || t.data_ptr() != nullptr), "the batch-independent layers take tensors with "
              "memory of their own; their gradients are not batched");
}
void check_gradient(const Tensor& t) {
  check_memory(t);
  // (a tangent on a gradient asks for a second derivative)
  TORCH_CHECK(!t._fw_grad(0).defined(), "the batch-independent layers are differentiable once: their gradients take no tangent");
}
template <typename T = void> T* ptr(const Tensor& t) {
  if (!t.defined()) return nullptr;
  check_memory(t);
  return static_cast<T*>(t.data_ptr());
}

// Saved tensors can pass through hooks (moved to the host and back, say): the kernels rely on these.
void check_saved(const char* name, bool ok) {
  TORCH_CHECK(ok, name, ": a saved tensor came back with another shape, type or device");
}
bool like(const Tensor& t, const Tensor& r) {
  return !t.defined() || (t.sizes() == r.sizes() && t.scalar_type() == r.scalar_type() && t.device() == r.device());
}

// Outputs and workspaces pass through here: filled with NaN / 0xFF first where that is asked for (BLADES_POISON, see _hip.py).
bool poison = false;
Tensor fresh(Tensor t) {
  if (poison && t.numel() > 0) t.is_floating_point() ? t.fill_(NAN) : t.fill_(0xFF);
  return t;
}

bool needs_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }

bool channels_last(const Tensor& t) {
  if (t.dim() == 4) return t.is_contiguous(at::MemoryFormat::ChannelsLast);
  return t.dim() == 2 ? t.is_contiguous() : t.movedim(1, -1).is_contiguous();
}
Tensor to_channels_last(const Tensor& t) {
  return !t.defined() || channels_last(t) ? t : t.movedim(1, -1).contiguous().movedim(-1, 1);
}
Tensor like_channels_last(const Tensor& x) {
  Tensor y = at::empty_like(x);
  if (channels_last(y)) return fresh(y);
  std::vector<int64_t> s{x.size(0)};
  for (int64_t i = 2; i < x.dim(); ++i) s.push_back(x.size(i));
  s.push_back(x.size(1));
  return fresh(at::empty(s, x.options())).movedim(-1, 1);
}

// A graph of a backward pass is only built to differentiate it again: its results then raise when that happens.
variable_list first_order(variable_list&& grads) {
  if (!at::GradMode::is_enabled()) return std::move(grads);
  const auto n = static_cast<int64_t>(grads.size());
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "the batch-independent layers are differentiable once", n);
  return (*node)(std::move(grads));
}

// ---------------------------------------------------------------------------------------------------------------
struct GroupNorm {
  std::vector<char> plan;
  long ws[2], strides[2];  // (of the weight and the bias, client to client)
  int vec, groups, act;
  long clients;
  float eps;

  groupnorm::Layer* layer() { return reinterpret_cast<groupnorm::Layer*>(plan.data()); }
  static long stride(const Tensor& t) { return t.defined() && t.dim() == 2 ? t.stride(0) : 0; }
  bool affine_fits(const Tensor& t, const Tensor& x, long C) const {
    return !t.defined() || (t.scalar_type() == at::kFloat && t.device() == x.device() && t.dim() > 0 && t.size(-1) == C &&
                            (t.dim() == 1 || (t.dim() == 2 && t.size(0) == clients)));
  }

  void make(const Tensor& x, const Tensor& w, const Tensor& b, int v) {
    const long N = x.size(0), C = x.size(1), P = x.numel() / (N * C);
    plan.resize(lib.gn_plan_size());
    strides[0] = stride(w); strides[1] = stride(b);
    auto fill = [&](int channels) {
      vec = channels;
      return lib.gn_plan(layer(), N, P, (int)C, groups, eps, act, (int)(N / clients), strides[0], strides[1], dtype_of(x),
                         vec, ws);
    };
    int rc = C > (1 << 24) ? 1 : fill(v);  // (the plan's counts are ints)
    if (rc == 2 && v > 1) rc = fill(1);  // wide groups of an odd number of channels
    if (rc != 0)
      throw py::value_error("group_norm: " + std::to_string(N) + " samples of " + std::to_string(C) + " channels in " +
                            std::to_string(groups) + " groups over " + std::to_string(P) + " pixels are not supported (fewer "
                            "than 2^24 samples, at most 2^24 channels, fewer than 2^30 pixels; a group has at most 2048 "
                            "channels, 1024 where C or an address rules out accesses of four)");
  }
};

bool aligned(const Tensor& a, const Tensor& b, const Tensor& c) {
  return ((reinterpret_cast<uintptr_t>(ptr(a)) | reinterpret_cast<uintptr_t>(ptr(b)) | reinterpret_cast<uintptr_t>(ptr(c))) &
          15) == 0;
}

Tensor affine(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor f = t.scalar_type() == at::kFloat ? t : t.to(at::kFloat);
  return f.stride(-1) == 1 ? f : f.contiguous();
}

struct GroupNormBackward : Node {
  SavedVariable x, w, b, stats, res, gate;
  std::shared_ptr<GroupNorm> g;
  bool has_w, has_b, has_res;
  at::ScalarType w_type, b_type;

  variable_list apply(variable_list&& grads) override;
  std::string name() const override { return "GroupNormBackward"; }
  void release_variables() override {
    for (SavedVariable* s : {&x, &w, &b, &stats, &res, &gate}) s->reset_data();
  }
};

variable_list GroupNormBackward::apply(variable_list&& grads) {
  variable_list out(4);
  Tensor gy = std::move(grads[0]);
  if (!gy.defined()) return out;
  check_gradient(gy);
  const bool nx = task_should_compute_output(0), nw = has_w && task_should_compute_output(1),
             nb = has_b && task_should_compute_output(2), nr = has_res && task_should_compute_output(3);
  {
    at::NoGradGuard no_grad;
    const auto self = shared_from_this();
    Tensor x_ = x.unpack(self), r_ = res.unpack(self), w_ = w.unpack(self), b_ = b.unpack(self);
    Tensor st = stats.unpack(self), gt = gate.unpack(self);
    std::shared_ptr<GroupNorm> p = g;
    const int64_t C = gy.size(1);
    check_saved("group_norm", like(x_, gy) && like(r_, gy) && p->affine_fits(w_, gy, C) && p->affine_fits(b_, gy, C) &&
                st.scalar_type() == at::kFloat && st.device() == gy.device() && st.numel() == 2 * gy.size(0) * p->groups &&
                (!gt.defined() || (gt.scalar_type() == at::kByte && gt.device() == gy.device() &&
                                   gt.numel() * p->vec == gy.numel())));
    Tensor g_ = to_channels_last(gy);
    x_ = to_channels_last(x_); r_ = to_channels_last(r_);
    w_ = affine(w_); b_ = affine(b_); st = st.contiguous();
    if (gt.defined()) gt = gt.contiguous();
    const c10::DeviceGuard guard(x_.device());
    if (GroupNorm::stride(w_) != p->strides[0] || GroupNorm::stride(b_) != p->strides[1]) {
      p = std::make_shared<GroupNorm>(*g);
      p->make(x_, w_, b_, g->vec);
    }
    if (p->vec > 1)
      for (Tensor* t : {&x_, &g_, &r_})
        if (!aligned(*t, Tensor(), Tensor())) *t = t->clone(at::MemoryFormat::Preserve);
    const auto f32 = x_.options().dtype(at::kFloat);
    const bool own_dres = nr && p->act != 0;
    if (nx) out[0] = like_channels_last(x_);
    if (nw) out[1] = fresh(at::empty(w_.sizes(), f32));
    if (nb) out[2] = fresh(at::empty(b_.sizes(), f32));
    if (own_dres) out[3] = like_channels_last(x_);
    Tensor ws = fresh(at::empty({p->ws[1]}, x_.options().dtype(at::kByte)));
    lib.gn_bwd(ptr(x_), ptr(r_), ptr(g_), ptr(gt), ptr<float>(w_), ptr<float>(b_), ptr<float>(st), ptr(out[0]), ptr(out[3]),
               nullptr, ptr<float>(out[1]), ptr<float>(out[2]), x_.size(1), 0, ptr<float>(ws), p->layer(), stream_of(x_));
    if (nr && !own_dres) out[3] = gy;
    if (nw && w_type != at::kFloat) out[1] = out[1].to(w_type);
    if (nb && b_type != at::kFloat) out[2] = out[2].to(b_type);
  }
  return first_order(std::move(out));
}

Tensor group_norm(const Tensor& x, int64_t groups, const MaybeTensor& weight, const MaybeTensor& bias, double eps, int64_t act,
                  const MaybeTensor& residual) {
  const Tensor none, &wt = weight ? *weight : none, &bs = bias ? *bias : none, &rs = residual ? *residual : none;
  const bool grad =
      at::GradMode::is_enabled() && (needs_grad(x) || needs_grad(wt) || needs_grad(bs) || needs_grad(rs));
  auto g = std::make_shared<GroupNorm>();
  g->groups = (int)groups; g->act = (int)act; g->eps = (float)eps;
  g->clients = wt.defined() && wt.dim() == 2 ? wt.size(0) : bs.defined() && bs.dim() == 2 ? bs.size(0) : 1;
  Tensor y, x_, w_, b_, r_, stats, gate;
  {
    at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(x.device());
    x_ = to_channels_last(x); r_ = to_channels_last(rs);
    w_ = affine(wt); b_ = affine(bs);
    g->make(x_, w_, b_, x_.size(1) % 4 == 0 && aligned(x_, r_, none) ? 4 : 1);
    y = like_channels_last(x_);
    if (grad || g->ws[0]) stats = fresh(at::empty({2, x_.size(0), groups}, x_.options().dtype(at::kFloat)));
    if (grad && r_.defined() && act == 1) gate = fresh(at::empty({x_.numel() / g->vec}, x_.options().dtype(at::kByte)));
    Tensor ws;
    if (g->ws[0]) ws = fresh(at::empty({g->ws[0]}, x_.options().dtype(at::kByte)));
    lib.gn_fwd(ptr(x_), ptr(r_), ptr<float>(w_), ptr<float>(b_), ptr(y), ptr(gate), ptr<float>(stats), ptr<float>(ws),
               g->layer(), stream_of(x_));
  }
  if (!grad) return y;
  auto node = std::shared_ptr<GroupNormBackward>(new GroupNormBackward(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(x, wt, bs, rs));
  node->x = SavedVariable(x_, false); node->w = SavedVariable(w_, false); node->b = SavedVariable(b_, false);
  node->stats = SavedVariable(stats, false); node->gate = SavedVariable(gate, false);
  if (act >= 2) node->res = SavedVariable(r_, false);  // (a ReLU's gate stands in for the residual)
  node->g = g;
  node->has_w = wt.defined(); node->has_b = bs.defined(); node->has_res = rs.defined();
  if (wt.defined()) node->w_type = wt.scalar_type();
  if (bs.defined()) node->b_type = bs.scalar_type();
  torch::autograd::set_history(y, node);
  return y;
}

// ---------------------------------------------------------------------------------------------------------------
Tensor drop(const Tensor& t, const Tensor& uids, const Tensor& tag, long tag_value, DropPlan p) {
  check_saved("client_dropout", uids.numel() == p.Kc && uids.scalar_type() == at::kLong && uids.device() == t.device() &&
              uids.is_contiguous() && (!tag.defined() || (tag.numel() == 1 && tag.scalar_type() == at::kLong &&
              tag.device() == t.device())));
  const c10::DeviceGuard guard(t.device());
  Tensor x = t;
  p.last = 0;
  if (!x.is_contiguous()) {
    p.last = x.dim() == 4 && x.is_contiguous(at::MemoryFormat::ChannelsLast);
    if (!p.last) x = x.contiguous();
  }
  Tensor y = fresh(at::empty_like(x));
  const int rc = lib.dropout(ptr(x), ptr(y), ptr<long>(uids), ptr<long>(tag), tag_value, &p, stream_of(x));
  if (rc != 0)
    throw py::value_error("client_dropout: rejected: a client's share of a layer has at most 1.7e10 elements (and at most 2^30 "
                          "samples, channels and pixels where draws are shared or maps are channels last)");
  return y;
}

struct ClientDropoutBackward : Node {
  // the ids and the tag are saved, so that changing them between the two passes raises instead of drawing another mask
  SavedVariable uids, tag;
  long tag_value;
  DropPlan p;

  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    if (!grads[0].defined()) return out;
    check_gradient(grads[0]);
    {
      at::NoGradGuard no_grad;
      out[0] = drop(grads[0], uids.unpack(shared_from_this()), tag.unpack(shared_from_this()), tag_value, p);
    }
    return first_order(std::move(out));
  }
  std::string name() const override { return "ClientDropoutBackward"; }
  void release_variables() override {
    uids.reset_data(); tag.reset_data();
  }
};

Tensor client_dropout(const Tensor& x, const Tensor& uids, const MaybeTensor& tag, int64_t tag_value, uint64_t seed,
                      uint64_t c3, uint64_t least, double scale, int64_t kind, bool inner) {
  const long K = uids.numel();
  DropPlan p{};
  p.Kc = (int)K; p.seed = seed; p.c3 = (unsigned)c3; p.least = (unsigned)least; p.scale = (float)scale;
  p.kind = (int)kind; p.inner = inner; p.dtype = dtype_of(x);
  p.B = inner ? x.size(0) : x.size(0) / K;
  p.C = inner ? x.size(1) / K : x.dim() > 1 ? x.size(1) : 1;
  p.HW = x.numel() / (K * p.B * p.C);
  const Tensor tg = tag ? *tag : Tensor();
  Tensor y;
  {
    at::NoGradGuard no_grad;
    y = drop(x, uids, tg, tag_value, p);
  }
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    auto node = std::shared_ptr<ClientDropoutBackward>(new ClientDropoutBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->uids = SavedVariable(uids, false); node->tag = SavedVariable(tg, false);
    node->tag_value = tag_value; node->p = p;
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---------------------------------------------------------------------------------------------------------------
struct Rope {
  std::vector<int> axes;
  double base;
  int slots;
};

// The launch plan of a shape: a few thousand words of frequencies, so the last ones are kept by their sizes.
struct RopeKey {
  std::vector<int64_t> v;
  double base;
  bool operator==(const RopeKey& o) const { return base == o.base && v == o.v; }
};
std::shared_ptr<std::vector<char>> rope_plan(const Tensor& x, const Tensor& pos, const Rope& r, int vec) {
  static thread_local std::vector<std::pair<RopeKey, std::shared_ptr<std::vector<char>>>> kept;
  const bool five = x.dim() == 5;
  const long R = x.size(0), N = x.size(1), psr = pos.dim() == 3 ? N * (long)r.axes.size() : 0;
  if ((double)x.size(-2) * (five ? x.size(2) : 1) > 1e9)  // (the plan's counts are ints)
    throw py::value_error("rope_axes: a token has at most 10^9 rows (slots times heads)");
  const int S = five ? (int)x.size(2) : 1, H = (int)x.size(-2), D = (int)x.size(-1), dt = dtype_of(x);
  const int pf = pos.scalar_type() == at::kFloat;
  RopeKey key{{pf, psr, R, N, S, H, D, x.stride(0), x.stride(1), five ? x.stride(2) : 0, x.stride(-2), r.slots, dt, vec}, r.base};
  for (int a : r.axes) key.v.push_back(a);
  for (auto& k : kept)
    if (k.first == key) return k.second;
  auto plan = std::make_shared<std::vector<char>>(lib.rope_plan_size());
  const int rc = lib.rope_plan(reinterpret_cast<rope::RopePlan*>(plan->data()), pf, psr, R, N, S, H, D, x.stride(0),
                               x.stride(1), five ? x.stride(2) : 0, x.stride(-2), r.slots, r.axes.data(), (int)r.axes.size(), r.base, dt, vec);
  if (rc != 0) throw py::value_error("rope_axes: rejected (rc=" + std::to_string(rc) + ")");
  if (kept.size() >= 16) kept.erase(kept.begin());
  kept.emplace_back(std::move(key), plan);
  return plan;
}

Tensor turn(const Tensor& t, const Tensor& pos, const Rope& r, int inverse) {
  const c10::DeviceGuard guard(t.device());
  if (t.numel() == 0) return fresh(at::empty(t.sizes(), t.options()));
  check_saved("rope_axes", (pos.scalar_type() == at::kFloat || pos.scalar_type() == at::kLong) && pos.device() == t.device() &&
              (pos.dim() == 2 || (pos.dim() == 3 && pos.size(0) == t.size(0))) && pos.size(-2) == t.size(1) &&
              pos.size(-1) == (int64_t)r.axes.size());
  Tensor x = t.stride(-1) == 1 ? t : t.contiguous();
  const Tensor p = pos.contiguous();
  const int w = x.scalar_type() == at::kFloat ? 4 : 8;
  auto step = [&] { return x.stride(0) | x.stride(1) | x.stride(2) | x.stride(-2); };
  const auto at_ = [&] { return reinterpret_cast<uintptr_t>(ptr(x)); };
  int vec = w;
  if (at_() % 16 || step() % w || x.size(-1) % w) {
    if (step() % 2 || at_() % (2 * x.element_size())) x = x.clone(at::MemoryFormat::Contiguous);
    vec = at_() % 16 || step() % w || x.size(-1) % w ? 2 : w;
  }
  const auto plan = rope_plan(x, p, r, vec);
  Tensor y = fresh(at::empty(x.sizes(), x.options()));
  const int rc = lib.rope(ptr(x), ptr(y), ptr(p), reinterpret_cast<rope::RopePlan*>(plan->data()), inverse, stream_of(x));
  if (rc != 0) throw py::value_error("rope_axes: rejected (rc=" + std::to_string(rc) + ")");
  return y;
}

struct RopeBackward : Node {
  SavedVariable pos;
  Rope r;

  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    if (!grads[0].defined()) return out;
    check_gradient(grads[0]);
    {
      at::NoGradGuard no_grad;
      out[0] = turn(grads[0], pos.unpack(shared_from_this()), r, 1);
    }
    return first_order(std::move(out));
  }
  std::string name() const override { return "RopeBackward"; }
  void release_variables() override {
    pos.reset_data();
  }
};

Tensor rope_axes(const Tensor& x, const Tensor& pos, const std::vector<int>& axes, double base, int64_t slots) {
  Rope r{axes, base, (int)slots};
  Tensor y;
  {
    at::NoGradGuard no_grad;
    y = turn(x, pos, r, 0);
  }
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    auto node = std::shared_ptr<RopeBackward>(new RopeBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->pos = SavedVariable(pos, false);
    node->r = std::move(r);
    torch::autograd::set_history(y, node);
  }
  return y;
}

void entries(const std::vector<uintptr_t>& a) {
  TORCH_CHECK(a.size() == 9, "nine entry points are expected");
  TORCH_CHECK(reinterpret_cast<decltype(lib.dropout_plan_size)>(a[4])() == (long)sizeof(DropPlan),
              "the kernels' library is of another build: build again");
  void* to[] = {&lib.gn_plan_size, &lib.gn_plan, &lib.gn_fwd, &lib.gn_bwd, &lib.dropout_plan_size, &lib.dropout,
                &lib.rope_plan_size, &lib.rope_plan, &lib.rope};
  for (size_t i = 0; i < a.size(); ++i) *static_cast<uintptr_t*>(to[i]) = a[i];
}

}  // namespace

PYBIND11_MODULE(_autograd, m) {
  m.def("entries", &entries);
  m.def("poison", [](bool on) { poison = on; });
  m.def("group_norm", &group_norm);
  m.def("client_dropout", &client_dropout);
  m.def("rope_axes", &rope_axes);
}
