// Autograd nodes of the decoder-step operators for CUDA tensors whose parameters keep ordinary gradients.  A node in C++
// runs its backward in the engine's thread without entering Python (a forward and backward of small heads: 91 -> 70 us
// of one pass); parameters with a main_grad take the Python nodes of ops/functional.py, which know its hooks.
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

namespace emb {

at::Tensor heads_fwd(at::Tensor qkv, at::Tensor cosv, at::Tensor sinv, int64_t nq, int64_t nk, bool interleaved,
                     c10::optional<at::Tensor> wq, c10::optional<at::Tensor> wk, double eps);
std::vector<at::Tensor> heads_bwd(at::Tensor dy, c10::optional<at::Tensor> qkv, at::Tensor cosv, at::Tensor sinv,
                                  int64_t nq, int64_t nk, bool interleaved, c10::optional<at::Tensor> wq,
                                  c10::optional<at::Tensor> wk, double eps, c10::optional<at::Tensor> dwq_accum,
                                  c10::optional<at::Tensor> dwk_accum);
std::vector<at::Tensor> moe_route_fwd(at::Tensor logits, int64_t k, bool sigmoid, c10::optional<at::Tensor> bias,
                                      int64_t groups, int64_t topg, bool renorm, double scaling);
at::Tensor moe_route_bwd(at::Tensor logits, at::Tensor experts, c10::optional<at::Tensor> dweights,
                         c10::optional<at::Tensor> dscore, bool sigmoid, bool renorm, double scaling);
std::vector<at::Tensor> linear_ce_fwd(at::Tensor x, at::Tensor w, at::Tensor labels, int64_t col0, int64_t vocab,
                                      int64_t ignore, bool raw);
std::vector<at::Tensor> linear_ce_bwd(at::Tensor dloss, at::Tensor x, at::Tensor w, at::Tensor labels, at::Tensor top,
                                      at::Tensor sum, int64_t col0, int64_t vocab, int64_t ignore, bool want_dx,
                                      bool want_dw, c10::optional<at::Tensor> dw_accum, int64_t piece);

namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

bool tracks(const at::Tensor& t) { return t.defined() && t.requires_grad(); }
at::Tensor or_none(const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); }
OptTensor given(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

// The nodes have no forward-mode rule: an input with a tangent is refused, or its derivative would silently be zero.
template <typename... T>
void no_tangents(const T&... inputs) {
  for (const at::Tensor& t : {at::Tensor(inputs)...})
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(),
                                "this operator does not support forward-mode differentiation");
}

// A node whose inputs are `inputs`, in the order of the gradients that apply() returns.
template <typename N, typename... T>
std::shared_ptr<N> new_node(const T&... inputs) {
  auto n = std::shared_ptr<N>(new N(), torch::autograd::deleteNode);
  n->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return n;
}

struct HeadsNode : torch::autograd::Node {
  SavedVariable qkv, wq, wk, cosv, sinv;
  int64_t nq = 0, nk = 0;
  double eps = 0;
  bool interleaved = false;

  variable_list apply(variable_list&& dy) override {
    variable_list out(3);
    if (!dy[0].defined()) return out;
    at::NoGradGuard no_grad;
    auto self = getptr();
    const auto q = wq.unpack(self), k = wk.unpack(self);
    auto g = heads_bwd(dy[0], given(qkv.unpack(self)), cosv.unpack(self), sinv.unpack(self), nq, nk, interleaved, given(q),
                       given(k), eps, c10::nullopt, c10::nullopt);
    for (size_t i = 0; i < g.size(); ++i) out[i] = std::move(g[i]);
    return out;
  }
  void release_variables() override {
    for (auto* v : {&qkv, &wq, &wk, &cosv, &sinv}) v->reset_data();
  }
  std::string name() const override { return "HeadsBackward"; }
};

struct RouteNode : torch::autograd::Node {
  SavedVariable logits, experts;
  bool sigmoid = false, renorm = false;
  double scaling = 1;

  variable_list apply(variable_list&& d) override {  // of weights and score_sum
    variable_list out(1);
    if (!d[0].defined() && !d[1].defined()) return out;
    at::NoGradGuard no_grad;
    auto self = getptr();
    out[0] = moe_route_bwd(logits.unpack(self), experts.unpack(self), given(d[0]), given(d[1]), sigmoid, renorm, scaling);
    return out;
  }
  void release_variables() override {
    logits.reset_data();
    experts.reset_data();
  }
  std::string name() const override { return "MoERouteBackward"; }
};

struct LinearCeNode : torch::autograd::Node {
  SavedVariable x, w, labels, top, sum;
  int64_t ignore = 0, piece = 0;

  variable_list apply(variable_list&& d) override {
    variable_list out(2);
    if (!d[0].defined()) return out;
    at::NoGradGuard no_grad;
    auto self = getptr();
    const auto wv = w.unpack(self);
    auto g = linear_ce_bwd(d[0], x.unpack(self), wv, labels.unpack(self), top.unpack(self), sum.unpack(self), 0, wv.size(0),
                           ignore, should_compute_output(0), should_compute_output(1), c10::nullopt, piece);
    return {std::move(g[0]), std::move(g[1])};
  }
  void release_variables() override {
    for (auto* v : {&x, &w, &labels, &top, &sum}) v->reset_data();
  }
  std::string name() const override { return "LinearCrossEntropyBackward"; }
};

}  // namespace

at::Tensor heads(at::Tensor qkv, OptTensor wq, OptTensor wk, at::Tensor cosv, at::Tensor sinv, int64_t nq, int64_t nk,
                 double eps, bool interleaved) {
  const auto q = or_none(wq), k = or_none(wk);
  no_tangents(qkv, q, k, cosv, sinv);
  at::Tensor out;
  {
    at::NoGradGuard no_grad;
    out = heads_fwd(qkv, cosv, sinv, nq, nk, interleaved, wq, wk, eps);
  }
  if (at::GradMode::is_enabled() && (tracks(qkv) || tracks(q) || tracks(k))) {
    auto n = new_node<HeadsNode>(qkv, q, k);
    if (q.defined()) {  // the rotation alone needs no input for its gradient
      n->qkv = SavedVariable(qkv, false);
      n->wq = SavedVariable(q, false);
      n->wk = SavedVariable(k, false);
    }
    n->cosv = SavedVariable(cosv, false);
    n->sinv = SavedVariable(sinv, false);
    n->nq = nq;
    n->nk = nk;
    n->eps = eps;
    n->interleaved = interleaved;
    torch::autograd::set_history(out, n);
  }
  return out;
}

std::vector<at::Tensor> moe_route(at::Tensor logits, OptTensor bias, int64_t k, bool sigmoid, int64_t groups, int64_t topg,
                                  bool renorm, double scaling) {
  no_tangents(logits, or_none(bias));
  std::vector<at::Tensor> r;
  {
    at::NoGradGuard no_grad;
    r = moe_route_fwd(logits, k, sigmoid, bias, groups, topg, renorm, scaling);
  }
  if (at::GradMode::is_enabled() && tracks(logits)) {
    auto n = new_node<RouteNode>(logits);
    n->logits = SavedVariable(logits, false);
    n->experts = SavedVariable(r[1], false);
    n->sigmoid = sigmoid;
    n->renorm = renorm;
    n->scaling = scaling;
    torch::autograd::set_history(r[0], n);
    torch::autograd::set_history(r[2], n);
  }
  return r;
}

at::Tensor linear_ce(at::Tensor x, at::Tensor w, at::Tensor labels, int64_t ignore, int64_t piece) {
  no_tangents(x, w);
  std::vector<at::Tensor> r;
  {
    at::NoGradGuard no_grad;
    r = linear_ce_fwd(x, w, labels, 0, w.dim() == 2 ? w.size(0) : 0, ignore, false);
  }
  if (at::GradMode::is_enabled() && (tracks(x) || tracks(w))) {
    auto n = new_node<LinearCeNode>(x, w);
    n->x = SavedVariable(x, false);
    n->w = SavedVariable(w, false);
    n->labels = SavedVariable(labels, false);
    n->top = SavedVariable(r[1], false);
    n->sum = SavedVariable(r[2], false);
    n->ignore = ignore;
    n->piece = piece;
    torch::autograd::set_history(r[0], n);
  }
  return r[0];
}

}  // namespace emb
