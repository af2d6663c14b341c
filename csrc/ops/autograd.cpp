// Autograd nodes of the decoder-step operators for CUDA tensors whose parameters keep ordinary gradients.  A node in C++
// runs its backward in the engine's thread without entering Python (a forward and backward of small heads: 91 -> 75 us
// of one pass); parameters with a main_grad take the Python nodes of ops/functional.py, which know its hooks.
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

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = c10::optional<at::Tensor>;

OptTensor given(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct HeadsNode : torch::autograd::Function<HeadsNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& qkv, const OptTensor& wq, const OptTensor& wk,
                            const at::Tensor& cosv, const at::Tensor& sinv, int64_t nq, int64_t nk, double eps,
                            bool interleaved) {
    auto out = heads_fwd(qkv, cosv, sinv, nq, nk, interleaved, wq, wk, eps);
    const bool norm = wq.has_value();
    ctx->save_for_backward({norm ? qkv : at::Tensor(), norm ? *wq : at::Tensor(), norm ? *wk : at::Tensor(), cosv, sinv});
    ctx->saved_data["nq"] = nq;
    ctx->saved_data["nk"] = nk;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["inter"] = interleaved;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto v = ctx->get_saved_variables();
    auto g = heads_bwd(dy[0], given(v[0]), v[3], v[4], ctx->saved_data["nq"].toInt(), ctx->saved_data["nk"].toInt(),
                       ctx->saved_data["inter"].toBool(), given(v[1]), given(v[2]), ctx->saved_data["eps"].toDouble(),
                       c10::nullopt, c10::nullopt);
    variable_list out(9);
    for (size_t i = 0; i < g.size(); ++i) out[i] = g[i];
    return out;
  }
};

struct RouteNode : torch::autograd::Function<RouteNode> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const OptTensor& bias, int64_t k,
                               bool sigmoid, int64_t groups, int64_t topg, bool renorm, double scaling) {
    auto r = moe_route_fwd(logits, k, sigmoid, bias, groups, topg, renorm, scaling);
    ctx->save_for_backward({logits, r[1]});
    ctx->saved_data["sigmoid"] = sigmoid;
    ctx->saved_data["renorm"] = renorm;
    ctx->saved_data["scaling"] = scaling;
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r[1], r[3]});
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto v = ctx->get_saved_variables();
    variable_list out(8);
    if (d[0].defined() || d[2].defined())
      out[0] = moe_route_bwd(v[0], v[1], given(d[0]), given(d[2]), ctx->saved_data["sigmoid"].toBool(),
                             ctx->saved_data["renorm"].toBool(), ctx->saved_data["scaling"].toDouble());
    return out;
  }
};

struct LinearCeNode : torch::autograd::Function<LinearCeNode> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& labels,
                            int64_t ignore, int64_t piece) {
    auto r = linear_ce_fwd(x, w, labels, 0, w.size(0), ignore, false);
    ctx->save_for_backward({x, w, labels, r[1], r[2]});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["piece"] = piece;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list d) {
    const auto v = ctx->get_saved_variables();
    auto g = linear_ce_bwd(d[0], v[0], v[1], v[2], v[3], v[4], 0, v[1].size(0), ctx->saved_data["ignore"].toInt(),
                           ctx->needs_input_grad(0), ctx->needs_input_grad(1), c10::nullopt,
                           ctx->saved_data["piece"].toInt());
    return {g[0], g[1], at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

at::Tensor heads(at::Tensor qkv, OptTensor wq, OptTensor wk, at::Tensor cosv, at::Tensor sinv, int64_t nq, int64_t nk,
                 double eps, bool interleaved) {
  return HeadsNode::apply(qkv, wq, wk, cosv, sinv, nq, nk, eps, interleaved);
}

std::vector<at::Tensor> moe_route(at::Tensor logits, OptTensor bias, int64_t k, bool sigmoid, int64_t groups, int64_t topg,
                                  bool renorm, double scaling) {
  return RouteNode::apply(logits, bias, k, sigmoid, groups, topg, renorm, scaling);
}

at::Tensor linear_ce(at::Tensor x, at::Tensor w, at::Tensor labels, int64_t ignore, int64_t piece) {
  return LinearCeNode::apply(x, w, labels, ignore, piece);
}

}  // namespace emb
