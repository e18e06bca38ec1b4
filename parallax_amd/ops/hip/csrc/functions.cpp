// Differentiable forms of linear_ce and rotary.  Their small calls take the
// GPU less time than the interpreter, whose lock a backward in Python also
// hands between the threads of the autograd engine (16 rows x 2,000 words,
// forward and backward: 118 us in Python, 102 us so).

#include <torch/extension.h>

#include <vector>

std::vector<at::Tensor> linear_ce_fwd(const at::Tensor& x,
                                      const at::Tensor& w,
                                      const c10::optional<at::Tensor>& bias,
                                      const at::Tensor& labels,
                                      int64_t ignore, double smoothing,
                                      int64_t reduction);
std::vector<at::Tensor> linear_ce_bwd(
    const at::Tensor& dloss, const at::Tensor& x, const at::Tensor& w,
    const c10::optional<at::Tensor>& bias, const at::Tensor& labels,
    const at::Tensor& saved, int64_t ignore, double smoothing,
    int64_t reduction, bool want_dx, bool want_dw, bool want_db);
std::vector<at::Tensor> rotary(const at::Tensor& q,
                               const c10::optional<at::Tensor>& k,
                               const at::Tensor& cos, const at::Tensor& sin,
                               const c10::optional<at::Tensor>& positions,
                               int64_t offset, bool interleaved, bool back);

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::tensor_list;

using Maybe = c10::optional<at::Tensor>;

Maybe maybe(const at::Tensor& t) { return t.defined() ? Maybe(t) : Maybe(); }

// An argument of a Function is never undefined: what is missing is passed
// as a tensor without gradient, and stands as undefined behind it.
at::Tensor or_other(const Maybe& t, const at::Tensor& other) {
  return t.has_value() ? *t : other;
}

// Passes `t` on; whoever differentiates it again gets an error, not zeros.
struct Once : public Function<Once> {
  static at::Tensor forward(AutogradContext*, const at::Tensor& t,
                            const at::Tensor&, const at::Tensor&,
                            const at::Tensor&) {
    return t.view_as(t);
  }
  static tensor_list backward(AutogradContext*, tensor_list) {
    TORCH_CHECK(false, "this gradient can not be differentiated again");
  }
};

at::Tensor once(const at::Tensor& t, const at::Tensor& a, const at::Tensor& b,
                const at::Tensor& c) {
  if (!t.defined() || !at::GradMode::is_enabled()) return t;
  return Once::apply(t, a, b, c);
}

struct LinearCE : public Function<LinearCE> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x,
                            const at::Tensor& w, const at::Tensor& bias,
                            const at::Tensor& labels, bool has_bias,
                            int64_t ignore, double smoothing,
                            int64_t reduction) {
    const at::Tensor b = has_bias ? bias : at::Tensor();
    auto r = linear_ce_fwd(x, w, maybe(b), labels, ignore, smoothing,
                           reduction);
    ctx->save_for_backward({x, w, b, labels, r[1]});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["smoothing"] = smoothing;
    ctx->saved_data["reduction"] = reduction;
    return r[0];
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list res(8);
    const auto s = ctx->get_saved_variables();
    const bool dx = ctx->needs_input_grad(0), dw = ctx->needs_input_grad(1);
    const bool db = s[2].defined() && ctx->needs_input_grad(2);
    if (!grads[0].defined() || !(dx || dw || db)) return res;
    std::vector<at::Tensor> r;
    {
      at::NoGradGuard no;
      r = linear_ce_bwd(grads[0].contiguous(), s[0], s[1], maybe(s[2]), s[3],
                        s[4], ctx->saved_data["ignore"].toInt(),
                        ctx->saved_data["smoothing"].toDouble(),
                        ctx->saved_data["reduction"].toInt(), dx, dw, db);
    }
    const at::Tensor other = dx ? s[0] : dw ? s[1] : s[2];
    for (int i = 0; i < 3; ++i)
      res[i] = once(r[i], other, grads[0], other);
    return res;
  }
};

struct Rotary : public Function<Rotary> {
  static tensor_list forward(AutogradContext* ctx, const at::Tensor& q,
                             const at::Tensor& k, const at::Tensor& cos,
                             const at::Tensor& sin,
                             const at::Tensor& positions, bool has_k,
                             bool has_positions, int64_t offset,
                             bool interleaved) {
    const at::Tensor at = has_positions ? positions : at::Tensor();
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({cos, sin, at});
    ctx->saved_data["offset"] = offset;
    ctx->saved_data["interleaved"] = interleaved;
    return rotary(q, has_k ? Maybe(k) : Maybe(), cos, sin, maybe(at), offset,
                  interleaved, false);
  }

  static tensor_list backward(AutogradContext* ctx, tensor_list grads) {
    tensor_list res(9);
    const auto s = ctx->get_saved_variables();
    std::vector<int> which;
    tensor_list live;
    for (int i = 0; i < (int)grads.size(); ++i) {
      if (!grads[i].defined() || !ctx->needs_input_grad(i)) continue;
      which.push_back(i);
      live.push_back(grads[i].stride(3) == 1 ? grads[i]
                                             : grads[i].contiguous());
    }
    if (live.empty()) return res;
    std::vector<at::Tensor> r;
    {
      at::NoGradGuard no;
      r = rotary(live[0],
                 live.size() > 1 ? Maybe(live[1]) : Maybe(), s[0], s[1],
                 maybe(s[2]), ctx->saved_data["offset"].toInt(),
                 ctx->saved_data["interleaved"].toBool(), true);
    }
    for (size_t i = 0; i < which.size(); ++i)
      res[which[i]] = once(r[i], live[0], live.back(), live[0]);
    return res;
  }
};

}  // namespace

at::Tensor linear_ce(const at::Tensor& x, const at::Tensor& w,
                     const c10::optional<at::Tensor>& bias,
                     const at::Tensor& labels, int64_t ignore,
                     double smoothing, int64_t reduction) {
  return LinearCE::apply(x, w, or_other(bias, labels), labels,
                         bias.has_value(), ignore, smoothing, reduction);
}

// {q'} or {q', k'}
std::vector<at::Tensor> rotary_positions(
    const at::Tensor& q, const c10::optional<at::Tensor>& k,
    const at::Tensor& cos, const at::Tensor& sin,
    const c10::optional<at::Tensor>& positions, int64_t offset,
    bool interleaved) {
  return Rotary::apply(q, or_other(k, cos), cos, sin,
                       or_other(positions, cos), k.has_value(),
                       positions.has_value(), offset, interleaved);
}
