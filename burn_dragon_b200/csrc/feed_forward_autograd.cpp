// feed_forward_autograd.cpp — linear_act and gated_linear as one node of the autograd graph: one crossing from Python
// forward, none backward (a node in Python took 180 us of host time for a forward and backward pass).
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include "feed_forward_host.h"

namespace bd {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Call {
  double bg0, bu0;
  int64_t act, keep;
  bool up_relu;
};

// The operands with their heads: x, z [M, K] or [M, H, K], weights [H, K, N], r and y [M, H, N].
at::Tensor with_heads(const at::Tensor& w) { return w.dim() == 3 ? w : w.unsqueeze(0); }
OptTensor with_heads(const OptTensor& w) { return w ? OptTensor(with_heads(*w)) : c10::nullopt; }
at::Tensor rows(const at::Tensor& t, bool heads) { return heads ? t : t.reshape({-1, t.size(-1)}); }
OptTensor rows(const OptTensor& t, bool heads) { return t ? OptTensor(rows(*t, heads)) : c10::nullopt; }
at::Tensor outputs(const at::Tensor& t, bool heads) { return heads ? t : t.reshape({-1, 1, t.size(-1)}); }

// As the kernels read it: 16-byte aligned rows, contiguous in the last dimension.
bool fits_rows(const at::Tensor& t) {
  if (t.stride(-1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) % 8 || t.stride(i) <= 0) return false;
  return true;
}
at::Tensor fit_rows(const at::Tensor& t) { return fits_rows(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

OptTensor given(const at::Tensor& t) { return t.defined() ? OptTensor(t) : c10::nullopt; }

class FeedForward : public torch::autograd::Function<FeedForward> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const OptTensor& z, const at::Tensor& wg,
                            const OptTensor& wu, const OptTensor& bg, const OptTensor& bu, const OptTensor& residual,
                            const Call& call, const at::Tensor& err) {
    const bool heads = wg.dim() == 3;
    const OptTensor r = residual ? OptTensor(outputs(*residual, heads)) : c10::nullopt;
    auto out = ff_forward(rows(x, heads), rows(z, heads), with_heads(wg), with_heads(wu), bg, bu, call.bg0, call.bu0, r,
                          call.act, call.up_relu, call.keep, err);
    const at::Tensor none;
    variable_list saved{x, z.value_or(none), wg, wu.value_or(none), bg.value_or(none), bu.value_or(none)};
    saved.insert(saved.end(), out.begin() + 1, out.end());
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["bg0"] = call.bg0;
    ctx->saved_data["bu0"] = call.bu0;
    ctx->saved_data["how"] = call.act | call.keep << 8 | (call.up_relu ? 1 << 16 : 0);
    ctx->saved_data["err"] = err;
    ctx->saved_data["residual"] = residual.has_value();
    if (heads) return out[0];
    auto shape = x.sizes().vec();
    shape.back() = wg.size(-1);
    return out[0].view(shape);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &wg = saved[2];
    const bool heads = wg.dim() == 3;
    const int64_t how = ctx->saved_data["how"].toInt();
    variable_list out(9);
    int64_t want = 0;
    size_t edge = 0;  // of the graph: the tensors that were given, in order
    for (int i = 0; i < 6; ++i)
      if (saved[i].defined() && ctx->needs_input_grad(edge++)) want |= 1 << i;
    {
      at::NoGradGuard no_grad;
      const std::vector<at::Tensor> held(saved.begin() + 6, saved.end());
      if (want) {
        auto got = ff_backward(fit_rows(outputs(grads[0], heads)), rows(x, heads), rows(given(saved[1]), heads), with_heads(wg),
                               with_heads(given(saved[3])), given(saved[4]), given(saved[5]), ctx->saved_data["bg0"].toDouble(),
                               ctx->saved_data["bu0"].toDouble(), held, how & 255, (how >> 16) & 1, (how >> 8) & 255, want,
                               ctx->saved_data["err"].toTensor());
        for (int i = 0; i < 6; ++i)
          if (want >> i & 1) out[i] = i < 2 ? got[i].view(saved[i].sizes()) : heads || i > 3 ? got[i] : got[i].squeeze(0);
      }
    }
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(edge)) out[6] = grads[0];
    if (at::GradMode::is_enabled()) {  // a graph of these gradients is wanted: it ends in an error, not in constants
      variable_list first(out.begin(), out.begin() + 6);
      for (auto& g : first)
        if (g.defined()) g = g.detach().set_requires_grad(true);
      auto error = std::make_shared<torch::autograd::DelayedError>("linear_act / gated_linear have no second derivative", 6);
      first = (*error)(std::move(first));
      std::copy(first.begin(), first.end(), out.begin());
    }
    return out;
  }
};

bool operand(const at::Tensor& t, const at::Tensor& like) {
  return t.is_cuda() && t.get_device() == like.get_device() && t.scalar_type() == like.scalar_type() &&
         !t._fw_grad(0).defined();
}

bool weight(const at::Tensor& w, const at::Tensor& like) {
  if (!operand(w, like) || w.dim() != like.dim() || w.sizes() != like.sizes()) return false;
  const int64_t inner = w.stride(-1) == 1 ? -1 : -2, other = -3 - inner;
  if (w.stride(inner) != 1 || w.stride(other) % 8 || w.stride(other) <= 0) return false;
  if ((w.stride(-1) == 1) != (like.stride(-1) == 1)) return false;
  if (w.dim() == 3 && (w.stride(0) % 8 || w.stride(0) <= 0)) return false;
  return reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0;
}

bool bias(const at::Tensor& b, const at::Tensor& w, bool heads) {
  return b.is_cuda() && b.get_device() == w.get_device() && (b.scalar_type() == w.scalar_type() || b.scalar_type() == at::kFloat) &&
         !b._fw_grad(0).defined() && b.is_contiguous() && reinterpret_cast<uintptr_t>(b.data_ptr()) % 16 == 0 &&
         (heads ? b.dim() == 2 && b.size(0) == w.size(0) && b.size(1) == w.size(2) : b.dim() == 1 && b.size(0) == w.size(1));
}

// Rows, or a weight (turned as it lies), with zeros behind.
at::Tensor grow_rows(const at::Tensor& t, int64_t cols) {
  if (t.size(-1) == cols) return t;
  auto shape = t.sizes().vec();
  shape.back() = cols;
  const at::Tensor flat = t.reshape({1, -1, t.size(-1)});
  return ff_pad(flat.stride(2) == 1 || flat.size(2) == 1 ? flat : flat.contiguous(), flat.size(1), cols).view(shape);
}
at::Tensor grow_weight(const at::Tensor& w, int64_t K8, int64_t N8) {
  if (w.size(0) == K8 && w.size(1) == N8) return w;
  if (w.stride(1) != 1 && w.stride(0) == 1) return ff_pad(w.t().unsqueeze(0), N8, K8).squeeze(0).t();
  return ff_pad((w.stride(1) == 1 ? w : w.contiguous()).unsqueeze(0), K8, N8).squeeze(0);
}

}  // namespace

OptTensor ff_call(const at::Tensor& x, const OptTensor& z, const at::Tensor& wg, const OptTensor& wu, const OptTensor& bg,
                  const OptTensor& bu, double bg0, double bu0, const OptTensor& residual, int64_t act, bool up_relu,
                  int64_t keep, const at::Tensor& err);

namespace {

// The call without gradients and heads at sizes that are not multiples of 8: operands padded by a kernel each.
OptTensor padded(const at::Tensor& x, const OptTensor& z, const at::Tensor& wg, const OptTensor& wu, const OptTensor& bg,
                 const OptTensor& bu, double bg0, double bu0, const OptTensor& residual, int64_t act, bool up_relu,
                 const at::Tensor& err) {
  const int64_t K = wg.size(0), N = wg.size(1), K8 = (K + 7) / 8 * 8, N8 = (N + 7) / 8 * 8;
  auto rows_like = [&](const at::Tensor& t, int64_t cols) {
    if (!operand(t, wg) || t.dim() != x.dim() || t.dim() < 1 || t.size(-1) != cols || t.numel() == 0) return false;
    for (int64_t i = 0; i + 1 < x.dim(); ++i)
      if (t.size(i) != x.size(i)) return false;
    return true;
  };
  if (K == 0 || N == 0 || !operand(wg, wg) || !rows_like(x, K) || (z && (!wu || !rows_like(*z, K))) ||
      (residual && (wu || !rows_like(*residual, N))) ||
      (wu && (!operand(*wu, wg) || wu->dim() != 2 || wu->sizes() != wg.sizes())))
    return c10::nullopt;
  for (const OptTensor* b : {&bg, &bu})
    if (*b && (!(*b)->is_cuda() || (*b)->get_device() != wg.get_device() || (*b)->dim() != 1 || (*b)->size(0) != N ||
               ((*b)->scalar_type() != wg.scalar_type() && (*b)->scalar_type() != at::kFloat) || (*b)->_fw_grad(0).defined()))
      return c10::nullopt;
  auto bias8 = [&](const OptTensor& b) { return b ? OptTensor(at::constant_pad_nd(*b, {0, N8 - N}).contiguous()) : b; };
  at::Tensor w2 = wu ? grow_weight(*wu, K8, N8) : at::Tensor();
  const at::Tensor w1 = grow_weight(wg, K8, N8);
  if (wu && (w2.stride(-1) == 1) != (w1.stride(-1) == 1)) return c10::nullopt;
  const OptTensor y = ff_call(grow_rows(x, K8), z ? OptTensor(grow_rows(*z, K8)) : z, w1, wu ? OptTensor(w2) : wu, bias8(bg),
                              bias8(bu), bg0, bu0, residual ? OptTensor(grow_rows(*residual, N8)) : residual, act, up_relu, 0, err);
  return y ? OptTensor(y->narrow(-1, 0, N)) : y;
}

}  // namespace

// y of linear_act (no wu) or gated_linear, with its node of the graph where a gradient is wanted; nothing where an argument
// needs a look first (a copy, padding, an error). keep: 0 recompute, 1 in 16 bits, 2 in 8 bits.
OptTensor ff_call(const at::Tensor& x, const OptTensor& z, const at::Tensor& wg, const OptTensor& wu, const OptTensor& bg,
                  const OptTensor& bu, double bg0, double bu0, const OptTensor& residual, int64_t act, bool up_relu,
                  int64_t keep, const at::Tensor& err) {
  if (!wg.is_cuda() || (wg.scalar_type() != at::kBFloat16 && wg.scalar_type() != at::kHalf)) return c10::nullopt;
  const bool heads = wg.dim() == 3;
  if (!heads && wg.dim() != 2) return c10::nullopt;
  const int64_t H = heads ? wg.size(0) : 1, K = wg.size(-2), N = wg.size(-1);
  if (!heads && (K % 8 || N % 8)) {
    bool wants = x.requires_grad() || wg.requires_grad();
    for (const OptTensor* t : {&z, &wu, &bg, &bu, &residual}) wants |= *t && (*t)->requires_grad();
    if (at::GradMode::is_enabled() && wants) return c10::nullopt;
    at::NoGradGuard no_grad;
    return padded(x, z, wg, wu, bg, bu, bg0, bu0, residual, act, up_relu, err);
  }
  if (K % 8 || N % 8 || K == 0 || N == 0 || H == 0 || !weight(wg, wg) || (wu && !weight(*wu, wg))) return c10::nullopt;
  auto input = [&](const at::Tensor& t) {
    if (!operand(t, wg) || t.dim() < 1 || t.size(-1) != K || t.numel() == 0) return false;
    if (heads ? !(t.dim() == 2 || (t.dim() == 3 && t.size(1) == H)) : t.dim() > 2 && !t.is_contiguous()) return false;
    return fits_rows(t);
  };
  if (!input(x) || (z && (!wu || !input(*z) || (heads ? z->size(0) != x.size(0) : z->sizes() != x.sizes())))) return c10::nullopt;
  if ((bg && !bias(*bg, wg, heads)) || (bu && !bias(*bu, wg, heads)) || (bg && bu && bg->scalar_type() != bu->scalar_type()))
    return c10::nullopt;
  if (residual) {
    if (!operand(*residual, wg) || heads || wu || residual->dim() != x.dim() || residual->size(-1) != N) return c10::nullopt;
    for (int64_t i = 0; i + 1 < x.dim(); ++i)
      if (residual->size(i) != x.size(i)) return c10::nullopt;
    if ((residual->dim() > 2 && !residual->is_contiguous()) || !fits_rows(*residual)) return c10::nullopt;
  }
  const at::Tensor* all[] = {&x, &wg};
  bool train = false;
  if (at::GradMode::is_enabled()) {
    for (const at::Tensor* t : all) train |= t->requires_grad();
    for (const OptTensor* t : {&z, &wu, &bg, &bu, &residual}) train |= *t && (*t)->requires_grad();
  }
  const bool nothing = !wu && act == 0;  // dp is dy
  const Call call{bg0, bu0, act, train && !nothing ? keep : 0, up_relu};
  if (train) return FeedForward::apply(x, z, wg, wu, bg, bu, residual, call, err);
  const OptTensor r = residual ? OptTensor(outputs(*residual, heads)) : c10::nullopt;
  at::Tensor y = ff_forward(rows(x, heads), rows(z, heads), with_heads(wg), with_heads(wu), bg, bu, bg0, bu0, r, act, up_relu, 0,
                            err)[0];
  if (heads) return y;
  auto shape = x.sizes().vec();
  shape.back() = N;
  return y.view(shape);
}

}  // namespace bd
