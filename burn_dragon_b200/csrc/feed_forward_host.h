// feed_forward_host.h — the feed-forward products (feed_forward.cu) as the autograd node calls them.
#pragma once
#include <torch/extension.h>

#include <vector>

namespace bd {

using OptTensor = c10::optional<at::Tensor>;

// y [M, H, N] and what the backward pass goes by: [held, exponents] a projection (none, 16-bit values, or codes).
std::vector<at::Tensor> ff_forward(const at::Tensor& x, const OptTensor& z, const at::Tensor& wg, const OptTensor& wu,
                                   const OptTensor& bg, const OptTensor& bu, double bg0, double bu0, const OptTensor& residual,
                                   int64_t act, bool up_relu, int64_t keep, const at::Tensor& err);

// dx, dz, dwg, dwu, dbg, dbu from dy [M, H, N]; what is not wanted (a bit each in `want`) is an empty tensor. `held`: as
// ff_forward gave it; empty: the pre-activations are computed again.
std::vector<at::Tensor> ff_backward(const at::Tensor& dy, const at::Tensor& x, const OptTensor& z, const at::Tensor& wg,
                                    const OptTensor& wu, const OptTensor& bg, const OptTensor& bu, double bg0, double bu0,
                                    const std::vector<at::Tensor>& held, int64_t act, bool up_relu, int64_t keep,
                                    int64_t want, const at::Tensor& err);

// t [B, R, C] of 16-bit values, the last dimension contiguous, grown to [B, R8, C8] by zeros (C8 a multiple of 8).
at::Tensor ff_pad(const at::Tensor& t, int64_t R8, int64_t C8);

}  // namespace bd
