// AdamW with 8-bit moments (see adamw8.cpp).
#pragma once
#include <torch/extension.h>
#include <vector>

namespace abacus {
namespace ops {
void adamw8_step(const std::vector<torch::Tensor>& weights, const std::vector<torch::Tensor>& grads,
                 const std::vector<torch::Tensor>& exp_avg, const std::vector<torch::Tensor>& exp_avg_scale,
                 const std::vector<torch::Tensor>& exp_rms, const std::vector<torch::Tensor>& exp_rms_scale, double lr,
                 double beta1, double beta2, double eps, double weight_decay, int64_t step);
}  // namespace ops
}  // namespace abacus
