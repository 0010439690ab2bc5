// Sorting routed rows by expert and moving them (see expert_rows.cu).
#pragma once
#include <torch/extension.h>

namespace abacus {
namespace ops {
void expert_plan(torch::Tensor indices, int64_t n_experts, torch::Tensor offsets, torch::Tensor order,
                 torch::Tensor slot, torch::Tensor counts);
int64_t expert_plan_parts(int64_t n);
void expert_dispatch(torch::Tensor x, torch::Tensor slot, torch::Tensor offsets, torch::Tensor xs);
void expert_combine(torch::Tensor ys, c10::optional<torch::Tensor> weights, torch::Tensor slot, torch::Tensor out);
void expert_combine_bwd(torch::Tensor dout, torch::Tensor ys, torch::Tensor weights, torch::Tensor slot,
                        torch::Tensor offsets, torch::Tensor dys, torch::Tensor dweights);
}  // namespace ops
}  // namespace abacus
