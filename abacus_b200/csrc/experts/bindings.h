// Torch entry points of the expert operators: the products (see ragged_bindings.cpp) ...
#pragma once
#include <torch/extension.h>
#include <tuple>
#include <vector>

namespace abacus {
namespace ragged {
torch::Tensor stage(torch::Tensor t, int64_t planes, c10::optional<torch::Tensor> offsets);
void rows(std::vector<torch::Tensor> a, std::vector<torch::Tensor> b, torch::Tensor offsets, torch::Tensor out,
          bool transposed);
void swiglu(torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up, torch::Tensor offsets, torch::Tensor g,
            torch::Tensor u, torch::Tensor h);
void swiglu_bwd(torch::Tensor dy, torch::Tensor w_down, torch::Tensor offsets, torch::Tensor g, torch::Tensor u,
                torch::Tensor dg, torch::Tensor du);
void weights(torch::Tensor x, std::vector<torch::Tensor> dy, torch::Tensor offsets, std::vector<torch::Tensor> dw);
}  // namespace ragged

// Differentiable operators (see functions.cpp).
namespace experts {
std::tuple<torch::Tensor, torch::Tensor, torch::Tensor> plan(torch::Tensor indices, int64_t n_experts);
torch::Tensor dispatch(torch::Tensor x, torch::Tensor offsets, torch::Tensor slot);
torch::Tensor combine(torch::Tensor ys, torch::Tensor weights, torch::Tensor offsets, torch::Tensor slot);
torch::Tensor matmul(torch::Tensor x, torch::Tensor w, torch::Tensor offsets, int64_t fp32_planes);
torch::Tensor swiglu_mlp(torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up, torch::Tensor w_down,
                         torch::Tensor offsets, int64_t fp32_planes);
}  // namespace experts
}  // namespace abacus
