// Torch entry points of the ragged expert products (see ragged_bindings.cpp).
#pragma once
#include <torch/extension.h>
#include <vector>

namespace abacus {
namespace ragged {
torch::Tensor stage(torch::Tensor t, int64_t planes);
void rows(std::vector<torch::Tensor> a, std::vector<torch::Tensor> b, torch::Tensor offsets, torch::Tensor out,
          bool transposed);
void swiglu(torch::Tensor x, torch::Tensor w_gate, torch::Tensor w_up, torch::Tensor offsets, torch::Tensor g,
            torch::Tensor u, torch::Tensor h);
void swiglu_bwd(torch::Tensor dy, torch::Tensor w_down, torch::Tensor offsets, torch::Tensor g, torch::Tensor u,
                torch::Tensor dg, torch::Tensor du);
void weights(torch::Tensor x, std::vector<torch::Tensor> dy, torch::Tensor offsets, std::vector<torch::Tensor> dw);
}  // namespace ragged
}  // namespace abacus
