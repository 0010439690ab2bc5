// Checks and batching of the AdamW step with 8-bit moments.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <cmath>
#include "../common/host.h"
#include "adamw8.h"
#include "adamw8_kernel.h"

namespace abacus {
namespace ops {
namespace {

bool aligned(const void* p, unsigned bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace

void adamw8_step(const std::vector<torch::Tensor>& weights, const std::vector<torch::Tensor>& grads,
                 const std::vector<torch::Tensor>& exp_avg, const std::vector<torch::Tensor>& exp_avg_scale,
                 const std::vector<torch::Tensor>& exp_rms, const std::vector<torch::Tensor>& exp_rms_scale, double lr,
                 double beta1, double beta2, double eps, double weight_decay, int64_t step) {
  const size_t count = weights.size();
  TORCH_CHECK(grads.size() == count && exp_avg.size() == count && exp_avg_scale.size() == count &&
                  exp_rms.size() == count && exp_rms_scale.size() == count,
              "adamw8: the lists differ in length");
  TORCH_CHECK(step >= 1, "adamw8: step must be at least 1, got ", step);
  if (count == 0) return;
  const c10::cuda::CUDAGuard guard(weights[0].device());
  Adam8Scalars s;
  s.b1 = static_cast<float>(beta1);
  s.c1 = static_cast<float>(1.0 - beta1);
  s.b2 = static_cast<float>(beta2);
  s.c2 = static_cast<float>(1.0 - beta2);
  // a m / (u / c + eps) = (a c) m / (u + eps c): one division an element.
  const double c = std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step)));
  s.eps = static_cast<float>(eps * c);
  s.decay = static_cast<float>(1.0 - lr * weight_decay);
  s.step_size = static_cast<float>(lr * c / (1.0 - std::pow(beta1, static_cast<double>(step))));
  s.step_mix = static_cast<unsigned>(static_cast<uint64_t>(step) * 0x7F4A7C15ull);
  const auto stream = at::cuda::getCurrentCUDAStream();
  // Every tensor is looked at before the first is changed.
  for (size_t i = 0; i < count; ++i) {
    const auto &w = weights[i], &g = grads[i], &m = exp_avg[i], &u = exp_rms[i], &ms = exp_avg_scale[i],
               &us = exp_rms_scale[i];
    const int64_t n = w.numel(), blocks = (n + kAdam8Block - 1) / kAdam8Block;
    for (const auto* t : {&w, &g, &m, &u, &ms, &us}) {
      TORCH_CHECK(t->is_cuda() && t->device() == weights[0].device() && t->is_contiguous(),
                  "adamw8: tensors must be contiguous and on one CUDA device (tensor ", i, ")");
    }
    TORCH_CHECK(w.scalar_type() == torch::kFloat32 && ms.scalar_type() == torch::kFloat32 &&
                    us.scalar_type() == torch::kFloat32 && m.scalar_type() == torch::kFloat8_e4m3fn &&
                    u.scalar_type() == torch::kFloat8_e4m3fn &&
                    (g.scalar_type() == torch::kFloat32 || g.scalar_type() == torch::kBFloat16),
                "adamw8: fp32 weights and scales, float8_e4m3fn moments, fp32 or bf16 gradients (tensor ", i, ")");
    TORCH_CHECK(g.numel() == n && m.numel() == n && u.numel() == n && ms.numel() == blocks && us.numel() == blocks,
                "adamw8: sizes of tensor ", i, " (", n, " weights need ", blocks, " scales of each moment)");
    TORCH_CHECK(blocks < (1ll << 31), "adamw8: tensor ", i, " is too large");
  }
  Adam8Batch b;
  unsigned long long ctas = 0;
  b.count = 0;
  auto flush = [&] {
    if (b.count == 0) return;
    b.first[b.count] = static_cast<unsigned>(ctas);
    b.shift = 0;
    while ((ctas - 1) >> b.shift >= sizeof(b.coarse)) ++b.shift;
    int tensor = 0;
    for (unsigned long long run = 0; run << b.shift < ctas; ++run) {
      while (b.first[tensor + 1] <= run << b.shift) ++tensor;
      b.coarse[run] = static_cast<uint8_t>(tensor);
    }
    C10_CUDA_CHECK(launch_adamw8(b, s, static_cast<unsigned>(ctas), stream));
    host::note_launch();
    b.count = 0;
    ctas = 0;
  };
  for (size_t i = 0; i < count; ++i) {
    const int64_t n = weights[i].numel();
    if (n == 0) continue;
    constexpr int64_t per_cta = static_cast<int64_t>(kAdam8Block) * kAdam8Warps;
    const unsigned long long need = (n + per_cta - 1) / per_cta;
    if (b.count == kAdam8Tensors || ctas + need >= (1ull << 31)) flush();
    const int c = b.count++;
    b.w[c] = weights[i].data_ptr<float>();
    b.g[c] = grads[i].data_ptr();
    b.m[c] = static_cast<uint8_t*>(exp_avg[i].data_ptr());
    b.m_scale[c] = exp_avg_scale[i].data_ptr<float>();
    b.u[c] = static_cast<uint8_t*>(exp_rms[i].data_ptr());
    b.u_scale[c] = exp_rms_scale[i].data_ptr<float>();
    b.numel[c] = n;
    b.first[c] = static_cast<unsigned>(ctas);
    b.g_bf16[c] = grads[i].scalar_type() == torch::kBFloat16;
    b.wide[c] = aligned(b.w[c], 16) && aligned(b.g[c], b.g_bf16[c] ? 8 : 16) && aligned(b.m[c], 4) && aligned(b.u[c], 4);
    ctas += need;
  }
  flush();
}

}  // namespace ops
}  // namespace abacus
