// The differentiable expert operators that abacus_b200/ops/experts.py exports for CUDA tensors: argument checks, workspaces
// and autograd nodes around the kernels. They are C++ nodes because a short batch is bound by the host: the same nodes in
// Python took 142 us for the routing of 256 tokens with its gradients, whose kernels take 17.
//
// None of them is differentiable twice; a backward pass that records a graph is refused.
#include <torch/extension.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include "../common/host.h"
#include "../ops/expert_rows.h"
#include "bindings.h"
#include "few.h"
#include "ragged.h"

namespace abacus {
namespace experts {
namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

bool row_type(const Tensor& t) { return t.scalar_type() == torch::kFloat32 || t.scalar_type() == torch::kBFloat16; }

void check_rows(const Tensor& t, const char* name, int64_t rows = -1) {
  TORCH_CHECK_VALUE(t.dim() == 2 && row_type(t), name, " must be a 2-D fp32 or bf16 tensor, got ", t.sizes(), " ",
                    t.scalar_type());
  TORCH_CHECK_VALUE(rows < 0 || t.size(0) == rows, name, " must have ", rows, " rows, got ", t.size(0));
}

// Rows that a kernel can walk: unit inner stride, no overlap.
Tensor walkable(const Tensor& t) {
  return t.stride(1) == 1 && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous();
}

void once_only(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " is not differentiable twice (create_graph=True)");
}

void check_plan(const Tensor& offsets, const Tensor& slot, const Tensor& like) {
  TORCH_CHECK_VALUE(offsets.device() == like.device() && slot.device() == like.device(),
                    "the rows and the plan must be on one device");
}

// Sum over each token's kept choices, weighted or not.
Tensor combine_rows(const Tensor& ys, c10::optional<Tensor> weights, const Tensor& slot) {
  auto out = torch::empty({slot.size(0), ys.size(1)}, ys.options());
  ops::expert_combine(ys, weights, slot, out);
  return out;
}

struct Dispatch : torch::autograd::Function<Dispatch> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& offsets, const Tensor& slot) {
    ctx->save_for_backward({slot});
    auto xs = torch::empty({slot.numel(), x.size(1)}, x.options());
    ops::expert_dispatch(walkable(x), slot, offsets, xs);
    return xs;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("dispatch_tokens");
    return {combine_rows(grads[0].contiguous(), c10::nullopt, ctx->get_saved_variables()[0]), Tensor(), Tensor()};
  }
};

struct Combine : torch::autograd::Function<Combine> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ys, const Tensor& weights, const Tensor& offsets,
                        const Tensor& slot) {
    ctx->save_for_backward({ys, weights, offsets, slot});
    return combine_rows(ys, weights, slot);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("combine_tokens");
    const auto saved = ctx->get_saved_variables();
    auto dys = torch::empty_like(saved[0]), dweights = torch::empty_like(saved[1]);
    ops::expert_combine_bwd(grads[0].contiguous(), saved[0], saved[1], saved[3], saved[2], dys, dweights);
    return {dys, dweights, Tensor(), Tensor()};
  }
};

// Whether TMA can read `t` where it lies.
bool read_in_place(const Tensor& t) {
  const int64_t d = t.dim();
  if (t.scalar_type() != torch::kBFloat16 || t.stride(d - 1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0)
    return false;
  bool aligned = t.size(d - 2) <= 1 || t.stride(d - 2) >= t.size(d - 1);
  for (int64_t i = 0; i < d - 1; ++i) aligned = aligned && (t.size(i) <= 1 || (t.stride(i) % 8 == 0 && t.stride(i) > 0));
  return aligned;
}

// `t` as the product kernels read it: bf16 planes first, rows 16-byte aligned. bf16 tensors laid out so already are used in
// place. With offsets, `t` holds the experts' matrices, and those of experts without rows are left out of a copy.
Tensor operand(const Tensor& t, int64_t planes, c10::optional<Tensor> offsets = c10::nullopt) {
  return read_in_place(t) ? t.unsqueeze(0) : ragged::stage(t, planes, offsets);
}

// ---------------------------------------------------------------- few rows (few.cu)
// Few rows, and matrices that the tensor-core path would copy first: fp32 ones, and bf16 ones whose rows are not whole
// 16-byte units. Other bf16 matrices are read in place there, and it is as fast or faster from one row an expert on
// (32 experts of 2048 x 2048: 50 us against 61 with one row each). The choice goes by sizes and type alone, so that a
// tensor's layout does not change its product's bits.
bool few(const Tensor& x, const Tensor& w, const Tensor& offsets) {
  const bool bf16 = w.scalar_type() == torch::kBFloat16;
  return ragged::few_rows(x.size(0), offsets.numel() - 1, bf16) && (!bf16 || w.size(2) % 8 != 0);
}

// Matrices whose rows lie in one piece.
Tensor rows_in_one_piece(const Tensor& w) { return w.stride(2) == 1 ? w : w.contiguous(); }

ragged::FewParams few_params(const Tensor& a, const Tensor& b, const Tensor& offsets, const Tensor& out) {
  ragged::FewParams p = {};
  p.a = a.data_ptr();
  p.b = b.data_ptr();
  p.out = out.data_ptr();
  p.a_bf16 = a.scalar_type() == torch::kBFloat16;
  p.b_bf16 = b.scalar_type() == torch::kBFloat16;
  p.out_bf16 = out.scalar_type() == torch::kBFloat16;
  p.ld_a = a.stride(0);
  p.offsets = offsets.data_ptr<int>();
  p.experts = static_cast<int>(offsets.numel() - 1);
  p.rows = static_cast<int>(a.size(0));
  p.status = host::status_ptr(static_cast<int>(a.get_device()));
  return p;
}

void launched(cudaError_t err) {
  C10_CUDA_CHECK(err);
  host::note_launch();
}

// out = a times the experts' matrices, or their transposes (with `add` added).
void few_rows_product(const Tensor& a, const Tensor& w, const Tensor& offsets, const Tensor& out, bool transposed,
                      const Tensor& add = Tensor()) {
  if (a.size(0) == 0) return;
  const c10::cuda::CUDAGuard guard(a.device());
  auto p = few_params(a, w, offsets, out);
  p.ld_b = w.stride(1);
  p.stride_b = w.stride(0);
  p.ld_out = out.stride(0);
  p.k = static_cast<int>(w.size(transposed ? 2 : 1));
  p.n = static_cast<int>(w.size(transposed ? 1 : 2));
  if (add.defined()) {
    p.add = add.data_ptr<float>();
    p.ld_add = add.stride(0);
  }
  const auto stream = at::cuda::getCurrentCUDAStream();
  launched(transposed ? launch_few_transposed(p, stream) : launch_few(p, stream));
}

void few_weights(const Tensor& a, const Tensor& b, const Tensor& offsets, const Tensor& out) {
  const c10::cuda::CUDAGuard guard(a.device());
  auto p = few_params(a, b, offsets, out);
  p.ld_b = b.stride(0);
  p.m = static_cast<int>(out.size(1));
  p.n = static_cast<int>(out.size(2));
  launched(launch_few_weights(p, at::cuda::getCurrentCUDAStream()));
}

Tensor like_matrix(const Tensor& w) { return torch::empty(w.sizes(), w.options()); }

// Empty ([planes,] rows, cols) whose rows start at 16-byte boundaries.
Tensor padded(int64_t planes, int64_t rows, int64_t cols, torch::TensorOptions options) {
  const int64_t unit = options.dtype() == torch::kBFloat16 ? 8 : 4, ld = (cols + unit - 1) / unit * unit;
  const auto t = planes ? torch::empty({planes, rows, ld}, options) : torch::empty({rows, ld}, options);
  return ld == cols ? t : t.narrow(-1, 0, cols);
}

struct RaggedMatmul : torch::autograd::Function<RaggedMatmul> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Tensor& offsets, int64_t planes) {
    if (few(x, w, offsets)) {
      const auto xr = walkable(x), wr = rows_in_one_piece(w);
      ctx->save_for_backward({xr, wr, offsets});
      ctx->saved_data["planes"] = static_cast<int64_t>(0);
      auto y = torch::empty({x.size(0), w.size(2)}, x.options());
      few_rows_product(xr, wr, offsets, y, false);
      return y;
    }
    // The backward reads x as an operand: where that is a copy it is kept in place of x (6 bytes an element in fp32; w's,
    // which would stay for the whole forward of a model, is made again).
    const auto xo = operand(x, planes);
    ctx->save_for_backward({xo, w, offsets});
    ctx->saved_data["planes"] = planes;
    auto y = torch::empty({x.size(0), w.size(2)}, x.options());
    ragged::rows({xo}, {operand(w, planes, offsets)}, offsets, y, false);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("ragged_matmul");
    const auto saved = ctx->get_saved_variables();
    const auto &x = saved[0], &w = saved[1], &offsets = saved[2];
    const int64_t planes = ctx->saved_data["planes"].toInt();
    Tensor dx, dw;
    if (planes == 0) {
      const auto dy = walkable(grads[0]);
      if (ctx->needs_input_grad(0)) {
        dx = torch::empty(x.sizes(), w.options());
        few_rows_product(dy, w, offsets, dx, true);
      }
      if (ctx->needs_input_grad(1)) {
        dw = like_matrix(w);
        few_weights(x, dy, offsets, dw);
      }
      return {dx, dw, Tensor(), Tensor()};
    }
    const auto dy = operand(grads[0], planes);
    if (ctx->needs_input_grad(0)) {
      dx = torch::empty({x.size(1), x.size(2)}, w.options());
      ragged::rows({dy}, {operand(w, planes, offsets)}, offsets, dx, true);
    }
    if (ctx->needs_input_grad(1)) {
      dw = like_matrix(w);
      ragged::weights(x, {dy}, offsets, {dw});
    }
    return {dx, dw, Tensor(), Tensor()};
  }
};

// The kernels write h and the gradients of gate and up as the operands (bf16 planes) of the products that read them; the
// operands of x and h are kept for the backward in place of the tensors.
struct RaggedSwiGLU : torch::autograd::Function<RaggedSwiGLU> {
  static variable_list backward_of_few(AutogradContext* ctx, const variable_list& saved, const Tensor& grad) {
    const auto &x = saved[0], &w_gate = saved[1], &w_up = saved[2], &w_down = saved[3], &offsets = saved[4], &g = saved[5],
               &u = saved[6], &h = saved[7];
    const auto dy = walkable(grad);
    const auto dgu = torch::empty({2, g.size(0), g.size(1)}, g.options());
    const auto dg = dgu[0], du = dgu[1];
    few_rows_product(dy, w_down, offsets, dg, true);  // dh, in the place of dg
    if (g.numel() > 0) {
      const c10::cuda::CUDAGuard guard(x.device());
      launched(ragged::launch_few_swiglu_bwd(dg.data_ptr<float>(), g.data_ptr<float>(), u.data_ptr<float>(),
                                             dg.data_ptr<float>(), du.data_ptr<float>(), g.numel(),
                                             at::cuda::getCurrentCUDAStream()));
    }
    variable_list out(6);
    if (ctx->needs_input_grad(0)) {
      const auto part = torch::empty(x.sizes(), g.options());
      out[0] = torch::empty(x.sizes(), w_gate.options());
      few_rows_product(dg, w_gate, offsets, part, true);
      few_rows_product(du, w_up, offsets, out[0], true, part);
    }
    const Tensor* matrices[3] = {&w_gate, &w_up, &w_down};
    for (int i = 0; i < 3; ++i) {
      if (!ctx->needs_input_grad(i + 1)) continue;
      out[i + 1] = like_matrix(*matrices[i]);
      few_weights(i < 2 ? x : h, i == 0 ? dg : i == 1 ? du : dy, offsets, out[i + 1]);
    }
    return out;
  }
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                        const Tensor& w_down, const Tensor& offsets, int64_t planes) {
    const int64_t rows = x.size(0), hidden = w_gate.size(2);
    const auto kept = x.options().dtype(torch::kFloat32);
    if (few(x, w_gate, offsets) || few(x, w_down, offsets)) {
      // gate, up and h stay fp32 throughout.
      const auto xr = walkable(x), wg = rows_in_one_piece(w_gate), wu = rows_in_one_piece(w_up), wd = rows_in_one_piece(w_down);
      const auto guh = torch::empty({3, rows, hidden}, kept);
      const auto g = guh[0], u = guh[1], h = guh[2];
      auto y = torch::empty({rows, w_down.size(2)}, x.options());
      few_rows_product(xr, wg, offsets, g, false);
      few_rows_product(xr, wu, offsets, u, false);
      if (rows > 0) {
        const c10::cuda::CUDAGuard guard(x.device());
        launched(ragged::launch_few_swiglu(g.data_ptr<float>(), u.data_ptr<float>(), h.data_ptr<float>(), g.numel(),
                                           at::cuda::getCurrentCUDAStream()));
      }
      few_rows_product(h, wd, offsets, y, false);
      ctx->save_for_backward({xr, wg, wu, wd, offsets, g, u, h});
      return y;
    }
    const auto g = padded(0, rows, hidden, kept), u = padded(0, rows, hidden, kept);
    const auto h = padded(planes, rows, hidden, x.options().dtype(torch::kBFloat16));
    auto y = torch::empty({rows, w_down.size(2)}, x.options());
    const auto xo = operand(x, planes);
    ragged::swiglu(xo, operand(w_gate, planes, offsets), operand(w_up, planes, offsets), offsets, g, u, h);
    ragged::rows({h}, {operand(w_down, planes, offsets)}, offsets, y, false);
    ctx->save_for_backward({xo, w_gate, w_up, w_down, offsets, g, u, h});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once_only("ragged_swiglu_mlp");
    const auto saved = ctx->get_saved_variables();
    const auto &x = saved[0], &w_gate = saved[1], &w_up = saved[2], &w_down = saved[3], &offsets = saved[4], &g = saved[5],
               &u = saved[6], &h = saved[7];
    if (h.dim() == 2) return backward_of_few(ctx, saved, grads[0]);
    const int64_t planes = h.size(0), rows = g.size(0), hidden = g.size(1);
    const auto dy = operand(grads[0], planes);
    const auto dg = padded(planes, rows, hidden, h.options()), du = padded(planes, rows, hidden, h.options());
    ragged::swiglu_bwd(dy, operand(w_down, planes, offsets), offsets, g, u, dg, du);
    variable_list out(6);
    if (ctx->needs_input_grad(0)) {
      out[0] = torch::empty({rows, x.size(2)}, w_gate.options());
      ragged::rows({dg, du}, {operand(w_gate, planes, offsets), operand(w_up, planes, offsets)}, offsets, out[0], true);
    }
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
      Tensor dw_gate = like_matrix(w_gate), dw_up = like_matrix(w_up);
      ragged::weights(x, {dg, du}, offsets, {dw_gate, dw_up});
      if (ctx->needs_input_grad(1)) out[1] = dw_gate;
      if (ctx->needs_input_grad(2)) out[2] = dw_up;
    }
    if (ctx->needs_input_grad(3)) {
      out[3] = like_matrix(w_down);
      ragged::weights(h, {dy}, offsets, {out[3]});
    }
    return out;
  }
};

int64_t planes_of(const Tensor& x, int64_t fp32_planes) { return x.scalar_type() == torch::kBFloat16 ? 1 : fp32_planes; }

void check_products(const Tensor& x, const Tensor& w, const char* name, int64_t in, int64_t out, const Tensor& offsets) {
  const int64_t experts = offsets.numel() - 1;
  TORCH_CHECK_VALUE(w.dim() == 3, name, " must be (experts, in, out), got ", w.sizes());
  TORCH_CHECK_VALUE(w.scalar_type() == x.scalar_type() && w.size(0) == experts && w.size(1) == in && w.size(2) == out, name,
                    " must be ", x.scalar_type(), " of shape [", experts, ", ", in, ", ", out, "], got ", w.scalar_type(),
                    " ", w.sizes());
  TORCH_CHECK_VALUE(w.device() == x.device() && offsets.device() == x.device(),
                    "the rows, the matrices and the offsets must be on one device");
  TORCH_CHECK_VALUE(in > 0 && out > 0, name, " has an empty dimension: ", w.sizes());
}

void check_offsets(const Tensor& offsets) {
  TORCH_CHECK_VALUE(offsets.dim() == 1 && offsets.numel() >= 2 && offsets.scalar_type() == torch::kInt32,
                    "offsets must be int32 of shape (experts + 1,), got ", offsets.sizes(), " ", offsets.scalar_type());
  TORCH_CHECK(offsets.numel() - 1 <= ragged::kMaxExperts, "ragged products take at most ", ragged::kMaxExperts,
              " experts, got ", offsets.numel() - 1);
}

}  // namespace

std::tuple<Tensor, Tensor, Tensor> plan(Tensor indices, int64_t n_experts) {
  TORCH_CHECK_VALUE(indices.dim() == 2 && (indices.scalar_type() == torch::kInt64 || indices.scalar_type() == torch::kInt32),
                    "indices must be a (tokens, choices) integer tensor, got ", indices.sizes(), " ", indices.scalar_type());
  TORCH_CHECK_VALUE(n_experts >= 1, "n_experts must be at least 1, got ", n_experts);
  const auto flat = indices.to(torch::kInt64).contiguous();
  const int64_t n = flat.numel(), bins = n_experts + 1, parts = ops::expert_plan_parts(n);
  // One allocation: offsets, order, slot, and the counts of the parts.
  const auto ints = torch::empty({bins + 2 * n + (parts > 1 ? parts * bins : 0)}, flat.options().dtype(torch::kInt32));
  const auto offsets = ints.narrow(0, 0, bins), order = ints.narrow(0, bins, n), slot = ints.narrow(0, bins + n, n);
  ops::expert_plan(flat, n_experts, offsets, order, slot, ints.narrow(0, bins + 2 * n, ints.numel() - bins - 2 * n));
  return {offsets, order, slot.view(indices.sizes())};
}

Tensor dispatch(Tensor x, Tensor offsets, Tensor slot) {
  check_rows(x, "x", slot.size(0));
  check_plan(offsets, slot, x);
  return Dispatch::apply(x, offsets, slot);
}

Tensor combine(Tensor ys, Tensor weights, Tensor offsets, Tensor slot) {
  check_rows(ys, "ys", slot.numel());
  TORCH_CHECK_VALUE(weights.sizes() == slot.sizes() && weights.scalar_type() == torch::kFloat32,
                    "weights must be fp32 of shape ", slot.sizes(), ", got ", weights.sizes(), " ", weights.scalar_type());
  check_plan(offsets, slot, ys);
  TORCH_CHECK_VALUE(weights.device() == ys.device(), "the rows and the weights must be on one device");
  return Combine::apply(ys.contiguous(), weights.contiguous(), offsets, slot);
}

Tensor matmul(Tensor x, Tensor w, Tensor offsets, int64_t fp32_planes) {
  check_rows(x, "x");
  check_offsets(offsets);
  check_products(x, w, "w", x.size(1), w.dim() == 3 ? w.size(2) : 0, offsets);
  return RaggedMatmul::apply(x, w, offsets.contiguous(), planes_of(x, fp32_planes));
}

Tensor swiglu_mlp(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, Tensor offsets, int64_t fp32_planes) {
  check_rows(x, "x");
  check_offsets(offsets);
  const int64_t hidden = w_gate.dim() == 3 ? w_gate.size(2) : 0;
  check_products(x, w_gate, "w_gate", x.size(1), hidden, offsets);
  check_products(x, w_up, "w_up", x.size(1), hidden, offsets);
  check_products(x, w_down, "w_down", hidden, w_down.dim() == 3 ? w_down.size(2) : 0, offsets);
  return RaggedSwiGLU::apply(x, w_gate, w_up, w_down, offsets.contiguous(), planes_of(x, fp32_planes));
}

}  // namespace experts
}  // namespace abacus
