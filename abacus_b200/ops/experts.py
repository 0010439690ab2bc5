"""Dropless mixture of experts: routed rows sorted by expert, and the experts' products over ragged counts.

    plan = expert_plan(indices_TK, n_experts)
    xs   = dispatch_tokens(x_TD, plan)                                # (T K, D), sorted by expert
    ys   = ragged_swiglu_mlp(xs, w_gate, w_up, w_down, plan.offsets)  # or ragged_matmul
    out  = combine_tokens(ys, weights_TK, plan)                       # (T, D)

Everything stays on the device: the number of rows of each expert is read by the kernels, never by the host, and no
expert's rows are padded. All functions are differentiable.

Types: fp32 or bf16 rows and matrices (both of one type), results in that type, sums in fp32. fp32 products follow
``precision.set_precision``: "fp32" multiplies three bf16 parts of each operand (all 24 bits of a number above 2^-110 or
so; the parts' smallest number is 2^-133), "tf32" two (16 bits). An infinite fp32 operand may give NaN where plain
arithmetic gives infinity (it meets the zero parts of the other operand), as in the framework's 3xTF32 products.
bf16 operands are multiplied as they are; ``ragged_swiglu_mlp`` rounds gate, up, their product and the two gradients
through it to bf16 between its products, as storing them does.

CUDA tensors run on ``csrc/experts`` and ``csrc/ops/expert_rows.cu`` (up to 256 experts for the products, 1024 for the
plan); CPU tensors run the formulas with ATen.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from abacus_b200.ops import precision
from abacus_b200.ops._ext import ext

_TYPES = (torch.float32, torch.bfloat16)


class ExpertPlan(NamedTuple):
    """Order of the T K (token, choice) assignments after a stable sort by expert, dropped ones last (int32).

    ``offsets`` (E + 1): first sorted row of each expert, then the end of the last one's.
    ``order`` (T K): assignment ``t * K + k`` of each sorted row.
    ``slot`` (T, K): sorted row of each assignment, -1 where it is dropped.
    """

    offsets: torch.Tensor
    order: torch.Tensor
    slot: torch.Tensor


def expert_plan(indices: torch.Tensor, n_experts: int) -> ExpertPlan:
    """Plan of ``indices`` (T, K), the experts that each token chose. An id outside [0, n_experts) drops the assignment."""
    if indices.ndim != 2 or indices.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"indices must be a (tokens, choices) integer tensor, got {tuple(indices.shape)} {indices.dtype}")
    if n_experts < 1:
        raise ValueError(f"n_experts must be at least 1, got {n_experts}")
    if indices.is_cuda:
        indices = indices.to(torch.int64).contiguous()
        n = indices.numel()
        parts = ext().expert_plan_parts(n)
        ints = torch.empty(n_experts + 1 + 2 * n + (parts * (n_experts + 1) if parts > 1 else 0), dtype=torch.int32, device=indices.device)
        offsets, order, slot, counts = ints.split([n_experts + 1, n, n, ints.numel() - 2 * n - n_experts - 1])
        ext().expert_plan(indices, n_experts, offsets, order, slot, counts)
        return ExpertPlan(offsets, order, slot.view(indices.shape))
    flat = indices.reshape(-1).long()
    kept = (flat >= 0) & (flat < n_experts)
    key = torch.where(kept, flat, n_experts)
    order = torch.argsort(key, stable=True)
    slot = torch.empty_like(order)
    slot[order] = torch.arange(order.numel())
    counts = torch.bincount(key, minlength=n_experts + 1)[:n_experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    slot = torch.where(kept, slot, -1).view(indices.shape)
    return ExpertPlan(offsets.to(torch.int32), order.to(torch.int32), slot.to(torch.int32))


def _check_rows(name: str, t: torch.Tensor, rows: int | None = None) -> None:
    if t.ndim != 2 or t.dtype not in _TYPES:
        raise ValueError(f"{name} must be a 2-D fp32 or bf16 tensor, got {tuple(t.shape)} {t.dtype}")
    if rows is not None and t.shape[0] != rows:
        raise ValueError(f"{name} must have {rows} rows, got {t.shape[0]}")


def _unit_inner(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, offsets, slot):
        ctx.save_for_backward(slot)
        tokens, choices = slot.shape
        if not x.is_cuda:
            xs = x.new_zeros(tokens * choices, x.shape[1])
            t, k = torch.nonzero(slot >= 0, as_tuple=True)
            xs[slot[t, k].long()] = x[t]
            return xs
        xs = torch.empty(tokens * choices, x.shape[1], dtype=x.dtype, device=x.device)
        ext().expert_dispatch(_unit_inner(x), slot, offsets, xs)
        return xs

    @staticmethod
    def backward(ctx, dxs):
        (slot,) = ctx.saved_tensors
        return _combine(dxs.contiguous(), None, slot), None, None


def _combine(ys: torch.Tensor, weights: torch.Tensor | None, slot: torch.Tensor) -> torch.Tensor:
    tokens, choices = slot.shape
    if ys.is_cuda:
        out = torch.empty(tokens, ys.shape[1], dtype=ys.dtype, device=ys.device)
        ext().expert_combine(ys, weights, slot, out)
        return out
    if choices == 0 or ys.shape[0] == 0:
        return ys.new_zeros(tokens, ys.shape[1])
    scale = (slot >= 0).float() if weights is None else torch.where(slot >= 0, weights, 0.0)
    rows = torch.where(slot[..., None] >= 0, ys.float()[slot.clamp(min=0).long()], 0.0)
    return (rows * scale[..., None]).sum(1).to(ys.dtype)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ys, weights, offsets, slot):
        ctx.save_for_backward(ys, weights, offsets, slot)
        return _combine(ys, weights, slot)

    @staticmethod
    def backward(ctx, dout):
        ys, weights, offsets, slot = ctx.saved_tensors
        dout = dout.contiguous()
        if ys.is_cuda:
            dys, dweights = torch.empty_like(ys), torch.empty_like(weights)
            ext().expert_combine_bwd(dout, ys, weights, slot, offsets, dys, dweights)
            return dys, dweights, None, None
        dys, dweights = torch.zeros_like(ys), torch.zeros_like(weights)
        t, k = torch.nonzero(slot >= 0, as_tuple=True)
        rows = slot[t, k].long()
        d = dout[t].float()
        dys[rows] = (weights[t, k, None] * d).to(ys.dtype)
        dweights[t, k] = (ys[rows].float() * d).sum(1)
        return dys, dweights, None, None


def dispatch_tokens(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """Rows of ``x`` (T, D) in the plan's order, one for each choice (T K, D); rows after the last expert's are zeros."""
    _check_rows("x", x, plan.slot.shape[0])
    return _Dispatch.apply(x, plan.offsets, plan.slot)


def combine_tokens(ys: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """``out[t] = sum_k weights[t, k] * ys[slot[t, k]]`` (T, D) of the sorted rows ``ys`` (T K, D), with fp32 ``weights``
    (T, K). Dropped assignments add nothing, whatever their weights hold."""
    _check_rows("ys", ys, plan.slot.numel())
    if weights.shape != plan.slot.shape or weights.dtype != torch.float32:
        raise ValueError(f"weights must be fp32 of shape {tuple(plan.slot.shape)}, got {tuple(weights.shape)} {weights.dtype}")
    return _Combine.apply(ys.contiguous(), weights.contiguous(), plan.offsets, plan.slot)


# ------------------------------------------------------------------ products
def _planes(t: torch.Tensor) -> int:
    return 1 if t.dtype == torch.bfloat16 else 3 if precision.passes() == 3 else 2


def _operand(t: torch.Tensor, planes: int | None = None) -> torch.Tensor:
    """``t`` as the product kernels read it: bf16 planes first, rows 16-byte aligned. bf16 tensors laid out so already
    are used in place. A backward pass gives the forward's number of planes, whatever the precision is by then."""
    if t.dtype == torch.bfloat16 and t.stride(-1) == 1 and t.data_ptr() % 16 == 0:
        aligned = all(t.shape[d] <= 1 or (t.stride(d) % 8 == 0 and t.stride(d) > 0) for d in range(t.ndim - 1))
        if aligned and (t.shape[-2] <= 1 or t.stride(-2) >= t.shape[-1]):
            return t.unsqueeze(0)
    return ext().ragged_stage(t, planes or _planes(t))


def _cpu_spans(offsets: torch.Tensor) -> list[tuple[int, int]]:
    ends = offsets.tolist()
    return list(zip(ends[:-1], ends[1:]))


class _RaggedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, offsets):
        ctx.planes = _planes(x)
        ctx.save_for_backward(x, w, offsets)
        y = torch.empty(x.shape[0], w.shape[2], dtype=x.dtype, device=x.device)
        ext().ragged_rows([_operand(x)], [_operand(w)], offsets, y, False)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w, offsets = ctx.saved_tensors
        dx = dw = None
        dy = _operand(dy, ctx.planes)
        if ctx.needs_input_grad[0]:
            dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            ext().ragged_rows([dy], [_operand(w, ctx.planes)], offsets, dx, True)
        if ctx.needs_input_grad[1]:
            dw = torch.empty(w.shape, dtype=w.dtype, device=w.device)
            ext().ragged_weights(_operand(x, ctx.planes), [dy], offsets, [dw])
        return dx, dw, None


def _padded(planes: int | None, rows: int, cols: int, dtype: torch.dtype, device) -> torch.Tensor:
    """Empty ([planes,] rows, cols) whose rows start at 16-byte boundaries."""
    unit = 8 if dtype == torch.bfloat16 else 4
    shape = (rows, -(-cols // unit) * unit)
    t = torch.empty(shape if planes is None else (planes, *shape), dtype=dtype, device=device)
    return t if shape[1] == cols else t[..., :cols]


class _RaggedSwiGLU(torch.autograd.Function):
    """The kernels write h and the gradients of gate and up as the operands (bf16 planes) of the products that read
    them; the operands of x and h are kept for the backward in place of the tensors."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, offsets):
        rows, hidden, planes = x.shape[0], w_gate.shape[2], _planes(x)
        g, u = (_padded(None, rows, hidden, x.dtype, x.device) for _ in range(2))
        h = _padded(planes, rows, hidden, torch.bfloat16, x.device)
        y = torch.empty(rows, w_down.shape[2], dtype=x.dtype, device=x.device)
        x = _operand(x)
        ext().ragged_swiglu(x, _operand(w_gate), _operand(w_up), offsets, g, u, h)
        ext().ragged_rows([h], [_operand(w_down)], offsets, y, False)
        ctx.save_for_backward(x, w_gate, w_up, w_down, offsets, g, u, h)
        return y

    @staticmethod
    def backward(ctx, dy):
        x, w_gate, w_up, w_down, offsets, g, u, h = ctx.saved_tensors
        planes, (rows, hidden) = h.shape[0], g.shape
        dy = _operand(dy, planes)
        dg, du = (_padded(planes, rows, hidden, torch.bfloat16, dy.device) for _ in range(2))
        ext().ragged_swiglu_bwd(dy, _operand(w_down, planes), offsets, g, u, dg, du)
        grads = [None] * 5
        if ctx.needs_input_grad[0]:
            grads[0] = torch.empty(x.shape[1:], dtype=g.dtype, device=g.device)
            ext().ragged_rows([dg, du], [_operand(w_gate, planes), _operand(w_up, planes)], offsets, grads[0], True)
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            grads[1], grads[2] = (torch.empty(w.shape, dtype=w.dtype, device=w.device) for w in (w_gate, w_up))
            ext().ragged_weights(x, [dg, du], offsets, [grads[1], grads[2]])
        if ctx.needs_input_grad[3]:
            grads[3] = torch.empty(w_down.shape, dtype=w_down.dtype, device=w_down.device)
            ext().ragged_weights(h, [dy], offsets, [grads[3]])
        return tuple(g if need else None for g, need in zip(grads, ctx.needs_input_grad))


def _check_products(x: torch.Tensor, mats: dict[str, torch.Tensor], shapes: dict[str, tuple[int, int]], offsets: torch.Tensor) -> None:
    _check_rows("x", x)
    if offsets.ndim != 1 or offsets.numel() < 2 or offsets.dtype != torch.int32:
        raise ValueError(f"offsets must be int32 of shape (experts + 1,), got {tuple(offsets.shape)} {offsets.dtype}")
    experts = offsets.numel() - 1
    for name, w in mats.items():
        want = (experts, *shapes[name])
        if tuple(w.shape) != want or w.dtype != x.dtype:
            raise ValueError(f"{name} must be {x.dtype} of shape {want}, got {w.dtype} {tuple(w.shape)}")
        if w.device != x.device or offsets.device != x.device:
            raise ValueError("the rows, the matrices and the offsets must be on one device")
        if 0 in w.shape:
            raise ValueError(f"{name} has an empty dimension: {tuple(w.shape)}")


def ragged_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``y[r] = x[r] @ w[e]`` for the rows ``offsets[e] <= r < offsets[e + 1]`` of ``x`` (S, D), with ``w`` (E, D, N).

    ``offsets`` starts at 0 and does not decrease. Rows at or after ``offsets[E]`` belong to nobody: their ``y`` and
    gradient are zeros and they add nothing to ``w``'s gradient, whatever they hold."""
    if w.ndim != 3:
        raise ValueError(f"w must be (experts, in, out), got {tuple(w.shape)}")
    _check_products(x, {"w": w}, {"w": (x.shape[-1], w.shape[2])}, offsets)
    if not x.is_cuda:
        parts = [x[a:b] @ w[e] for e, (a, b) in enumerate(_cpu_spans(offsets))]
        return torch.cat([*parts, x.new_zeros(x.shape[0] - int(offsets[-1]), w.shape[2])])
    return _RaggedMatmul.apply(x, w, offsets.contiguous())


def ragged_swiglu_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``(silu(x Wg) * (x Wu)) Wd`` of each sorted row with its expert's matrices: ``x`` (S, D), ``w_gate`` and ``w_up``
    (E, D, H), ``w_down`` (E, H, D'). Offsets and rows that nobody owns as in ``ragged_matmul``."""
    if w_gate.ndim != 3 or w_down.ndim != 3:
        raise ValueError(f"the matrices must be (experts, in, out), got {tuple(w_gate.shape)} and {tuple(w_down.shape)}")
    d, hidden = x.shape[-1], w_gate.shape[2]
    _check_products(x, {"w_gate": w_gate, "w_up": w_up, "w_down": w_down},
                    {"w_gate": (d, hidden), "w_up": (d, hidden), "w_down": (hidden, w_down.shape[2])}, offsets)
    if not x.is_cuda:
        parts = [(torch.nn.functional.silu(x[a:b] @ w_gate[e]) * (x[a:b] @ w_up[e])) @ w_down[e]
                 for e, (a, b) in enumerate(_cpu_spans(offsets))]
        return torch.cat([*parts, x.new_zeros(x.shape[0] - int(offsets[-1]), w_down.shape[2])])
    return _RaggedSwiGLU.apply(x, w_gate, w_up, w_down, offsets.contiguous())
