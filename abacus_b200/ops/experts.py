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
bf16 operands are multiplied as they are. ``ragged_swiglu_mlp`` keeps gate and up in fp32 and rounds h = silu(gate) up and
the gradients of gate and up to bf16, because they are operands of bf16 products (the kernels for few rows keep them in
fp32 too). Sums are fp32 at any length; those over an expert's rows in bf16 are made of runs of 2^14 rows.

CUDA tensors run on ``csrc/experts`` and ``csrc/ops/expert_rows.cu`` (up to 256 experts for the products, 1024 for the
plan; differentiable once); CPU tensors run the formulas with ATen.
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
    if indices.is_cuda:
        return ExpertPlan(*ext().expert_plan(indices, n_experts))
    if indices.ndim != 2 or indices.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"indices must be a (tokens, choices) integer tensor, got {tuple(indices.shape)} {indices.dtype}")
    if n_experts < 1:
        raise ValueError(f"n_experts must be at least 1, got {n_experts}")
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


def dispatch_tokens(x: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """Rows of ``x`` (T, D) in the plan's order, one for each choice (T K, D); rows after the last expert's are zeros."""
    if x.is_cuda:
        return ext().expert_dispatch(x, plan.offsets, plan.slot)
    _check_rows("x", x, plan.slot.shape[0])
    t, k = torch.nonzero(plan.slot >= 0, as_tuple=True)
    return x.new_zeros(plan.slot.numel(), x.shape[1]).index_copy(0, plan.slot[t, k].long(), x.index_select(0, t))


def combine_tokens(ys: torch.Tensor, weights: torch.Tensor, plan: ExpertPlan) -> torch.Tensor:
    """``out[t] = sum_k weights[t, k] * ys[slot[t, k]]`` (T, D) of the sorted rows ``ys`` (T K, D), with fp32 ``weights``
    (T, K). Dropped assignments add nothing, whatever their weights hold."""
    if ys.is_cuda:
        return ext().expert_combine(ys, weights, plan.offsets, plan.slot)
    slot = plan.slot
    _check_rows("ys", ys, slot.numel())
    if weights.shape != slot.shape or weights.dtype != torch.float32:
        raise ValueError(f"weights must be fp32 of shape {tuple(slot.shape)}, got {tuple(weights.shape)} {weights.dtype}")
    t, k = torch.nonzero(slot >= 0, as_tuple=True)
    rows = ys.index_select(0, slot[t, k].long()).float() * weights[t, k, None]
    return rows.new_zeros(slot.shape[0], ys.shape[1]).index_add(0, t, rows).to(ys.dtype)


# ------------------------------------------------------------------ products
def _fp32_planes() -> int:
    return 3 if precision.passes() == 3 else 2


def _cpu_spans(offsets: torch.Tensor, rows: int) -> list[tuple[int, int]]:
    ends = offsets.tolist()
    if ends[0] != 0 or ends[-1] > rows or any(b < a for a, b in zip(ends[:-1], ends[1:])):
        raise ValueError(f"offsets must start at 0, not decrease and end within the {rows} rows, got {ends}")
    return list(zip(ends[:-1], ends[1:]))


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

    ``offsets`` starts at 0, does not decrease and ends within the rows: CPU tensors raise if not; on the GPU, where nobody
    waits for them, the device status says so (``_ext.check_status``), and the results are in bounds but say nothing. Rows at or after ``offsets[E]`` belong to nobody: their ``y`` and
    gradient are zeros and they add nothing to ``w``'s gradient, whatever they hold."""
    if x.is_cuda:
        return ext().ragged_matmul(x, w, offsets, _fp32_planes())
    if w.ndim != 3:
        raise ValueError(f"w must be (experts, in, out), got {tuple(w.shape)}")
    _check_products(x, {"w": w}, {"w": (x.shape[-1], w.shape[2])}, offsets)
    parts = [x[a:b] @ w[e] for e, (a, b) in enumerate(_cpu_spans(offsets, x.shape[0]))]
    return torch.cat([*parts, x.new_zeros(x.shape[0] - int(offsets[-1]), w.shape[2])])


def ragged_swiglu_mlp(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    """``(silu(x Wg) * (x Wu)) Wd`` of each sorted row with its expert's matrices: ``x`` (S, D), ``w_gate`` and ``w_up``
    (E, D, H), ``w_down`` (E, H, D'). Offsets and rows that nobody owns as in ``ragged_matmul``."""
    if x.is_cuda:
        return ext().ragged_swiglu_mlp(x, w_gate, w_up, w_down, offsets, _fp32_planes())
    if w_gate.ndim != 3 or w_down.ndim != 3:
        raise ValueError(f"the matrices must be (experts, in, out), got {tuple(w_gate.shape)} and {tuple(w_down.shape)}")
    d, hidden = x.shape[-1], w_gate.shape[2]
    _check_products(x, {"w_gate": w_gate, "w_up": w_up, "w_down": w_down},
                    {"w_gate": (d, hidden), "w_up": (d, hidden), "w_down": (hidden, w_down.shape[2])}, offsets)
    parts = [(torch.nn.functional.silu(x[a:b] @ w_gate[e]) * (x[a:b] @ w_up[e])) @ w_down[e]
             for e, (a, b) in enumerate(_cpu_spans(offsets, x.shape[0]))]
    return torch.cat([*parts, x.new_zeros(x.shape[0] - int(offsets[-1]), w_down.shape[2])])
