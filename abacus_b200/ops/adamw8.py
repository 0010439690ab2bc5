"""AdamW over many tensors with both moments in 8 bits.

The moments of a tensor are four flat tensors: ``exp_avg`` and ``exp_rms`` (the
root of the second moment), ``float8_e4m3fn`` with the tensor's number of
elements, and for each of them one fp32 scale per 256 consecutive elements, a
power of two. A step is

    m <- b1 m + (1 - b1) g
    u <- sqrt(b2 u^2 + (1 - b2) g^2)
    w <- w (1 - lr wd) - lr / (1 - b1^t) * m / (u / sqrt(1 - b2^t) + eps)

in fp32, after which m and u are rounded to 8 bits stochastically, with random
bits that an integer hash makes of (element number in the tensor, step): the
same inputs give the same outputs. CPU and GPU take the same random bits; their
moments agree but for a code in a million or so, their weights to fp32's rounding.
A second moment that is not zero never rounds to zero. A gradient that is
infinite or NaN spoils its own element (moments NaN, as in 32 bits), not its block.

The price of one scale for 256 elements: an element whose u is below some 2^-17
of its block's largest is held at the smallest code, which is larger than what
it stands for, and moves by that much less than it would with 32-bit moments
(gradients of 1e-7 among one of 1: 0.0025 in 200 steps of 1e-3 in place of 0.18).

CUDA tensors run on ``csrc/ops/adamw8_kernel.cu`` (one launch for up to 128 tensors);
CPU tensors run the formulation below.
"""
from __future__ import annotations

import math

import torch

from abacus_b200.ops._ext import ext

BLOCK = 256
_MASK32 = 0xFFFFFFFF


def fresh_state(numel: int, device) -> dict[str, torch.Tensor]:
    """Zero moments of a tensor with ``numel`` elements."""
    blocks = -(-numel // BLOCK)
    code = lambda: torch.zeros(numel, dtype=torch.float8_e4m3fn, device=device)  # noqa: E731
    scale = lambda: torch.zeros(blocks, dtype=torch.float32, device=device)  # noqa: E731
    return {"exp_avg": code(), "exp_avg_scale": scale(), "exp_rms": code(), "exp_rms_scale": scale()}


def _blocks(flat: torch.Tensor) -> torch.Tensor:
    """(blocks, 256), the last block filled up with zeros."""
    missing = -flat.numel() % BLOCK
    return torch.nn.functional.pad(flat, (0, missing)).view(-1, BLOCK)


def dequantize(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """The fp32 values (flat) that codes and scales stand for."""
    return (_blocks(codes.reshape(-1).float()) * scale[:, None]).reshape(-1)[: codes.numel()]


def _scales(blocks: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(scale, 1 / scale) that bring each block's largest finite magnitude into [128, 256)."""
    largest = torch.where(torch.isfinite(blocks), blocks.abs(), 0.0).amax(1)
    exponent = ((largest.view(torch.int32) >> 23) - 7).clamp(min=1)
    return (exponent << 23).view(torch.float32), ((254 - exponent) << 23).view(torch.float32)


def quantize(values: torch.Tensor, positive: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of fp32 values, rounded to nearest: what a checkpoint's 32-bit moments become. With ``positive``
    (second moments) no value that is not zero becomes zero."""
    blocks = _blocks(values.reshape(-1).float())
    scale, inverse = _scales(blocks)
    scaled = blocks * inverse[:, None]
    if positive:
        scaled = torch.where(scaled > 0, scaled.clamp(min=2.0**-9), scaled)
    # Infinities become NaN, as in a step (the conversion alone would depend on the device).
    codes = torch.where(torch.isfinite(blocks), scaled, math.nan).to(torch.float8_e4m3fn)
    return codes.reshape(-1)[: values.numel()].clone(), scale


def _noise(numel: int, step: int, device) -> torch.Tensor:
    x = torch.arange(numel, device=device) * 0x9E3779B1 + step * 0x7F4A7C15 & _MASK32
    x = ((x ^ (x >> 16)) * 0x6C62272F) & _MASK32
    x = ((x ^ (x >> 15)) * 0x2F0B4C47) & _MASK32
    return x ^ (x >> 16)


def _stochastic(blocks: torch.Tensor, noise16: torch.Tensor, positive: bool) -> tuple[torch.Tensor, torch.Tensor]:
    scale, inverse = _scales(blocks)
    a = blocks.abs() * inverse[:, None]
    base = torch.where(a < 2.0**-6, 2.0**-6, 0.0)
    bits = (a + base).view(torch.int32) + (noise16 << 4).to(torch.int32)
    q = (bits & -(1 << 20)).view(torch.float32) - base
    if positive:
        q = torch.where(a > 0, q.clamp(min=2.0**-9), q)
    q = torch.where(torch.isfinite(blocks), torch.copysign(q, blocks), math.nan)
    return q.to(torch.float8_e4m3fn), scale


def _step_cpu(w, g, m, m_scale, u, u_scale, lr, beta1, beta2, eps, weight_decay, step):
    n = w.numel()
    grad = g.reshape(-1).float()
    m_new = dequantize(m, m_scale) * beta1 + grad * (1 - beta1)
    u_old = dequantize(u, u_scale)
    u_new = torch.sqrt(u_old * u_old * beta2 + grad * grad * (1 - beta2))
    ratio = m_new / (u_new / math.sqrt(1 - beta2**step) + eps)
    flat = w.view(-1)
    flat.copy_(flat * (1 - lr * weight_decay) - ratio * (lr / (1 - beta1**step)))
    noise = _noise(-(-n // BLOCK) * BLOCK, step, w.device).view(-1, BLOCK)
    for value, bits, codes, scale, positive in ((m_new, noise & 0xFFFF, m, m_scale, False), (u_new, noise >> 16, u, u_scale, True)):
        q, new_scale = _stochastic(_blocks(value), bits, positive)
        codes.view(-1).copy_(q.reshape(-1)[:n])
        scale.copy_(new_scale)


@torch.no_grad()
def step_(
    weights: list[torch.Tensor],
    grads: list[torch.Tensor],
    exp_avg: list[torch.Tensor],
    exp_avg_scale: list[torch.Tensor],
    exp_rms: list[torch.Tensor],
    exp_rms_scale: list[torch.Tensor],
    *,
    lr: float,
    betas: tuple[float, float] = (0.9, 0.999),
    eps: float = 1e-8,
    weight_decay: float = 1e-2,
    step: int,
) -> None:
    """One step of every tensor, in place. ``step`` counts from 1. Weights are
    contiguous fp32 tensors, gradients contiguous fp32 or bf16 ones; the
    moments are laid out as ``fresh_state`` lays them out."""
    lists = (weights, grads, exp_avg, exp_avg_scale, exp_rms, exp_rms_scale)
    if len({len(x) for x in lists}) != 1:
        raise ValueError(f"adamw8: the lists differ in length: {[len(x) for x in lists]}")
    if step < 1:
        raise ValueError(f"adamw8: step must be at least 1, got {step}")
    if not weights:
        return
    if weights[0].is_cuda:
        ext().adamw8_step(*lists, float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay), int(step))
        return
    for w, g, m, ms, u, us in zip(*lists):
        n = w.numel()
        blocks = -(-n // BLOCK)
        if w.dtype != torch.float32 or m.dtype != torch.float8_e4m3fn or u.dtype != torch.float8_e4m3fn:
            raise ValueError("adamw8: fp32 weights and float8_e4m3fn moments are needed")
        if g.numel() != n or m.numel() != n or u.numel() != n or ms.numel() != blocks or us.numel() != blocks:
            raise ValueError(f"adamw8: sizes of a tensor ({n} weights need {blocks} scales of each moment)")
    for tensors in zip(*lists):
        if tensors[0].numel():
            _step_cpu(*tensors, lr, *betas, eps, weight_decay, step)
