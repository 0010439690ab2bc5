"""AdamW with 8-bit moments (CPU formulation): definition, statistics of its rounding, refusals."""
import math

import pytest
import torch

from abacus_b200.ops import adamw8


def _tensor(n, seed, kind=torch.float32):
    g = torch.Generator().manual_seed(seed)
    w, grad = torch.randn(n, generator=g), torch.randn(n, generator=g).to(kind)
    return w, grad, adamw8.fresh_state(n, "cpu")


def _step(w, grad, st, step, **kw):
    adamw8.step_([w], [grad], [st["exp_avg"]], [st["exp_avg_scale"]], [st["exp_rms"]], [st["exp_rms_scale"]], lr=1e-3, step=step, **kw)


@pytest.mark.parametrize("n", [1, 255, 256, 257, 1000])
def test_first_step_is_adamw_and_moments_are_neighbours_on_the_grid(n):
    w, grad, st = _tensor(n, n)
    before = w.double()
    _step(w, grad, st, 1, weight_decay=0.1)
    g = grad.double()
    want = before * (1 - 1e-3 * 0.1) - 1e-3 * g / (g.abs() + 1e-8)
    torch.testing.assert_close(w.double(), want, rtol=1e-6, atol=1e-6)
    for key, value in (("exp_avg", 0.1 * g), ("exp_rms", (0.001 * g * g).sqrt())):
        scale = st[key + "_scale"].double().repeat_interleave(256)[:n]
        got = st[key].double() * scale
        # e4m3 steps are 2^-3 of the power of two below a number, and never under 2^-9 of the scale.
        a = value.abs() / scale
        grid = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0**-6))) - 3)
        assert torch.all((got.abs() / scale - a).abs() <= grid * 1.0001)
        for b in range(0, n, 256):
            top = (value[b : b + 256].abs() / scale[b]).max()
            assert 127.99 <= top < 256.01


def test_rounding_is_unbiased_over_steps():
    """A constant gradient keeps m at its value on average: 4000 steps' mean error is below 4 standard errors, each step's
    rounding being off by at most a grid step (2^-3 relative, variance at most 2^-8)."""
    n = 256
    w, grad, st = _tensor(n, 0)
    grad = grad.abs() + 0.5
    total = torch.zeros(n, dtype=torch.float64)
    for step in range(1, 4001):
        value = adamw8.dequantize(st["exp_avg"], st["exp_avg_scale"]) * 0.9 + grad * 0.1
        _step(w, grad, st, step)
        total += (adamw8.dequantize(st["exp_avg"], st["exp_avg_scale"]) - value).double() / value.double()
    assert float(total.abs().max() / 4000) < 4 * 2**-4 / math.sqrt(4000)


def test_second_moment_decays_to_a_smaller_gradient():
    """With beta2 = 0.999 a step moves the root of the second moment by a two-thousandth, far less than half of an e4m3
    step. After 3000 steps at a hundredth of the first gradient it follows all the same: sqrt(0.999^3000) = 0.223."""
    n = 512
    w, grad, st = _tensor(n, 1)
    big = torch.ones(n)
    for step in range(1, 401):
        _step(w, big, st, step)
    start = adamw8.dequantize(st["exp_rms"], st["exp_rms_scale"]).mean()
    for step in range(401, 3401):
        _step(w, big * 0.01, st, step)
    ratio = float(adamw8.dequantize(st["exp_rms"], st["exp_rms_scale"]).mean() / start)
    assert 0.19 < ratio < 0.26


def test_training_follows_32_bit_moments():
    """A least-squares fit ends where AdamW with 32-bit moments ends."""
    g = torch.Generator().manual_seed(2)
    a, target = torch.randn(512, 64, generator=g), torch.randn(512, generator=g)
    ends = {}
    for bits in (8, 32):
        w = torch.zeros(64)
        st = adamw8.fresh_state(64, "cpu")
        ref = torch.optim.AdamW([w], lr=2e-3, weight_decay=0.0)
        for step in range(1, 1501):
            grad = a.t() @ (a @ w - target) / 512
            if bits == 8:
                adamw8.step_([w], [grad], [st["exp_avg"]], [st["exp_avg_scale"]], [st["exp_rms"]], [st["exp_rms_scale"]],
                             lr=2e-3, weight_decay=0.0, step=step)
            else:
                w.grad = grad
                ref.step()
        ends[bits] = float(((a @ w - target) ** 2).mean())
    assert abs(ends[8] - ends[32]) < 0.01 * ends[32]


def test_zero_infinite_and_nan_gradients():
    w, grad, st = _tensor(600, 3)
    grad[:256] = 0
    grad[300], grad[301] = float("inf"), float("nan")
    before = w.clone()
    _step(w, grad, st, 1, weight_decay=0.0)
    assert torch.equal(w[:256], before[:256]) and torch.all(st["exp_avg"][:256].float() == 0) and torch.all(st["exp_rms"][:256].float() == 0)
    bad = torch.zeros(600, dtype=torch.bool)
    bad[300] = bad[301] = True
    assert torch.isnan(st["exp_avg"].float()[bad]).all() and torch.isnan(st["exp_rms"].float()[bad]).all()
    assert torch.isfinite(w[~bad]).all() and torch.isfinite(st["exp_avg"].float()[~bad]).all()


def test_second_moments_do_not_vanish():
    """An element a millionth of its block's largest keeps a second moment: the next step divides by it."""
    w, grad, st = _tensor(256, 4)
    grad = torch.full((256,), 1e-6)
    grad[0] = 1.0
    for step in range(1, 6):
        _step(w, grad, st, step)
        assert torch.all(st["exp_rms"].float() > 0)


def test_quantize_keeps_what_is_representable():
    g = torch.Generator().manual_seed(5)
    codes, scale = adamw8.quantize(torch.randn(1000, generator=g))
    values = adamw8.dequantize(codes, scale)
    again, scale2 = adamw8.quantize(values)
    assert torch.equal(adamw8.dequantize(again, scale2), values)
    assert torch.isnan(adamw8.quantize(torch.tensor([float("inf"), 1.0]))[0].float()[0])


def test_refusals():
    w, grad, st = _tensor(300, 6)
    args = ([w], [grad], [st["exp_avg"]], [st["exp_avg_scale"]], [st["exp_rms"]], [st["exp_rms_scale"]])
    with pytest.raises(ValueError, match="step"):
        adamw8.step_(*args, lr=1e-3, step=0)
    with pytest.raises(ValueError, match="length"):
        adamw8.step_(args[0], [], *args[2:], lr=1e-3, step=1)
    with pytest.raises(ValueError, match="scales"):
        adamw8.step_(*args[:3], [st["exp_avg_scale"][:1]], *args[4:], lr=1e-3, step=1)
    with pytest.raises(ValueError, match="float8"):
        adamw8.step_(*args[:2], [w.clone()], *args[3:], lr=1e-3, step=1)
