"""Weight gradients of an expert with very many rows: the sum over its rows is an fp32 sum at any length.

A run of 2^14 rows stays in an accumulator that truncates: each of its 2^10 sixteen-row steps loses below one unit in the
last place, 2^-23 of what is there by then, half of the end's on average, so a run's mean error is below 2^-14 and the
runs' sum adds 2^-24 a run. A bf16 result is then rounded once, by 2^-8 at most and without a bias. The mean over the
outputs, which random signs of the rounding leave 4 standard errors of 2^-8 / sqrt(3) uncertain, shows the truncation.
"""
import pytest
import torch

from abacus_b200.ops import experts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,n", [(256, 264), (96, 96)])  # tiles of two CTAs and of one
@pytest.mark.parametrize("rows", [(1 << 14) - 1, (1 << 14) + 1, 1 << 17, (1 << 20) + 100])
def test_sums_of_positive_numbers(d, n, rows):
    g = torch.Generator(device="cuda").manual_seed(rows)
    # Columns of different scales, so that the results spread over the numbers between two powers of two.
    x = ((torch.rand(rows, d, device="cuda", generator=g) + 0.5) * (1 + torch.rand(d, device="cuda", generator=g))).bfloat16()
    dy = ((torch.rand(rows, n, device="cuda", generator=g) + 0.5) * (1 + torch.rand(n, device="cuda", generator=g))).bfloat16()
    w = torch.zeros(2, d, n, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    offsets = torch.tensor([0, 37, rows], dtype=torch.int32, device="cuda")
    (dw,) = torch.autograd.grad(experts.ragged_matmul(x, w, offsets), w, dy)
    want = torch.zeros(d, n, dtype=torch.float64, device="cuda")
    for a in range(37, rows, 1 << 16):
        want += x[a : a + (1 << 16)].double().t() @ dy[a : a + (1 << 16)].double()
    off = dw[1].double() / want - 1
    assert float(off.abs().max()) <= 2.0**-8 + 2.0**-13
    assert abs(float(off.mean())) <= 2.0**-14 + 4 * 2.0**-8 / (3 * d * n) ** 0.5
    (again,) = torch.autograd.grad(experts.ragged_matmul(x, w, offsets), w, dy)
    assert torch.equal(again, dw)


@pytest.mark.parametrize("counts", [[40000, 0, 16384, 16448, 20, 70001], [(1 << 15) + 64, 1 << 15]])
def test_experts_of_different_lengths(counts):
    """Tiles of one run and of several in one launch, random signs: one rounding to bf16 and the truncation above."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, d, n = sum(counts), 300, 520
    x = torch.randn(rows, d, device="cuda", generator=g).bfloat16()
    dy = torch.randn(rows, n, device="cuda", generator=g).bfloat16()
    w = torch.zeros(len(counts), d, n, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ends = torch.tensor([0] + counts).cumsum(0)
    (dw,) = torch.autograd.grad(experts.ragged_matmul(x, w, ends.to("cuda", torch.int32)), w, dy)
    for e, (a, b) in enumerate(zip(ends[:-1].tolist(), ends[1:].tolist())):
        want = x[a:b].double().t() @ dy[a:b].double()
        assert float((dw[e].double() - want).norm()) <= (2.0**-8 + 2.0**-13) * float(want.norm())
