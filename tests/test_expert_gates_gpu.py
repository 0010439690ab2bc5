"""SwiGLU experts element by element over gates from -30 to 30, in fp32, against 64 bits.

Matrices of zeros and ones make gate = x0, up = x1 and y = h, and three bf16 parts carry such products without an error.
What is left in silu(g): one unit in the last place of the exponential (2^-23) and two of the quotient, a rounding of
2^-24 each of 1 + e, two products, and of adding the parts of the result up (three): 12 times 2^-24. In the derivative
sig (1 + g (1 - sig)) the roundings of sig come back times g, and the terms may cancel, so its error goes by
sig (1 + |g|) instead of by its size: a factor of two on the same count covers both appearances of sig.
"""
import pytest
import torch

from abacus_b200.ops import experts, precision

pytestmark = pytest.mark.gpu

BOUND = 12 * 2.0**-24


@pytest.mark.parametrize("rows", [8, 2000])  # the kernels for few rows, and the tensor cores
def test_gates_in_fp32(rows):
    precision.set_precision("fp32")
    gate = torch.linspace(-30, 30, rows, device="cuda")
    x = torch.zeros(rows, 8, device="cuda")
    x[:, 0], x[:, 1] = gate, 1.0
    mats = [torch.zeros(1, 8, 8, device="cuda") for _ in range(3)]
    mats[0][0, 0], mats[1][0, 1], mats[2][0, 0, 0] = 1.0, 1.0, 1.0
    x.requires_grad_()
    y = experts.ragged_swiglu_mlp(x, *mats, torch.tensor([0, rows], dtype=torch.int32, device="cuda"))
    dy = torch.zeros_like(y)
    dy[:, 0] = 1.0
    (dx,) = torch.autograd.grad(y, x, dy)
    g = gate.double()
    sig = 1 / (1 + torch.exp(-g))
    silu = g * sig
    assert torch.all((y[:, 0].double() - silu).abs() <= BOUND * silu.abs())
    # Column 0 of h alone reaches y, so its gate's and its up's gradients are those of x0 and x1.
    assert torch.all((dx[:, 1].double() - silu).abs() <= BOUND * silu.abs())
    assert torch.all((dx[:, 0].double() - sig * (1 + g * (1 - sig))).abs() <= 2 * BOUND * sig * (1 + g.abs()))
