"""The SwiGLU experts where the other tests do not go: as many experts as there may be, two bf16 parts, and how many
roundings a bf16 result holds. Against 64 bits, as 2-norms of the difference over the result's.

bf16: gate and up stay in fp32; h and the gradients of gate and up are rounded to bf16 once, each result once. A rounding
moves a number by 2^-8 at most, uniformly, so 2^-8 / sqrt(3) in the norm at worst, and two of them 2^-8 sqrt(2 / 3); sums
whose terms partly cancel show the first one larger, for which a tenth is added. fp32: 2e-6 a product in three parts, 2^-15
in two, and at most four in a row (a gradient of x has gate or up, the derivative through down, and itself).
"""
import pytest
import torch

from abacus_b200.ops import experts, precision
from abacus_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu

BOUND = {"bf16": 1.1 * 2.0**-8 * (2 / 3) ** 0.5, "fp32": 4 * 2e-6, "tf32": 4 * 2.0**-15}
COUNTS = {
    "256 experts, short": [(7 * i) % 11 for i in range(256)],
    "256 experts, tiles of one CTA": [(37 * i) % 311 for i in range(256)],
    "256 experts, tiles of two": [(53 * i) % 601 for i in range(256)],
    "256 experts, most rows in one": [3] * 100 + [2000] + [1] * 155,
    "few experts": [700, 0, 90],
}


@pytest.fixture(autouse=True)
def _healthy():
    yield
    precision.set_precision("fp32")
    torch.cuda.synchronize()
    check_status()


@pytest.mark.parametrize("kind", ["bf16", "fp32", "tf32"])
@pytest.mark.parametrize("counts", COUNTS.values(), ids=COUNTS.keys())
@pytest.mark.parametrize("d,hidden", [(72, 88), (264, 136)])
def test_swiglu_mlp_and_gradients(kind, counts, d, hidden):
    precision.set_precision("tf32" if kind == "tf32" else "fp32")
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    g = torch.Generator(device="cuda").manual_seed(d)
    rows, e = sum(counts), len(counts)
    x = torch.randn(rows, d, device="cuda", generator=g).to(dtype).requires_grad_()
    shapes = ((d, hidden), (d, hidden), (hidden, d))
    mats = [(torch.randn(e, *s, device="cuda", generator=g) * s[0] ** -0.5).to(dtype).requires_grad_() for s in shapes]
    dy = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    ends = torch.tensor([0] + counts).cumsum(0)
    xd, md = x.detach().double().requires_grad_(), [m.detach().double().requires_grad_() for m in mats]
    parts = []
    for i, (a, b) in enumerate(zip(ends[:-1].tolist(), ends[1:].tolist())):
        parts.append((torch.nn.functional.silu(xd[a:b] @ md[0][i]) * (xd[a:b] @ md[1][i])) @ md[2][i])
    want = torch.cat(parts)
    want = [want.detach(), *torch.autograd.grad(want, (xd, *md), dy.double())]
    y = experts.ragged_swiglu_mlp(x, *mats, ends.to("cuda", torch.int32))
    for got, exact in zip([y.detach(), *torch.autograd.grad(y, (x, *mats), dy)], want):
        assert float((got.double() - exact).norm()) <= BOUND[kind] * float(exact.norm())
