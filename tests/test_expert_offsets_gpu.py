"""Offsets that do not start at 0, decrease, or end after the rows: the device status names them, whichever kernels run.

The kernels keep inside their tensors: every offset that they use is cut to the rows.
"""
import pytest
import torch

from abacus_b200.ops import experts
from abacus_b200.ops._ext import check_status, ext

pytestmark = pytest.mark.gpu


def _bad(rows):
    t = rows // 4
    return {"late start": [t, 2 * t, 3 * t, rows], "decrease": [0, 3 * t, t, rows], "past the rows": [0, t, 2 * t, rows + 7],
            "negative": [0, -5, t, rows]}


def _status():
    torch.cuda.synchronize()
    try:
        check_status()
    except RuntimeError as error:
        return str(error)
    return "healthy"


@pytest.fixture(autouse=True)
def _healthy_before_and_after():
    assert _status() == "healthy"
    yield
    _status()


@pytest.mark.parametrize("kind", ["late start", "decrease", "past the rows", "negative"])
@pytest.mark.parametrize("dtype,rows", [(torch.float32, 20), (torch.bfloat16, 20), (torch.float32, 600), (torch.bfloat16, 600)])
def test_bad_offsets_are_reported(kind, dtype, rows):
    offsets = torch.tensor(_bad(rows)[kind], dtype=torch.int32, device="cuda")
    x, dy = (torch.randn(rows, n, device="cuda").to(dtype) for n in (64, 40))
    w = torch.randn(3, 64, 40, device="cuda").to(dtype).requires_grad_()
    y = experts.ragged_matmul(x, w, offsets)
    assert "status 6" in _status()
    # The weight gradient looks at them too.
    (dw,) = torch.autograd.grad(y, w, dy)
    assert "status 6" in _status()
    assert y.shape == (rows, 40) and dw.shape == w.shape


def test_good_offsets_are_not():
    for rows in (20, 600):
        for ends in ([0, 0, 0, 0], [0, rows, rows, rows], [0, 5, 5, rows - 3]):
            x = torch.randn(rows, 64, device="cuda", requires_grad=True)
            w = torch.randn(3, 64, 40, device="cuda", requires_grad=True)
            y = experts.ragged_matmul(x, w, torch.tensor(ends, dtype=torch.int32, device="cuda"))
            torch.autograd.grad(y.sum(), (x, w))
            assert _status() == "healthy"
    assert ext().read_status(0) == 0
