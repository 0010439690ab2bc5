"""Layouts of the rows that the expert operators take, against their contiguous copies."""
import pytest
import torch

from abacus_b200.ops import experts

pytestmark = pytest.mark.gpu


def _grads(out, inputs, gradient):
    return torch.autograd.grad(out, inputs, gradient)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 300])
def test_rows_of_one_column(dtype, tokens):
    """A row seen through a transpose is contiguous, with a stride of its length between columns that are not there."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    plan = experts.expert_plan(torch.randint(-1, 4, (tokens, 2), device="cuda", generator=g), 4)

    def column(n):
        t = torch.randn(1, n, device="cuda", generator=g).to(dtype).t()
        assert t.stride() == (1, n)
        return t

    x, ys, w = column(tokens), column(2 * tokens), torch.rand(tokens, 2, device="cuda", generator=g)
    dxs, dout = column(2 * tokens), column(tokens)
    both = []
    for plain in (False, True):
        view = (lambda t: t.reshape(-1).clone().view(-1, 1)) if plain else (lambda t: t)
        a, b, c = (view(t).detach().requires_grad_() if t is not w else w.clone().requires_grad_() for t in (x, ys, w))
        xs, out = experts.dispatch_tokens(a, plan), experts.combine_tokens(b, c, plan)
        both.append((xs, out, *_grads((xs, out), (a, b, c), (view(dxs), view(dout)))))
    for got, want in zip(*both):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [3, 500])
def test_products_of_one_column(dtype, rows):
    g = torch.Generator(device="cuda").manual_seed(rows)
    offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
    x, dy = (torch.randn(1, rows, device="cuda", generator=g).to(dtype).t() for _ in range(2))
    w = torch.randn(2, 1, 1, device="cuda", generator=g).to(dtype)
    both = []
    for plain in (False, True):
        view = (lambda t: t.reshape(-1).clone().view(-1, 1)) if plain else (lambda t: t)
        a, b = view(x).detach().requires_grad_(), w.clone().requires_grad_()
        y = experts.ragged_matmul(a, b, offsets)
        both.append((y, *_grads(y, (a, b), view(dy))))
    for got, want in zip(*both):
        assert torch.equal(got, want)
