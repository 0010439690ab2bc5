"""Dropless expert operators on CPU: plan, rows, products, and what they refuse."""
import pytest
import torch

from abacus_b200.ops import experts


def _plan_by_hand(indices, n_experts):
    rows = [(e if 0 <= e < n_experts else n_experts, i) for i, e in enumerate(indices.reshape(-1).tolist())]
    order = [i for _, i in sorted(rows)]
    offsets = [sum(1 for e, _ in rows if e < k) for k in range(n_experts + 1)]
    slot = [0] * len(rows)
    for place, i in enumerate(order):
        slot[i] = place if rows[i][0] < n_experts else -1
    return offsets, order, slot


@pytest.mark.parametrize("tokens,choices,n_experts", [(0, 2, 3), (1, 1, 1), (7, 3, 5), (50, 2, 4)])
def test_plan_is_the_stable_sort(tokens, choices, n_experts):
    g = torch.Generator().manual_seed(tokens)
    indices = torch.randint(-1, n_experts + 1, (tokens, choices), generator=g)
    plan = experts.expert_plan(indices, n_experts)
    offsets, order, slot = _plan_by_hand(indices, n_experts)
    assert plan.offsets.tolist() == offsets and plan.order.tolist() == order and plan.slot.reshape(-1).tolist() == slot


def test_dispatch_and_combine_match_their_formulas_and_differences():
    g = torch.Generator().manual_seed(1)
    indices = torch.randint(-1, 3, (6, 2), generator=g)
    plan = experts.expert_plan(indices, 3)
    x = torch.randn(6, 5, generator=g, requires_grad=True)
    w = torch.rand(6, 2, generator=g, requires_grad=True)
    ys = torch.randn(12, 5, generator=g, requires_grad=True)
    xs = experts.dispatch_tokens(x, plan)
    out = experts.combine_tokens(ys, w, plan)
    for t in range(6):
        want = torch.zeros(5)
        for k in range(2):
            s = plan.slot[t, k]
            if s >= 0:
                assert torch.equal(xs[s], x[t])
                want = want + w[t, k] * ys[s]
        torch.testing.assert_close(out[t], want)
    assert torch.all(xs[int(plan.offsets[-1]):] == 0)
    dxs, dout = torch.randn(12, 5, generator=g), torch.randn(6, 5, generator=g)
    grads = torch.autograd.grad((xs, out), (x, ys, w), (dxs, dout))

    def loss(x_, ys_, w_):
        return (experts.dispatch_tokens(x_, plan) * dxs).sum().double() + (experts.combine_tokens(ys_, w_, plan) * dout).sum().double()

    # The loss is linear in each input, so a difference is exact up to fp32 rounding of the loss: 1e-6 of its size over the step.
    for which, grad in enumerate(grads):
        direction = torch.randn(grad.shape, generator=g)
        args = [x.detach(), ys.detach(), w.detach()]
        up, down = list(args), list(args)
        up[which], down[which] = args[which] + direction, args[which] - direction
        assert abs(float((loss(*up) - loss(*down)) / 2 - (grad * direction).sum())) < 1e-4


@pytest.mark.parametrize("counts,idle", [([3, 0, 4], 2), ([0, 0], 3), ([5], 0)])
def test_products_on_cpu(counts, idle):
    g = torch.Generator().manual_seed(2)
    offsets = torch.tensor([0] + counts).cumsum(0).to(torch.int32)
    rows, e = sum(counts) + idle, len(counts)
    x = torch.randn(rows, 4, generator=g, dtype=torch.float32, requires_grad=True)
    w = torch.randn(e, 4, 6, generator=g, requires_grad=True)
    y = experts.ragged_matmul(x, w, offsets)
    owner = [i for i, c in enumerate(counts) for _ in range(c)]
    for r in range(rows):
        want = x[r] @ w[owner[r]] if r < len(owner) else torch.zeros(6)
        torch.testing.assert_close(y[r], want)
    y.sum().backward()
    assert torch.all(x.grad[len(owner):] == 0)
    wd = torch.randn(e, 6, 4, generator=g)
    z = experts.ragged_swiglu_mlp(x, w, w, wd, offsets)
    for r in range(rows):
        if r < len(owner):
            a = x[r] @ w[owner[r]]
            torch.testing.assert_close(z[r], (torch.nn.functional.silu(a) * a) @ wd[owner[r]])
        else:
            assert torch.all(z[r] == 0)


def test_refusals():
    x, w, off = torch.zeros(4, 8), torch.zeros(2, 8, 3), torch.tensor([0, 2, 4], dtype=torch.int32)
    with pytest.raises(ValueError, match="indices"):
        experts.expert_plan(torch.zeros(4, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match="indices"):
        experts.expert_plan(torch.zeros(4, 1), 2)
    with pytest.raises(ValueError, match="n_experts"):
        experts.expert_plan(torch.zeros(4, 1, dtype=torch.int64), 0)
    plan = experts.expert_plan(torch.zeros(4, 1, dtype=torch.int64), 2)
    with pytest.raises(ValueError, match="rows"):
        experts.dispatch_tokens(torch.zeros(5, 8), plan)
    with pytest.raises(ValueError, match="2-D"):
        experts.dispatch_tokens(torch.zeros(4, 8, dtype=torch.float64), plan)
    with pytest.raises(ValueError, match="weights"):
        experts.combine_tokens(x, torch.zeros(4, 2), plan)
    with pytest.raises(ValueError, match="weights"):
        experts.combine_tokens(x, torch.zeros(4, 1, dtype=torch.bfloat16), plan)
    with pytest.raises(ValueError, match="offsets"):
        experts.ragged_matmul(x, w, off.long())
    with pytest.raises(ValueError, match="w must be"):
        experts.ragged_matmul(x, w.bfloat16(), off)
    with pytest.raises(ValueError, match="w must be"):
        experts.ragged_matmul(x, torch.zeros(3, 8, 3), off)
    with pytest.raises(ValueError, match="w must be"):
        experts.ragged_matmul(x, torch.zeros(8, 3), off)
    with pytest.raises(ValueError, match="empty"):
        experts.ragged_matmul(x, torch.zeros(2, 8, 0), off)
    with pytest.raises(ValueError, match="w_down"):
        experts.ragged_swiglu_mlp(x, w, w, torch.zeros(2, 4, 8), off)
