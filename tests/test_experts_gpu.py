"""Dropless expert operators on the GPU against plain formulas in 64 bits.

Tolerances, as 2-norms of the difference over the 2-norm of the result. A bf16 result is rounded once: at most 2^-8
relative an element. The SwiGLU experts round gate, up, h and the gradients of gate and up to bf16 on the way (2^-8
each, independent), so six times 2^-8 bounds their sums. fp32 products of three planes drop 2^-25 of a product and add
with one rounding per 64-deep chunk plus the chunk's own truncation, below 2e-6 of the result's norm at these lengths;
two planes drop 2^-16 of it. Row sums of a few terms are rounded 2^-24 a term.
"""
import pytest
import torch

from abacus_b200.ops import experts, precision
from abacus_b200.ops._ext import check_status

pytestmark = pytest.mark.gpu

BF16 = 2.0**-8


@pytest.fixture(autouse=True)
def _healthy():
    yield
    precision.set_precision("fp32")
    torch.cuda.synchronize()
    check_status()


def _off(got, want):
    assert got.shape == want.shape
    want = want.double()
    norm = want.norm().item()
    diff = (got.double() - want).norm().item()
    return diff / norm if norm else diff


def _offsets(counts):
    return torch.tensor([0] + list(counts)).cumsum(0).to(device="cuda", dtype=torch.int32)


def _spans(counts):
    ends = torch.tensor([0] + list(counts)).cumsum(0).tolist()
    return list(enumerate(zip(ends[:-1], ends[1:])))


def _exact_products(x, w, dy, counts):
    x, w, dy = x.double(), w.double(), dy.double()
    y, dx, dw = x.new_zeros(x.shape[0], w.shape[2]), torch.zeros_like(x), torch.zeros_like(w)
    for e, (a, b) in _spans(counts):
        y[a:b], dx[a:b], dw[e] = x[a:b] @ w[e], dy[a:b] @ w[e].t(), x[a:b].t() @ dy[a:b]
    return y, dx, dw


COUNTS = {
    "one row": [1],
    "one row of many experts": [0, 0, 1, 0],
    "edges of a stage and of a tile": [63, 64, 65, 127, 128, 129, 255, 256, 257],
    "uneven": [700, 0, 3, 1500, 0, 90],
    "nobody": [0, 0, 0],
}
SIZES = [(64, 64), (8, 8), (7, 13), (129, 130), (200, 328), (515, 257)]


@pytest.mark.parametrize("kind,tol", [("bf16", BF16), ("fp32", 2e-6), ("tf32", 2.0**-15)])
@pytest.mark.parametrize("counts", COUNTS.values(), ids=COUNTS.keys())
@pytest.mark.parametrize("d,n", SIZES)
def test_products_and_gradients(kind, tol, counts, d, n):
    precision.set_precision("tf32" if kind == "tf32" else "fp32")
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    idle = 70
    g = torch.Generator(device="cuda").manual_seed(d * 1000 + n)
    rows = sum(counts) + idle
    x = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    w = torch.randn(len(counts), d, n, device="cuda", generator=g).to(dtype)
    dy = torch.randn(rows, n, device="cuda", generator=g).to(dtype)
    want = _exact_products(x, w, dy, counts)
    # Rows that nobody owns may hold anything.
    x[sum(counts):] = float("nan")
    dy[sum(counts):] = float("inf")
    x, w = x.requires_grad_(), w.requires_grad_()
    y = experts.ragged_matmul(x, w, _offsets(counts))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    for got, exact in zip((y, dx, dw), want):
        assert got.dtype == dtype
        assert torch.isfinite(got).all()
        assert _off(got, exact) <= tol
    for t in (y, dx):
        assert torch.all(t[sum(counts):] == 0)
    for e, c in enumerate(counts):
        if c == 0:
            assert torch.all(dw[e] == 0)


@pytest.mark.parametrize("kind,tol", [("bf16", 6 * BF16), ("fp32", 8e-6)])
@pytest.mark.parametrize("counts", COUNTS.values(), ids=COUNTS.keys())
@pytest.mark.parametrize("d,hidden", [(64, 128), (40, 24), (7, 13), (264, 200)])
def test_swiglu_mlp_and_gradients(kind, tol, counts, d, hidden):
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    idle = 5
    g = torch.Generator(device="cuda").manual_seed(d + hidden)
    rows, e = sum(counts) + idle, len(counts)
    x = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    mats = [(torch.randn(e, *s, device="cuda", generator=g) * s[0] ** -0.5).to(dtype) for s in ((d, hidden), (d, hidden), (hidden, d))]
    dy = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    want_y = torch.zeros(rows, d, dtype=torch.float64, device="cuda")
    xd, md = x.double().requires_grad_(), [m.double().requires_grad_() for m in mats]
    parts = [(torch.nn.functional.silu(xd[a:b] @ md[0][i]) * (xd[a:b] @ md[1][i])) @ md[2][i] for i, (a, b) in _spans(counts)]
    want_y = torch.cat([*parts, want_y[sum(counts):]])
    want = [want_y, *torch.autograd.grad(want_y, (xd, *md), dy.double())]
    x[sum(counts):] = float("inf")
    dy[sum(counts):] = float("nan")
    x, mats = x.requires_grad_(), [m.requires_grad_() for m in mats]
    y = experts.ragged_swiglu_mlp(x, *mats, _offsets(counts))
    got = [y, *torch.autograd.grad(y, (x, *mats), dy)]
    for a, b in zip(got, want):
        assert torch.isfinite(a).all()
        assert _off(a, b) <= tol


FEW = {
    "a row": ([1], 0),
    "a row of many experts, rows of nobody": ([0] * 20 + [1] + [0] * 5, 30),
    "each number of rows of a block": ([1, 2, 3, 4, 5, 8, 9, 16, 17] + [0] * 9, 2),
    "most in one expert": ([0, 3, 120, 0, 0, 0, 0, 0, 1] + [0] * 24, 0),
    "nobody": ([0, 0, 0], 5),
}


@pytest.mark.parametrize("kind,tol", [("bf16", BF16), ("fp32", 2e-6)])
@pytest.mark.parametrize("counts,idle", FEW.values(), ids=FEW.keys())
@pytest.mark.parametrize("d,n", [(1, 1), (8, 16), (7, 13), (72, 1100), (1033, 35), (520, 2056)])
def test_products_of_few_rows(kind, tol, counts, idle, d, n):
    """fp32 sums of up to 2056 products added in short runs: a few 2^-24 of the norm."""
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    rows = sum(counts) + idle
    assert rows <= 4 * len(counts) and rows <= 256  # what takes the kernels for few rows (fp32, and bf16 of odd widths)
    g = torch.Generator(device="cuda").manual_seed(d + n)
    x = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    w = torch.randn(len(counts), d, n, device="cuda", generator=g).to(dtype)
    dy = torch.randn(rows, n, device="cuda", generator=g).to(dtype)
    want = _exact_products(x, w, dy, counts)
    x[sum(counts):] = float("nan")
    dy[sum(counts):] = float("inf")
    got = _run(x, w, dy, _offsets(counts))
    for a, b in zip(got, want):
        assert a.dtype == dtype and torch.isfinite(a).all() and _off(a, b) <= tol
    # Layouts: a slice of wider rows, matrices seen through a transpose.
    wide = torch.zeros(rows, d + 3, device="cuda", dtype=dtype)
    wide[:, 1 : d + 1] = x
    for a, b in zip(_run(wide[:, 1 : d + 1], w.transpose(1, 2).contiguous().transpose(1, 2), dy, _offsets(counts)), got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind,tol", [("bf16", 3 * BF16), ("fp32", 8e-6)])
@pytest.mark.parametrize("counts,idle", FEW.values(), ids=FEW.keys())
@pytest.mark.parametrize("d,hidden", [(7, 13), (136, 264)])
def test_swiglu_mlp_of_few_rows(kind, tol, counts, idle, d, hidden):
    dtype = torch.bfloat16 if kind == "bf16" else torch.float32
    rows, e = sum(counts) + idle, len(counts)
    g = torch.Generator(device="cuda").manual_seed(d)
    x = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    mats = [(torch.randn(e, *s, device="cuda", generator=g) * s[0] ** -0.5).to(dtype) for s in ((d, hidden), (d, hidden), (hidden, d))]
    dy = torch.randn(rows, d, device="cuda", generator=g).to(dtype)
    xd, md = x.double().requires_grad_(), [m.double().requires_grad_() for m in mats]
    parts = [(torch.nn.functional.silu(xd[a:b] @ md[0][i]) * (xd[a:b] @ md[1][i])) @ md[2][i] for i, (a, b) in _spans(counts)]
    want_y = torch.cat([*parts, xd.new_zeros(idle, d)])
    want = [want_y, *torch.autograd.grad(want_y, (xd, *md), dy.double())]
    x[sum(counts):] = float("inf")
    dy[sum(counts):] = float("nan")
    x, mats = x.requires_grad_(), [m.requires_grad_() for m in mats]
    y = experts.ragged_swiglu_mlp(x, *mats, _offsets(counts))
    for a, b in zip([y, *torch.autograd.grad(y, (x, *mats), dy)], want):
        assert a.dtype == dtype and torch.isfinite(a).all() and _off(a, b) <= tol


def test_gradient_agrees_with_differences():
    """Directional derivative of a smooth loss: central differences at step s are off by s^2 of the third derivative and by
    the loss's fp32 rounding over s; 1e-3 relative covers both at s = 1e-2."""
    counts = [65, 0, 130]
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(sum(counts), 72, device="cuda", generator=g)
    mats = [torch.randn(3, *s, device="cuda", generator=g) * s[0] ** -0.5 for s in ((72, 96), (72, 96), (96, 72))]
    probe = torch.randn(sum(counts), 72, device="cuda", generator=g)
    off = _offsets(counts)

    def loss(args):
        return (experts.ragged_swiglu_mlp(*args, off).double() * probe.double()).sum()

    args = [t.requires_grad_() for t in (x, *mats)]
    grads = torch.autograd.grad(loss(args), args)
    for i, grad in enumerate(grads):
        direction = grad / grad.norm()
        step = 1e-2
        up, down = [t.detach() for t in args], [t.detach() for t in args]
        up[i], down[i] = up[i] + step * direction, down[i] - step * direction
        slope = float((loss(up) - loss(down)) / (2 * step))
        assert abs(slope - float(grad.norm())) <= 1e-3 * float(grad.norm())


def test_neighbours_do_not_leak():
    """Infinite and NaN rows of one expert stay in that expert, in every direction, at every alignment of its rows."""
    counts = [33, 64, 31, 200]
    off = _offsets(counts)
    for dtype in (torch.bfloat16, torch.float32):
        g = torch.Generator(device="cuda").manual_seed(4)
        x = torch.randn(sum(counts), 136, device="cuda", generator=g).to(dtype)
        w = torch.randn(4, 136, 144, device="cuda", generator=g).to(dtype)
        dy = torch.randn(sum(counts), 144, device="cuda", generator=g).to(dtype)
        y0, dx0, dw0 = _run(x, w, dy, off)
        x[33 + 5], dy[33 + 9] = float("inf"), float("nan")
        y1, dx1, dw1 = _run(x, w, dy, off)
        keep = torch.ones(sum(counts), dtype=torch.bool, device="cuda")
        keep[38] = keep[42] = False
        assert torch.equal(y0[keep], y1[keep]) and torch.equal(dx0[keep], dx1[keep])
        for e in (0, 2, 3):
            assert torch.equal(dw0[e], dw1[e])
        assert not torch.isfinite(y1[38]).any() and torch.isnan(dx1[42]).all() and not torch.isfinite(dw1[1]).any()


def _run(x, w, dy, off):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    y = experts.ragged_matmul(x, w, off)
    return (y.detach(), *torch.autograd.grad(y, (x, w), dy))


def test_layouts_other_than_contiguous():
    """Slices, transposes and broadcast gradients give what their contiguous copies give."""
    counts = [100, 37]
    off = _offsets(counts)
    g = torch.Generator(device="cuda").manual_seed(5)
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.randn(137, 300, device="cuda", generator=g).to(dtype)
        base = torch.randn(2, 80, 96, device="cuda", generator=g).to(dtype)
        for x in (wide[:, :96], wide[:, 1:97], wide.t().contiguous().t()[:, 3:99]):
            for w in (base.transpose(1, 2), base.transpose(1, 2).contiguous(), torch.randn(2, 96, 240, device="cuda", generator=g).to(dtype)[:, :, 5:85]):
                for dy in (torch.ones(1, 1, device="cuda", dtype=dtype).expand(137, 80), torch.randn(80, 137, device="cuda", generator=g).to(dtype).t()):
                    got = _run(x, w, dy, off)
                    want = _run(x.contiguous(), w.contiguous(), dy.contiguous(), off)
                    for a, b in zip(got, want):
                        assert torch.equal(a, b)


def test_results_repeat_and_follow_their_stream():
    counts = [900, 11, 300]
    off = _offsets(counts)
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(sum(counts), 512, device="cuda", generator=g)
    w = torch.randn(3, 512, 320, device="cuda", generator=g)
    dy = torch.randn(sum(counts), 320, device="cuda", generator=g)
    first = _run(x, w, dy, off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = _run(x, w, dy, off)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_range_of_fp32():
    """Large numbers survive the split into bf16 parts, and small ones down to 2^-110 or so (below that the third part is
    under bf16's smallest number, 2^-133)."""
    off = _offsets([4])
    x = torch.tensor([[3.4e38, 0.0], [1e-30, 1e-30], [float("inf"), 1.0], [-3.4028234e38, 0.0]], device="cuda")
    w = torch.eye(2, device="cuda").reshape(1, 2, 2)
    y = experts.ragged_matmul(x, w, off)
    assert torch.isfinite(y[0]).all() and abs(y[0, 0].item() / 3.4e38 - 1) < 1e-6
    assert abs(y[1, 0].item() / 1e-30 - 1) < 1e-6
    assert not torch.isfinite(y[2, 0])
    assert abs(y[3, 0].item() / -3.4028234e38 - 1) < 1e-6


def test_bad_offsets_stay_in_bounds():
    """Offsets that decrease are the caller's mistake: the kernels read and write inside their tensors, and the device
    status says so."""
    x, w = torch.randn(300, 64, device="cuda"), torch.randn(3, 64, 64, device="cuda")
    experts.ragged_matmul(x, w, torch.tensor([0, 200, 100, 300], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="status"):
        check_status()


def test_no_rows():
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.zeros(0, 24, device="cuda", dtype=dtype, requires_grad=True)
        mats = [torch.randn(3, *s, device="cuda").to(dtype).requires_grad_() for s in ((24, 40), (24, 40), (40, 24))]
        off = _offsets([0, 0, 0])
        for y, args in ((experts.ragged_matmul(x, mats[0], off), (x, mats[0])), (experts.ragged_swiglu_mlp(x, *mats, off), (x, *mats))):
            assert y.shape[0] == 0
            for grad, t in zip(torch.autograd.grad(y, args, torch.zeros_like(y)), args):
                assert grad.shape == t.shape and torch.all(grad == 0)


def test_differentiable_once():
    off = _offsets([4, 3])
    x = torch.randn(7, 16, device="cuda", requires_grad=True)
    w = torch.randn(2, 16, 16, device="cuda", requires_grad=True)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        torch.autograd.grad(experts.ragged_matmul(x, w, off).sum(), x, create_graph=True)
    plan = experts.expert_plan(torch.zeros(7, 1, dtype=torch.int64, device="cuda"), 2)
    with pytest.raises(RuntimeError, match="not differentiable twice"):
        torch.autograd.grad(experts.dispatch_tokens(x, plan).sum(), x, create_graph=True)


def test_only_the_gradients_that_are_asked_for():
    off = _offsets([5, 9])
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.randn(14, 32, device="cuda").to(dtype)
        mats = [torch.randn(2, *s, device="cuda").to(dtype) for s in ((32, 48), (32, 48), (48, 32))]
        full = [t.clone().requires_grad_() for t in (x, *mats)]
        want = torch.autograd.grad(experts.ragged_swiglu_mlp(*full, off).float().square().sum(), full)
        for i in range(4):
            args = [x, *mats]
            args[i] = args[i].clone().requires_grad_()
            (got,) = torch.autograd.grad(experts.ragged_swiglu_mlp(*args, off).float().square().sum(), args[i])
            assert torch.equal(got, want[i])


def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    w = torch.zeros(300, 8, 8, device="cuda")
    with pytest.raises(RuntimeError, match="at most 256 experts"):
        experts.ragged_matmul(x, w, torch.zeros(301, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="one device"):
        experts.ragged_matmul(x, w[:2], torch.tensor([0, 2, 4], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="1 to 1024 experts"):
        experts.expert_plan(torch.zeros(4, 1, dtype=torch.int64, device="cuda"), 2000)


# ------------------------------------------------------------------ routing
@pytest.mark.parametrize("tokens,choices,n_experts", [(0, 2, 4), (1, 1, 1), (1, 8, 8), (255, 2, 8), (1024, 2, 64), (1025, 2, 64), (3001, 3, 17), (70000, 2, 1000), (40000, 8, 128)])
def test_plan(tokens, choices, n_experts):
    g = torch.Generator().manual_seed(tokens + n_experts)
    indices = torch.randint(-1, n_experts + 1, (tokens, choices), generator=g)
    plan = experts.expert_plan(indices.cuda(), n_experts)
    want = experts.expert_plan(indices, n_experts)  # the CPU form is tested against the definition
    for a, b in zip(plan, want):
        assert torch.equal(a.cpu(), b)


def test_plan_of_more_assignments_than_parts_of_the_smallest_size():
    """Above 2^20 assignments a block takes more of them."""
    g = torch.Generator().manual_seed(9)
    indices = torch.randint(-1, 6, (700001, 2), generator=g)
    for a, b in zip(experts.expert_plan(indices.cuda(), 5), experts.expert_plan(indices, 5)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("indices", ["all to one", "all dropped", "int32"])
def test_plan_of_one_sided_routings(indices):
    idx = {"all to one": torch.full((5000, 2), 3), "all dropped": torch.full((5000, 2), -1),
           "int32": torch.arange(5000, dtype=torch.int32).view(-1, 1) % 9}[indices]
    for a, b in zip(experts.expert_plan(idx.cuda(), 8), experts.expert_plan(idx, 8)):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,choices,dim", [(1, 1, 1), (5, 2, 8), (300, 3, 770), (257, 8, 129), (2000, 2, 768)])
def test_dispatch_combine_and_gradients(dtype, tokens, choices, dim):
    g = torch.Generator(device="cuda").manual_seed(dim)
    indices = torch.randint(-1, 6, (tokens, choices), device="cuda", generator=g)
    plan = experts.expert_plan(indices, 6)
    n, used = tokens * choices, int(plan.offsets[-1])
    x = torch.randn(tokens, dim, device="cuda", generator=g).to(dtype).requires_grad_()
    w = torch.rand(tokens, choices, device="cuda", generator=g)
    w = torch.where(plan.slot >= 0, w, float("nan")).requires_grad_()  # a dropped assignment's weight counts for nothing
    ys = torch.randn(n, dim, device="cuda", generator=g).to(dtype)
    ys[used:] = float("inf")
    ys = ys.requires_grad_()
    dxs = torch.randn(n, dim, device="cuda", generator=g).to(dtype)
    dxs[used:] = float("nan")
    dout = torch.randn(tokens, dim, device="cuda", generator=g).to(dtype)
    xs = experts.dispatch_tokens(x, plan)
    out = experts.combine_tokens(ys, w, plan)
    dx, dys, dw = torch.autograd.grad((xs, out), (x, ys, w), (dxs, dout))
    place = plan.slot.clamp(min=0).long()
    kept = plan.slot >= 0
    want_xs = torch.zeros(n, dim, dtype=torch.float64, device="cuda")
    t, k = torch.nonzero(kept, as_tuple=True)
    want_xs[place[t, k]] = x.detach().double()[t]
    rows = torch.where(kept[..., None], ys.detach().double()[place], 0.0)
    wk = torch.where(kept, w.detach().double(), 0.0)
    want_dys = torch.zeros(n, dim, dtype=torch.float64, device="cuda")
    want_dys[place[t, k]] = wk[t, k, None] * dout.double()[t]
    assert torch.equal(xs.detach().double(), want_xs)
    tol = BF16 if dtype == torch.bfloat16 else 1e-6
    for got, want in ((out, (rows * wk[..., None]).sum(1)), (dx, torch.where(kept[..., None], dxs.double()[place], 0.0).sum(1)), (dys, want_dys)):
        assert _off(got, want) <= tol
    assert _off(dw, (rows * dout.double()[:, None]).sum(-1)) <= 1e-5
    strided = torch.randn(tokens, dim + 3, device="cuda", generator=g).to(dtype)[:, 1 : dim + 1]
    assert torch.equal(experts.dispatch_tokens(strided, plan), experts.dispatch_tokens(strided.contiguous(), plan))
