"""AdamW with 8-bit moments: the kernel against the CPU formulation and against 64 bits.

The rounding's random bits are a hash of (element, step), so both sides round alike except where fp32 arithmetic lands
on the other side of a threshold: a value's relative error of 2^-22 moves a 2^-3 grid step's threshold, of 2^16 places,
with a chance below 2^-19 * 8; fewer than one code in a thousand is asked. Weights differ by fp32 rounding, 1e-6 of
their size and of the step's.
"""
import pytest
import torch

from abacus_b200.ops import adamw8

pytestmark = pytest.mark.gpu


def _many(numels, kind, seed, shift=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in numels:
        # `shift` elements in front of each tensor take its alignment away.
        w, grad = torch.randn(n + shift, generator=g)[shift:], (torch.randn(n + shift, generator=g) * 0.01)[shift:].to(kind)
        out.append((w, grad, adamw8.fresh_state(n, "cpu")))
    return out


def _lists(tensors, device, shift=0):
    def put(t):
        if not shift:
            return t.to(device).clone()
        room = torch.empty(t.numel() + shift, dtype=t.dtype, device=device)[shift:]
        room.copy_(t)
        return room

    keys = ("exp_avg", "exp_avg_scale", "exp_rms", "exp_rms_scale")
    return ([put(w) for w, _, _ in tensors], [put(g) for _, g, _ in tensors], *([put(st[k]) for _, _, st in tensors] for k in keys))


@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("numels,shift", [([1], 0), ([0, 5, 256, 257], 0), ([4096, 100003, 17], 0), ([4096, 1001], 1), ([300] * 200, 0)])
def test_kernel_matches_cpu_over_steps(kind, numels, shift):
    tensors = _many(numels, kind, len(numels), shift)
    gpu, cpu = _lists(tensors, "cuda", shift), _lists(tensors, "cpu")
    for step in range(1, 4):
        adamw8.step_(*gpu, lr=1e-3, weight_decay=0.1, step=step)
        adamw8.step_(*cpu, lr=1e-3, weight_decay=0.1, step=step)
        for a, b in zip(gpu[0], cpu[0]):
            torch.testing.assert_close(a.cpu(), b, rtol=1e-6, atol=2e-8 + 1e-6)
        for which in (2, 4):
            a, b = (torch.cat([t.cpu().float() for t in side[which]]) for side in (gpu, cpu))
            assert (a != b).float().mean() <= 1e-3
        for which in (3, 5):
            for a, b in zip(gpu[which], cpu[which]):
                assert torch.equal(a.cpu(), b)
        # The next step starts from the same state on both sides.
        for a, b in zip(gpu, cpu):
            for s, t in zip(a, b):
                s.copy_(t)


def test_kernel_against_64_bits():
    tensors = _many([50000], torch.float32, 9)
    gpu = _lists(tensors, "cuda")
    w, m, v = tensors[0][0].double(), torch.zeros(50000, dtype=torch.float64), torch.zeros(50000, dtype=torch.float64)
    for step in range(1, 4):
        g = tensors[0][1].double()
        m = 0.9 * m + (1 - 0.9) * g
        v = 0.999 * v + (1 - 0.999) * g * g
        w = w * (1 - 1e-3 * 1e-2) - 1e-3 * (m / (1 - 0.9**step)) / ((v / (1 - 0.999**step)).sqrt() + 1e-8)
        adamw8.step_(*gpu, lr=1e-3, step=step)
        torch.testing.assert_close(gpu[0][0].cpu().double(), w, rtol=1e-6, atol=1e-6)
        # The next step's moments are what 8 bits kept.
        w = gpu[0][0].cpu().double()
        m = adamw8.dequantize(gpu[2][0].cpu(), gpu[3][0].cpu()).double()
        v = adamw8.dequantize(gpu[4][0].cpu(), gpu[5][0].cpu()).double() ** 2


def test_infinite_and_nan_gradients_spoil_their_element_alone():
    tensors = _many([700], torch.float32, 3)
    tensors[0][1][10], tensors[0][1][300] = float("nan"), float("-inf")
    gpu = _lists(tensors, "cuda")
    adamw8.step_(*gpu, lr=1e-3, step=1)
    bad = torch.zeros(700, dtype=torch.bool)
    bad[10] = bad[300] = True
    for which in (2, 4):
        assert torch.equal(torch.isnan(gpu[which][0].float()).cpu(), bad)
    assert torch.isfinite(gpu[0][0].cpu()[~bad]).all()


def test_refusals():
    gpu = _lists(_many([300], torch.float32, 1), "cuda")
    with pytest.raises(RuntimeError, match="contiguous"):
        adamw8.step_([torch.zeros(600, device="cuda")[::2]], *gpu[1:], lr=1e-3, step=1)
    with pytest.raises(RuntimeError, match="gradients"):
        adamw8.step_(gpu[0], [gpu[1][0].half()], *gpu[2:], lr=1e-3, step=1)
    with pytest.raises(RuntimeError, match="scales"):
        adamw8.step_(*gpu[:3], [gpu[3][0][:1]], *gpu[4:], lr=1e-3, step=1)
    with pytest.raises(RuntimeError, match="one CUDA device"):
        adamw8.step_(gpu[0], [gpu[1][0].cpu()], *gpu[2:], lr=1e-3, step=1)


def test_codes_are_the_cpu_formulation_s_over_many_elements():
    """Both sides compute the moments with the same roundings (the kernel's root is rounded to nearest but for one number
    in a million, which then changes a code with a chance below 2^-16), so a million elements give the same codes, step
    after step, and weights stay together although an unlike code would change an update by an eighth."""
    n = 1 << 20
    g = torch.Generator().manual_seed(11)
    # Magnitudes over twenty octaves, neighbours far apart, zeros among them.
    grad = torch.randn(n, generator=g) * torch.exp2(torch.randint(-20, 0, (n,), generator=g).float()) * (torch.rand(n, generator=g) > 0.1)
    tensors = [(torch.randn(n, generator=g), grad, adamw8.fresh_state(n, "cpu"))]
    gpu, cpu = _lists(tensors, "cuda"), _lists(tensors, "cpu")
    for step in range(1, 6):
        scale = 0.5 + torch.rand(n, generator=g)
        cpu[1][0].copy_(grad * scale)
        gpu[1][0].copy_(cpu[1][0])
        adamw8.step_(*gpu, lr=1e-3, step=step)
        adamw8.step_(*cpu, lr=1e-3, step=step)
        for which in (2, 4):
            assert (gpu[which][0].cpu().float() != cpu[which][0].float()).sum() <= 1
    torch.testing.assert_close(gpu[0][0].cpu(), cpu[0][0], rtol=1e-6, atol=1e-5)


@pytest.mark.parametrize("size", [1e-18, 1e-6, 1e5, 1e15])
def test_gradients_of_any_size(size):
    """Scales from 2^-68 to 2^43, on both sides of 2^14, where the kernel takes the scaling in one product or in two."""
    g = torch.Generator().manual_seed(13)
    n = 20000
    tensors = [(torch.randn(n, generator=g), torch.randn(n, generator=g) * size, adamw8.fresh_state(n, "cpu"))]
    gpu, cpu = _lists(tensors, "cuda"), _lists(tensors, "cpu")
    for step in range(1, 4):
        adamw8.step_(*gpu, lr=1e-3, step=step)
        adamw8.step_(*cpu, lr=1e-3, step=step)
        for which in (2, 4):
            assert (gpu[which][0].cpu().float() != cpu[which][0].float()).sum() <= 1
        for which in (3, 5):
            assert torch.equal(gpu[which][0].cpu(), cpu[which][0])
    torch.testing.assert_close(gpu[0][0].cpu(), cpu[0][0], rtol=1e-6, atol=1e-5)
