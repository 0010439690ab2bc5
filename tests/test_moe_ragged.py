"""MoE on the ragged operators, AdamW's 8-bit state in the optimizer, trainer and checkpoints (CPU)."""
import os
import subprocess
import sys

import pytest
import torch

from abacus_b200.models.moe import MoE
from abacus_b200.models.transformer_moe import TransformerMoe
from abacus_b200.optim.adamw import AdamW
from abacus_b200.trainer import Trainer
from abacus_b200.utils import checkpoint


def _pair(capacity_factor=None, router="softmax", **kwargs):
    torch.manual_seed(0)
    plain = MoE(8, 4, 2, hidden_dim=12, router=router, capacity_factor=capacity_factor)
    ragged = MoE(8, 4, 2, hidden_dim=12, router=router, capacity_factor=capacity_factor, ragged=True, **kwargs)
    ragged.load_state_dict(plain.state_dict())
    return plain, ragged


@pytest.mark.parametrize("capacity_factor", [None, 0.6])
@pytest.mark.parametrize("router", ["softmax", "sigmoid"])
def test_ragged_moe_equals_the_expert_loop(capacity_factor, router):
    plain, ragged = _pair(capacity_factor, router)
    x = torch.randn(2, 9, 8)
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    ya, yb = plain(a), ragged(b)
    torch.testing.assert_close(ya, yb)
    probe = torch.randn_like(ya)
    (ya * probe).sum().backward()
    (yb * probe).sum().backward()
    torch.testing.assert_close(a.grad, b.grad)
    for p, q in zip(plain.parameters(), ragged.parameters()):
        torch.testing.assert_close(p.grad, q.grad)


def test_bf16_experts_stay_near():
    plain, ragged = _pair(expert_dtype=torch.bfloat16)
    x = torch.randn(2, 9, 8)
    a, b = plain(x), ragged(x)
    assert b.dtype == torch.float32
    # Rows, matrices, gate, up, h and the rows' result are rounded to 8 bits: a dozen roundings of 2^-8 at most.
    assert (a - b).norm() <= 12 * 2.0**-8 * a.norm()


def test_refusals():
    with pytest.raises(ValueError, match="ragged"):
        MoE(8, 4, 2, expert_dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="expert_dtype"):
        MoE(8, 4, 2, ragged=True, expert_dtype=torch.float16)
    with pytest.raises(ValueError, match="expert parallel"):
        TransformerMoe(8, 2, 4, 1, 11, 2, 1, expert_parallel=True, ragged=True)
    with pytest.raises(ValueError, match="state_bits"):
        AdamW(torch.nn.Linear(2, 2), state_bits=16)
    lin = torch.nn.Linear(2, 2).bfloat16()
    opt = AdamW(lin, state_bits=8)
    lin.weight.grad = torch.zeros_like(lin.weight)
    with pytest.raises(ValueError, match="fp32 weights"):
        opt.step()


def test_8_bit_optimizer_over_an_owned_range_and_its_checkpoint(tmp_path):
    torch.manual_seed(1)
    sliced, full = torch.nn.Linear(30, 20), torch.nn.Linear(30, 20)
    full.load_state_dict(sliced.state_dict())
    owned = {id(sliced.weight): (256, 600), id(sliced.bias): (0, 20)}
    opt, ref = AdamW(sliced, owned=owned, state_bits=8), AdamW(full, state_bits=8)
    for step in range(3):
        for p, q in zip(sliced.parameters(), full.parameters()):
            p.grad = torch.randn(p.shape, generator=torch.Generator().manual_seed(step))
            q.grad = p.grad.clone()
        opt.step()
        ref.step()
    # The step's arithmetic is the same; the moments differ by the random bits, which count from the range's start.
    torch.testing.assert_close(sliced.weight.view(-1)[256:], full.weight.view(-1)[256:], rtol=0.0, atol=6e-4)
    torch.testing.assert_close(sliced.bias, full.bias)
    assert opt.state[id(sliced.weight)]["exp_avg"].numel() == 344
    saved = ref.state_dict_by_name(full)
    assert saved["weight"]["exp_avg"].dtype == torch.float32 and saved["weight"]["exp_avg_sq"].shape == full.weight.shape
    again = AdamW(full, state_bits=8)
    again.load_state_dict_by_name(full, saved)
    for name, entry in again.state_dict_by_name(full).items():
        assert entry["step"] == 3
        for key in ("exp_avg", "exp_avg_sq"):
            torch.testing.assert_close(entry[key], saved[name][key])
    wide = AdamW(full)
    wide.load_state_dict_by_name(full, saved)
    assert torch.equal(wide.state[id(full.weight)]["exp_avg"], saved["weight"]["exp_avg"])


def test_training_with_8_bit_moments_and_resuming(tmp_path):
    def trainer(bits):
        torch.manual_seed(3)
        model = TransformerMoe(16, 2, 8, 1, 31, 3, 2, hidden_dim=24, router="softmax", ragged=True)
        return Trainer(model, total_steps=40, device="cpu", state_bits=bits)

    g = torch.Generator().manual_seed(4)
    batches = [torch.randint(0, 31, (2, 12), generator=g) for _ in range(12)]
    eight, wide = trainer(8), trainer(32)
    losses = {8: [], 32: []}
    for b in batches:
        losses[8].append(float(eight.step(b)[0]))
        losses[32].append(float(wide.step(b)[0]))
    # The first step is the same step; later ones drift by the rounding of moments, a few percent of an update.
    assert abs(losses[8][0] - losses[32][0]) < 1e-5
    assert abs(losses[8][-1] - losses[32][-1]) < 0.02
    path = os.path.join(tmp_path, "c.pt")
    checkpoint.save_checkpoint(path, eight.model, eight.optimizer, eight.scheduler)
    resumed = trainer(8)
    checkpoint.load_checkpoint(path, resumed.model, resumed.optimizer, resumed.scheduler)
    next_batch = torch.randint(0, 31, (2, 12), generator=g)
    torch.testing.assert_close(resumed.step(next_batch)[0], eight.step(next_batch)[0])


def test_example_runs(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, CUDA_VISIBLE_DEVICES="")
    cmd = [sys.executable, os.path.join(root, "examples", "train_gpt_moe.py"), "--synthetic", "6", "--synthetic-length", "16",
           "--vocab-size", "64", "--top-k", "2", "--ragged-experts", "--expert-dtype", "bf16", "--state-bits", "8"]
    out = subprocess.run(cmd, cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr[-2000:]
