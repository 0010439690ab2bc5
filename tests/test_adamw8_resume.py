"""Checkpoints of AdamW with 8-bit moments: every parameter's state comes back, whatever width wrote it.

What a checkpoint holds is on the 8-bit grid, so loading it changes a code only where a block's largest moment had been
rounded up to 256 scales: the scale doubles and a code below the grid of the new one moves by 2^-9 of the old scale at
most, 2^-16 of the largest moment. A run that goes on from 32-bit moments rounds each of them once, by 2^-4 of its size
or by half of that smallest step.
"""
import os

import pytest
import torch

from _dist import run_ranks
from abacus_b200.models.transformer_moe import TransformerMoe
from abacus_b200.trainer import Trainer
from abacus_b200.transformer import Transformer
from abacus_b200.utils import checkpoint

KW = dict(dim=16, n_heads=4, head_dim=4, n_blocks=2, vocab_size=24, hidden_dim=32)


def _trainer(bits, seed=3):
    torch.manual_seed(seed)
    model = TransformerMoe(16, 2, 8, 1, 31, 3, 2, hidden_dim=24, router="softmax", ragged=True)
    return Trainer(model, total_steps=40, device="cpu", state_bits=bits)


def _batches(count):
    g = torch.Generator().manual_seed(4)
    return [torch.randint(0, 31, (2, 12), generator=g) for _ in range(count)]


def _same_moments(got, want, rounding=0.0):
    """States of one parameter, moments in 32 bits."""
    assert got["step"] == want["step"]
    for key, root in (("exp_avg", False), ("exp_avg_sq", True)):
        a, b = got[key].double().reshape(-1), want[key].double().reshape(-1)
        a, b = (a.sqrt(), b.sqrt()) if root else (a, b)
        assert a.shape == b.shape
        assert torch.all((a - b).abs() <= rounding * b.abs() + 2.0**-16 * b.abs().max()), key


@pytest.mark.parametrize("written,read", [(8, 8), (32, 8), (8, 32)])
def test_every_parameter_is_restored_and_training_goes_on(tmp_path, written, read):
    first = _trainer(written)
    batches = _batches(9)
    for b in batches[:6]:
        first.step(b)
    path = os.path.join(tmp_path, "c.pt")
    checkpoint.save_checkpoint(path, first.model, first.optimizer, first.scheduler)
    second = _trainer(read, seed=8)
    checkpoint.load_checkpoint(path, second.model, second.optimizer, second.scheduler)
    saved, restored = (t.optimizer.state_dict_by_name(t.model) for t in (first, second))
    assert set(restored) == set(saved) == {name for name, _ in second.model.named_parameters()}
    for name in saved:
        assert saved[name]["step"] == 6
        _same_moments(restored[name], saved[name], 2.0**-4 if (written, read) == (32, 8) else 0.0)
    # The loss of the first step depends on the weights alone, that of the later ones on the moments too. A parameter that
    # starts from nothing moves by the whole learning rate; what rounding a moment moves is a small part of it.
    before = [p.detach().clone() for p in first.model.parameters()]
    for i, b in enumerate(batches[6:]):
        l1, l2 = float(first.step(b)[0]), float(second.step(b)[0])
        assert abs(l1 - l2) <= (1e-5 if written == read else 2e-3), i
    with torch.no_grad():
        moved = torch.cat([(p - q).abs().flatten() for p, q in zip(first.model.parameters(), before)]).mean()
        apart = torch.cat([(p - q).abs().flatten() for p, q in zip(first.model.parameters(), second.model.parameters())]).mean()
    assert float(apart) <= (0.01 if written == read else 0.1) * float(moved)


def _zero(rank, world, path, stage):
    from abacus_b200.distributed.data_parallel import DataParallel

    torch.manual_seed(0)
    model = Transformer(**KW)
    trainer = Trainer(model, DataParallel(model, stage=stage), total_steps=8, device="cpu", state_bits=8)
    tokens = torch.randint(0, 24, (2, 8), generator=torch.Generator().manual_seed(10 + rank))
    for _ in range(2):
        trainer.step(tokens)
    checkpoint.save_checkpoint(path, model, trainer.optimizer, trainer.scheduler, parallel=trainer.parallel)
    torch.manual_seed(7)
    fresh = Transformer(**KW)
    checkpoint.load_checkpoint(path, fresh)  # weights before the ZeRO wrapper shards them
    again = Trainer(fresh, DataParallel(fresh, stage=stage), total_steps=8, device="cpu", state_bits=8)
    checkpoint.load_checkpoint(path, fresh, again.optimizer, again.scheduler, parallel=again.parallel)
    owned = 0
    for p1, p2 in zip(model.parameters(), fresh.parameters()):
        s1, s2 = trainer.optimizer.state.get(id(p1)), again.optimizer.state.get(id(p2))
        assert (s1 is None) == (s2 is None)
        if s1 is not None:
            owned += 1
            _same_moments({"step": s2["step"], **again.optimizer.moments(s2)}, {"step": s1["step"], **trainer.optimizer.moments(s1)})
            assert s2["step"] == 2 and s2["exp_avg"].dtype == torch.float8_e4m3fn
    assert owned > 1
    for _ in range(2):
        l1, l2 = float(trainer.step(tokens)[0]), float(again.step(tokens)[0])
        assert abs(l1 - l2) <= 1e-5


@pytest.mark.parametrize("stage", [1, 2, 3])
def test_zero_ranges_are_restored(tmp_path, stage):
    path = str(tmp_path / "zero.pt")
    run_ranks(_zero, 2, path, stage)
    saved = torch.load(path, weights_only=False)["optimizer"]
    for name, p in Transformer(**KW).named_parameters():
        assert saved[name]["exp_avg"].shape == p.shape and saved[name]["step"] == 2, name
