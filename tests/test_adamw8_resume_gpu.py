"""A run with 8-bit moments and bf16 ragged experts goes on from its checkpoint on the GPU.

Loading changes a code only where a block's largest moment had been rounded up to 256 scales, by 2^-16 of that moment at
most, so the two runs' weights stay within a hundredth of what they move.
"""
import os

import pytest
import torch

from abacus_b200.models.transformer_moe import TransformerMoe
from abacus_b200.trainer import Trainer
from abacus_b200.utils import checkpoint

pytestmark = pytest.mark.gpu


def _trainer(bits, seed):
    torch.manual_seed(seed)
    model = TransformerMoe(64, 1, 64, 2, 256, 4, 2, hidden_dim=96, router="softmax", ragged=True, expert_dtype=torch.bfloat16)
    return Trainer(model.cuda(), total_steps=40, device="cuda", state_bits=bits)


@pytest.mark.parametrize("written", [8, 32])
def test_resume(tmp_path, written):
    first = _trainer(written, 1)
    g = torch.Generator().manual_seed(2)
    batches = [torch.randint(0, 256, (4, 64), generator=g) for _ in range(8)]
    for b in batches[:5]:
        first.step(b.cuda())
    path = os.path.join(tmp_path, "c.pt")
    checkpoint.save_checkpoint(path, first.model, first.optimizer, first.scheduler)
    second = _trainer(8, 3)
    checkpoint.load_checkpoint(path, second.model, second.optimizer, second.scheduler)
    saved, restored = (t.optimizer.state_dict_by_name(t.model) for t in (first, second))
    assert set(restored) == set(saved) == {name for name, _ in second.model.named_parameters()}
    for name, want in saved.items():
        assert restored[name]["step"] == want["step"] == 5
        for key, root in (("exp_avg", False), ("exp_avg_sq", True)):
            a, b = restored[name][key].double().reshape(-1), want[key].double().reshape(-1)
            a, b = (a.sqrt(), b.sqrt()) if root else (a, b)
            assert torch.all((a - b).abs() <= (0 if written == 8 else 2.0**-4) * b.abs() + 2.0**-16 * b.abs().max())
    if written == 8:
        before = [p.detach().clone() for p in first.model.parameters()]
        for b in batches[5:]:
            first.step(b.cuda())
            second.step(b.cuda())
        with torch.no_grad():
            ps = list(zip(first.model.parameters(), second.model.parameters(), before))
            moved, apart = (torch.cat([(p - x).abs().flatten() for p, x in pairs]).mean() for pairs in
                            ([(p, o) for p, _, o in ps], [(p, q) for p, q, _ in ps]))
        assert float(apart) <= 0.01 * float(moved)
