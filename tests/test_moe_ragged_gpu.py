"""The MoE model on the ragged operators against the framework's other expert paths, and trained with 8-bit moments."""
import pytest
import torch

from abacus_b200.models.transformer_moe import TransformerMoe
from abacus_b200.ops._ext import check_status, ext
from abacus_b200.trainer import Trainer

pytestmark = pytest.mark.gpu


def _models(**kwargs):
    made = []
    for ragged in (False, True):
        torch.manual_seed(0)
        extra = dict(ragged=True, **kwargs) if ragged else {}
        made.append(TransformerMoe(128, 2, 64, 2, 512, 4, 2, hidden_dim=192, router="softmax", init_std=0.5, **extra).cuda())
    return made


@pytest.mark.parametrize("kind,tol", [(None, 2e-5), (torch.bfloat16, 24 * 2.0**-8)])
def test_model_matches_the_expert_loop(kind, tol):
    """fp32: both paths are fp32 products, apart by the order of their sums. bf16: two layers of experts, a dozen roundings
    of 2^-8 each."""
    plain, ragged = _models(expert_dtype=kind)
    tokens = torch.randint(0, 512, (3, 65), device="cuda")
    got = []
    for model in (plain, ragged):
        logits = model(tokens)
        logits.square().mean().backward()
        got.append([logits.detach(), *(p.grad for n, p in model.named_parameters() if "moe.w_" in n)])
    check_status()
    for a, b in zip(*got):
        assert (a - b).norm() <= tol * a.norm()


def test_no_host_synchronisation():
    _, model = _models()
    tokens = torch.randint(0, 512, (2, 33), device="cuda")
    moe = model.blocks[0].moe
    x = torch.randn(2, 33, 128, device="cuda", requires_grad=True)
    moe(x).sum().backward()  # allocations and launches' first-time work
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        moe(x).sum().backward()
    finally:
        torch.cuda.set_sync_debug_mode("default")
    model(tokens)


def test_trainer_with_bf16_experts_and_8_bit_moments():
    _, model = _models(expert_dtype=torch.bfloat16)
    trainer = Trainer(model, total_steps=40, lr=1e-3, state_bits=8)
    tokens = torch.randint(0, 512, (4, 64), generator=torch.Generator().manual_seed(1))
    before = ext().launch_count()
    losses = [float(trainer.step(tokens)[0]) for _ in range(20)]
    check_status()
    assert ext().launch_count() > before
    assert losses[-1] < losses[0] - 0.1
    state = trainer.optimizer.state[id(model.blocks[0].moe.w_up_EDM)]
    assert state["exp_avg"].dtype == torch.float8_e4m3fn and state["step"] == 20
