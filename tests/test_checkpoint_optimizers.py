"""Checkpoints take any optimizer that keeps ``state`` by parameter id, ``lr`` and ``load_state_dict_by_name``."""
import torch

from abacus_b200.transformer import Transformer
from abacus_b200.utils.checkpoint import load_checkpoint, save_checkpoint


class _Plain:
    """Adam's 32-bit moments and nothing else of AdamW."""

    def __init__(self, model):
        self.lr = 0.5
        self.state = {id(p): {"step": 3, "exp_avg": torch.randn(p.shape), "exp_avg_sq": torch.rand(p.shape)} for p in model.parameters()}

    def load_state_dict_by_name(self, model, state):
        self.loaded = state


def test_state_of_another_optimizer_is_saved_and_loaded(tmp_path):
    torch.manual_seed(0)
    model = Transformer(dim=16, n_heads=4, head_dim=4, n_blocks=1, vocab_size=24, hidden_dim=32)
    opt = _Plain(model)
    save_checkpoint(tmp_path / "c.pt", model, opt)
    load_checkpoint(tmp_path / "c.pt", model, opt)
    for name, p in model.named_parameters():
        assert opt.loaded[name]["step"] == 3
        for key in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(opt.loaded[name][key], opt.state[id(p)][key])
