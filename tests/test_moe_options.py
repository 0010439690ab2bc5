"""Options of the ragged experts are refused where they would have no effect (CPU)."""
import pytest
import torch

from abacus_b200.models.transformer_moe import TransformerMoe


@pytest.mark.parametrize("options", [dict(ragged=True), dict(expert_dtype=torch.bfloat16), dict(expert_dtype=torch.float32),
                                     dict(ragged=True, expert_dtype=torch.bfloat16)])
def test_expert_parallel_refuses_them(options):
    with pytest.raises(ValueError, match="expert parallel"):
        TransformerMoe(8, 2, 4, 1, 11, 2, 1, expert_parallel=True, **options)
    TransformerMoe(8, 2, 4, 1, 11, 2, 1, expert_parallel=True)
