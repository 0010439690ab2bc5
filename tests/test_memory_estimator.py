"""Moments in the memory estimate (CPU)."""
import pytest

from abacus_b200.memory_estimator import estimate
from abacus_b200.ops import adamw8

SIZES = dict(dim=64, heads=2, head_dim=32, blocks=2, hidden=128, vocab=512, batch=4, seq_len=32)


def _bytes(state):
    return sum(t.numel() * t.element_size() for t in state.values())


@pytest.mark.parametrize("dp,zero", [(1, 0), (8, 1), (8, 3)])
def test_moments(dp, zero):
    wide, narrow = (estimate(**SIZES, dp=dp, zero=zero, state_bits=bits) for bits in (32, 8))
    params = wide["params_M"] * 1e6 / (dp if zero else 1)
    assert wide["adam_GB"] * 1024**3 == pytest.approx(8 * params)
    # What the optimizer allocates for as many elements in whole blocks.
    elements = 1 << 16
    assert narrow["adam_GB"] * 1024**3 == pytest.approx(params * _bytes(adamw8.fresh_state(elements, "cpu")) / elements)
    assert wide["total_GB"] - narrow["total_GB"] == pytest.approx(wide["adam_GB"] - narrow["adam_GB"])
    assert estimate(**SIZES, dp=dp, zero=zero) == wide
