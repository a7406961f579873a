"""The operators around the attention at the largest sizes that they take."""

import pytest
import torch

from recap_b200 import Norm, gated_residual, modulated_norm, rotate_qk

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


def _needs(gigabytes):
    if torch.cuda.mem_get_info()[0] < gigabytes * 2**30:
        pytest.skip(f"needs {gigabytes} GB")


@pytest.mark.parametrize("gated", [False, True])
def test_most_tokens(gated):
    """2^31 - 1 tokens of eight channels, all of them one row: each output row is that row's."""
    _needs(48)
    tokens = 2**31 - 1
    row = torch.randn(1, 8, device=DEV).to(BF)
    x = row.expand(tokens, 8)
    want = gated_residual(row, row)[0] if gated else modulated_norm(row, Norm("rms"))
    got = gated_residual(x, x)[0] if gated else modulated_norm(x, Norm("rms"))
    for lo in range(0, tokens, 2**28):
        assert bool((got[lo:lo + 2**28] == want).all())


@pytest.mark.parametrize("heads", [2**25 + 1, 2**27 - 3])
def test_many_heads(heads):
    """Heads whose cost, counted in instructions, passes 2^31."""
    _needs(8)
    row = torch.randn(1, 1, 1, 8, device=DEV).to(BF)
    norm = Norm("rms")
    want = rotate_qk(row, None, query_norm=norm)[0]
    assert bool((rotate_qk(row.expand(1, heads, 1, 8), None, query_norm=norm)[0] == want).all())
