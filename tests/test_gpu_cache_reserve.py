"""Page reservation where the needs of many sequences add up past 32 bits."""
import pytest
import torch

from ssa_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("max_blocks,served", [((1 << 21) - 1, 2), (1 << 21, 3)])
def test_needs_beyond_32_bits(max_blocks, served, cuda):
    """1024 sequences that each ask for a whole row of a table of 2^31 entries,
    with pages for a few: those are served in order, the others refused."""
    B, bs = 1024, 16
    P = served * max_blocks + 12345
    table = torch.full((B, max_blocks), -1, dtype=torch.int32, device=cuda)
    free = torch.arange(P, dtype=torch.int32, device=cuda)
    lens = torch.zeros(B, dtype=torch.int32, device=cuda)
    new = torch.full((B,), max_blocks * bs, dtype=torch.int32, device=cuda)
    state = torch.tensor([P, 5], dtype=torch.int32, device=cuda)
    start, after, st = ops.cache_reserve(lens, new, table, free, state, bs)
    assert start.tolist() == [0] * B
    assert after.tolist() == [max_blocks * bs] * served + [0] * (B - served)
    assert st.tolist() == [12345, 5 + B - served]
    want = free.flip(0)[:served * max_blocks].view(served, max_blocks)
    assert torch.equal(table[:served], want)
    assert int(table[served:].max()) == -1
