"""Lengths that outrun a step's rows: no token is counted that was not stored."""
import pytest
import torch

from ssa_b200 import BlockCache
from test_gpu_serving import _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompt", [False, True])
def test_new_lens_beyond_the_rows_count_as_the_rows(prompt, cuda):
    m, g = _model(torch.bfloat16, cuda), torch.Generator().manual_seed(1)
    ids = torch.randint(0, 50, (3, 20), generator=g).to(cuda)
    nxt = torch.randint(0, 50, (3, 1), generator=g).to(cuda)
    got = []
    for new in ([20, 45, 7], [20, 20, 7]):
        cache = m.new_cache(3, 64, block_size=16)
        cache.k_codes.fill_(99), cache.v_codes.fill_(99), cache.amax.fill_(50.0)  # what another sequence left
        new = torch.tensor(new, dtype=torch.int32, device=cuda)
        out = (m.prefill if prompt else m.step)(ids, cache, new)
        assert cache.lens.tolist() == [20, 20, 7]
        assert sorted(cache.table[cache.table >= 0].tolist()) == sorted(set(cache.table[cache.table >= 0].tolist()))
        assert int(cache.state[0]) == cache.num_blocks - 5
        got.append((out, m.step(nxt, cache)))
        assert new.tolist() in ([20, 45, 7], [20, 20, 7])  # the argument is not written
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_append_of_fewer_rows_than_reserved_is_refused(cuda):
    cache = BlockCache(2, 2, 64, 64, block_size=16)
    x = torch.randn(2, 2, 5, 64, device=cuda, dtype=torch.bfloat16)
    cache.reserve(8)
    before = cache.tail.clone()
    with pytest.raises(ValueError, match="reserved"):
        cache.append(x, x)
    assert torch.equal(cache.tail, before)
    cache.reserve(5)
    cache.append(x, x)
    with pytest.raises(ValueError, match="rows"):
        cache.reserve(9, limit=8)
    cache.reserve(torch.tensor([1, 9], dtype=torch.int32, device=cuda), limit=5)
    assert (cache.lens - cache.start).tolist() == [1, 5]
    cache.append(x, x)
    with pytest.raises(ValueError, match="reserved"):
        cache.append(x[:, :, :4], x[:, :, :4])
