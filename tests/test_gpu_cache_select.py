"""The block selection where its order is hard to find: scores that are
infinite or NaN, hundreds of equal scores, and a narrow band of scores below
an outlier. Lists are whole numbers and have to be equal."""
import math

import pytest
import torch

import cache_ref as R
from test_gpu_cache import Pool

pytestmark = pytest.mark.gpu


def _order(scores, top, sink, local):
    """Ascending block numbers: forced ones, then NaN, then by score; ties to the lowest block."""
    n = len(scores)
    key = [(0, 0.0) if i < sink or i >= n - local else (1, 0.0) if math.isnan(s) else (2, -s) for i, s in enumerate(scores.tolist())]
    return sorted(sorted(range(n), key=lambda i: key[i] + (i,))[:top])


def _check(pool, q, top, sink=1, local=1):
    B, H, n, d = q.shape
    rep = H // pool.n_kv
    got = pool.select(q, top, sink=sink, local=local).cpu()
    bd, am, tab = pool.bounds.cpu().double(), pool.amax.cpu().double(), pool.table.cpu().long()
    for b in range(B):
        start = int(pool.start[b])
        for t in range(n):
            pages = tab[b, :(start + t) // pool.bs + 1]
            for h in range(pool.n_kv):
                s = R.select_scores(q[b, h * rep:(h + 1) * rep, t].cpu().double(), bd[pages, h], am[pages, h, 0])
                want = _order(s, top, sink, local)
                assert got[b, t, h].tolist() == want + [-1] * (top - len(want)), (b, t, h)


def _pool(cuda, blocks, n, seed=0):
    """One sequence of `blocks` blocks of 16 tokens; n = 80 tokens of two kv heads
    are enough units for one thread block each, one token is a cluster's."""
    pool = Pool(cuda, 1, 2, 32, 16, blocks, torch.bfloat16, seed=seed)
    pool.bounds = pool.bounds.sort(2).values
    pool.lens = torch.tensor([blocks * 16], dtype=torch.int32, device=cuda)
    pool.start = pool.lens - n
    q = torch.randn(1, 4, n, 32, generator=torch.Generator().manual_seed(seed + 1)).to(cuda, torch.bfloat16)
    return pool, q


@pytest.mark.parametrize("n", [1, 80])
@pytest.mark.parametrize("blocks,bad", [(60, 3), (60, 20), (60, 58), (1000, 4), (1000, 200), (1000, 700)])
@pytest.mark.parametrize("value", [math.inf, math.nan])
def test_select_with_scores_that_are_not_finite(value, blocks, bad, n, cuda):
    """Pages whose amax is infinite or NaN, fewer and more than places. An
    infinite amax gives plus or minus infinity, or NaN where the sum is 0."""
    pool, q = _pool(cuda, blocks, n)
    g = torch.Generator().manual_seed(bad)
    at = torch.randperm(blocks, generator=g)[:bad]
    pool.amax[pool.table[0, at.to(cuda)].long()] = value
    pool.bounds[pool.table[0, at[:bad // 2].to(cuda)].long()] = 0  # as an append leaves them
    _check(pool, q, 8)


@pytest.mark.parametrize("n", [1, 80])
def test_select_of_many_equal_scores(n, cuda):
    """More equal scores than are ranked one by one: the lowest blocks are listed."""
    pool, q = _pool(cuda, 1000, n, seed=3)
    pool.bounds[:] = pool.bounds[:1]
    pool.amax.fill_(0.75)
    _check(pool, q, 40, sink=2, local=3)
    pool.amax[pool.table[0, 500:510].long()] = 0.8125
    pool.amax[pool.table[0, 700:].long()] = 0.6875
    _check(pool, q, 40, sink=2, local=3)


@pytest.mark.parametrize("n", [1, 80])
def test_select_below_an_outlier(n, cuda):
    """One score far above and hundreds of different ones close together: the
    last listed one is found in a second pass over a part of the range."""
    pool, q = _pool(cuda, 1000, n, seed=4)
    pool.bounds[:] = pool.bounds[:1].abs()
    q = q.abs()
    pool.amax = 1 + torch.arange(pool.P * 4, device=cuda).view(pool.P, 2, 2).float() * 2.0 ** -14
    pool.amax[pool.table[0, 321].long()] = 2.0 ** 60
    _check(pool, q, 40)
