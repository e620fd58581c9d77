"""Cache attention where the pages of V differ: a page of zeros beside small
values, and pages that stand for NaN, which only the output may see."""
import math

import pytest
import torch

import cache_ref as R
from test_gpu_cache import BF, F32, Pool, _held, _kv, _widen

pytestmark = pytest.mark.gpu


def _rows(pool, q, blocks=None):
    """Each row's reference: (b, h, t, scores (seen keys) float64, v (seen keys, d) float64)."""
    B, H, n, _ = q.shape
    rep, qc = H // pool.n_kv, q.cpu().double()
    for b in range(B):
        length, start = int(pool.lens[b]), int(pool.start[b])
        k, v = _held(pool, b, length)
        for h in range(H):
            for t in range(min(n, length - start)):
                seen = torch.arange(length) <= start + t
                if blocks is not None:
                    on = torch.zeros(-(-length // pool.bs), dtype=torch.bool)
                    on[[e for e in blocks[b, t, h // rep].tolist() if 0 <= e < len(on)]] = True
                    seen &= on.repeat_interleave(pool.bs)[:length]
                yield b, h, t, qc[b, h, t] @ k[h // rep][seen].T, v[h // rep][seen], k[h // rep][seen]


def _tolerance(q, p, v, reach, ref, d):
    """Like cache_ref.attention_tolerance, but against the sum of p |v| instead of
    the greatest |v|: a weight's rounding is relative to itself as long as it is
    one of fp16's normal numbers. The offset leaves the largest p |step| at 2^13
    or more, and what rounds to fp16 below 2^-14 is off by at most 2^-25: 2^-38 of
    the largest p amax a key."""
    half = torch.finfo(q.dtype).eps / 2
    weight = 2.0 ** -11 if q.dtype == BF else 2.0 ** -21
    rel = 2 * (d + 8) * 2.0 ** -23 * reach + 2 * (weight + 2.0 ** -21) + (len(p) / 64 + 48) * 2.0 ** -23
    mass = (p[:, None] * v.abs()).sum(0)
    return half * ref.abs() * (1 + 2.0 ** -7) + rel * mass + len(p) * 2.0 ** -38 * (p * v.abs().amax(1)).max()


# dtype, kv heads, query heads a kv head, d. 300 heads are more work than thread blocks, so that a warp of the few-row
# kernel goes through several pages; 64 rows and more are the many-row kernel's.
ZEROS = [(BF, 300, 4, 128), (F32, 300, 4, 64), (BF, 300, 16, 64), (F32, 300, 32, 96), (BF, 1, 128, 64), (BF, 1, 64, 128)]


@pytest.mark.parametrize("where", ["first", "middle", "last"])
@pytest.mark.parametrize("octaves", [0, 12])
@pytest.mark.parametrize("amax", [1e15, 1e-3, 1e-5, 1e-7, 1e-12])
@pytest.mark.parametrize("case", range(len(ZEROS)))
def test_page_of_zeros_beside_small_values(case, amax, octaves, where, cuda):
    """A page of zeros takes its share of the weights' sum and nothing else,
    whatever its scores and however small the other pages' values are."""
    dtype, n_kv, rep, d = ZEROS[case]
    bs, L, scale = 16, 512, d ** -0.5
    g = torch.Generator().manual_seed(case)
    pool = Pool(cuda, 1, n_kv, d, bs, L // bs, dtype, seed=case)
    one = torch.randn(d, generator=g)
    q = (one * (1 + torch.arange(rep) / 256)[:, None]).to(dtype)
    k = 0.1 * torch.randn(L, d, generator=g)
    z = {"first": 0, "middle": 5, "last": L // bs - 1}[where] * bs
    k[z:z + bs] = one * (octaves * math.log(2) / (scale * float(one @ one)))
    v = (0.25 + 0.75 * torch.rand(L, d, generator=g)) * amax
    v[z:z + bs] = 0
    pool.advance([L])
    every = lambda x: x.to(cuda, dtype).expand(1, n_kv, L, d).contiguous()  # noqa: E731
    pool.append(every(k), every(v))
    pool.start = pool.lens - 1
    if rep >= 64:
        _widen(pool, -(-2 ** 24 // (rep * bs)))
    out, lse = pool.attend(q.to(cuda).repeat(n_kv, 1)[None, :, None].contiguous(), scale, want_lse=True)
    out, lse = out.cpu().double().view(n_kv, rep, d), lse.cpu().double().view(n_kv, rep)
    sub = Pool.__new__(Pool)
    sub.__dict__.update(pool.__dict__, n_kv=1)  # the heads hold the same
    for b, h, t, s, vs, ks in _rows(sub, q[None, :, None]):
        p = torch.softmax(s * scale, 0)
        ref = p @ vs
        reach = float((q[h].double().abs() @ ks.abs().T * scale).max())
        tol = _tolerance(q, p, vs, reach, ref, d)
        err = (out[:, h] - ref).abs()
        assert (err <= tol).all(), (h, float((err / tol).max()))
        # the offset and the logarithm of the sum may each be as far as 128 from zero: 2^-17 between them
        assert ((lse[:, h] - torch.logsumexp(s * scale, 0)).abs() <= (d + 8) * 2.0 ** -23 * reach + 2.0 ** -17).all()


def test_only_zeros(cuda):
    """A sequence whose V is all zero gives 0 and the lse of its scores."""
    for dtype, _, H, d in ZEROS:
        pool = Pool(cuda, 1, 1, d, 16, 8, dtype)
        pool.advance([100])
        g = torch.Generator().manual_seed(1)
        k, q = _kv(g, 1, 100, 1, d, dtype, cuda), _kv(g, 1, 1, H, d, dtype, cuda)
        pool.append(k, torch.zeros_like(k))
        pool.start = pool.lens - 1
        if H >= 64:
            _widen(pool, -(-2 ** 24 // (H * 16)))
        out, lse = pool.attend(q, 0.125, want_lse=True)
        assert not out.any()
        for b, h, t, s, vs, ks in _rows(pool, q):
            reach = float((q[b, h, t].cpu().double().abs() @ ks.abs().T * 0.125).max())
            ref = float(torch.logsumexp(s * 0.125, 0))
            assert abs(float(lse[b, h, t]) - ref) <= (d + 8) * 2.0 ** -23 * reach + 2.0 ** -17 + abs(ref) * 2.0 ** -22

@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("case", range(len(ZEROS)))
def test_lse_does_not_depend_on_values(case, value, listed, cuda):
    """A page of V that is not finite makes the outputs of the rows that see it
    NaN. Their lse, and rows before the page or without it in their list, do not
    see it."""
    dtype, _, H, d = ZEROS[case]
    n, bs, L = 20, 16, 70
    g = torch.Generator().manual_seed(case)
    pool = Pool(cuda, 2, 1, d, bs, 6, dtype, seed=case)
    k, v = _kv(g, 2, L, 1, d, dtype, cuda), _kv(g, 2, L, 1, d, dtype, cuda)
    v[1, 0, 58, 7] = value  # block 3, positions 48 .. 63
    pool.advance([L, L])
    pool.append(k, v)
    pool.start = pool.lens - n  # rows at 50 .. 69 ...
    pool.start[1] = 40          # ... and 40 .. 59 of a sequence of 60: the first eight end before the block
    pool.lens[1] = 60
    q = _kv(g, 2, n, H, d, dtype, cuda)
    blocks = None
    if listed:
        blocks = torch.tensor([0, 2, 3, -1], dtype=torch.int32).expand(2, n, 1, 4).contiguous()
        blocks[1, ::3] = torch.tensor([2, 1, -1, 0], dtype=torch.int32)
        blocks = blocks.to(cuda)
    elif H >= 64:
        _widen(pool, -(-2 ** 24 // (2 * n * H * bs)))
    out, lse = pool.attend(q, 0.1, blocks=blocks, want_lse=True)
    count = 0
    for b, h, t, s, vs, ks in _rows(pool, q, None if blocks is None else blocks.cpu()):
        bad = bool(torch.isnan(vs).any() | torch.isinf(vs).any())
        count += bad
        assert bool(torch.isnan(out[b, h, t]).all()) == bad and bool(torch.isfinite(out[b, h, t]).all()) != bad, (b, h, t)
        reach = float((q[b, h, t].cpu().double().abs() @ ks.abs().T * 0.1).max())
        ref = float(torch.logsumexp(s * 0.1, 0))
        assert abs(float(lse[b, h, t]) - ref) <= (d + 8) * 2.0 ** -23 * reach + 2.0 ** -17 + abs(ref) * 2.0 ** -22, (b, h, t)
    assert count == H * (8 if listed else 12)
