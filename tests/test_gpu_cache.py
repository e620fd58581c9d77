"""The 8-bit block cache's operators (ops.cache_reserve / cache_append /
cache_select / cache_attention) against a restatement in 64 bits: whole
numbers equal, outputs within bounds counted from their roundings."""
import math

import pytest
import torch

import cache_ref as R
from ssa_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


class Pool:
    """Cache buffers of B sequences, their pages scattered over the pool."""

    def __init__(self, dev, B, n_kv, d, bs, max_blocks, dtype, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.P, self.bs, self.d, self.n_kv, self.B = B * max_blocks + spare, bs, d, n_kv, B
        self.table = torch.randperm(self.P, generator=g)[:B * max_blocks].view(B, max_blocks).int().to(dev)
        fill = lambda *s: torch.randint(-127, 128, s, generator=g).to(torch.int8).to(dev)  # noqa: E731
        self.k, self.v = fill(self.P, n_kv, bs, d), fill(self.P, n_kv, bs, d)
        self.bounds = fill(self.P, n_kv, 2, d)
        self.amax = torch.rand(self.P, n_kv, 2, generator=g).to(dev) + 0.5
        self.tail = torch.randn(B, n_kv, 2, bs, d, generator=g).to(dev, dtype)
        self.start = torch.zeros(B, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(B, dtype=torch.int32, device=dev)

    def advance(self, new):
        self.start = self.lens.clone()
        self.lens = self.lens + torch.tensor(new, dtype=torch.int32, device=self.lens.device)

    def append(self, k, v, **kw):
        return ops.cache_append(k, v, self.k, self.v, self.amax, self.bounds, self.tail, self.table, self.start, self.lens, **kw)

    def attend(self, q, scale, **kw):
        return ops.cache_attention(q, self.k, self.v, self.amax, self.table, self.start, self.lens, scale, **kw)

    def select(self, q, top, **kw):
        return ops.cache_select(q, self.bounds, self.amax, self.table, self.start, self.lens, top, self.bs, **kw)

    def state(self):
        return [t.clone() for t in (self.k, self.v, self.amax, self.bounds, self.tail)]


def _kv(g, B, n, n_kv, d, dtype, dev, strided=False):
    """(B, n_kv, n, d) views of a projection's (B, n, n_kv * d) output."""
    wide = 2 if strided else 1
    w = torch.exp(torch.randn(n_kv * d * wide, generator=g))
    x = (torch.randn(B, n, n_kv * d * wide, generator=g) * w).to(dev, dtype)[..., -n_kv * d:]
    return x.unflatten(-1, (n_kv, d)).transpose(1, 2)


def _check_pages(pool, seqs):
    """Codes, amax and bounds of every sequence's pages equal the definition's."""
    k, v, am, bd, tab = (t.cpu() for t in (pool.k, pool.v, pool.amax, pool.bounds, pool.table))
    for b, s in enumerate(seqs):
        for i, (ck, cv, a) in enumerate(s.pages(pool.bs)):
            pg, n = int(tab[b, i]), ck.shape[1]
            assert torch.equal(k[pg, :, :n].double(), ck), (b, i)
            assert torch.equal(v[pg, :, :n].double(), cv), (b, i)
            assert torch.equal(am[pg], a.float())
            if n == pool.bs:
                assert torch.equal(bd[pg, :, 0].double(), ck.amin(1)) and torch.equal(bd[pg, :, 1].double(), ck.amax(1))


# ---------------------------------------------------------------- append
APPENDS = [  # dtype, n_kv, d, bs, steps: new tokens of each sequence
    (BF, 2, 128, 64, [[5, 0, 70], [1, 1, 1], [130, 64, 0], [1, 63, 59]]),
    (BF, 1, 64, 16, [[1, 15, 16], [1, 1, 1], [33, 0, 200]]),
    (F32, 2, 64, 32, [[31, 1, 32], [1, 2, 3], [100, 64, 0]]),
    (F32, 3, 32, 16, [[17, 16, 0], [16, 1, 48]]),
    (BF, 2, 96, 32, [[40, 0, 1], [1, 1, 31], [7, 90, 32]]),
    (F32, 1, 128, 64, [[129, 1, 64], [1, 127, 1]]),
]


@pytest.mark.parametrize("case", range(len(APPENDS)))
def test_append_equals_the_definition(case, cuda):
    dtype, n_kv, d, bs, steps = APPENDS[case]
    g = torch.Generator().manual_seed(case)
    B = 3
    pool = Pool(cuda, B, n_kv, d, bs, 8 if bs > 16 else 16, dtype)
    seqs = [R.Seq(n_kv, d) for _ in range(B)]
    untouched = [t.clone() for t in (pool.k, pool.v, pool.amax, pool.bounds)]
    for i, new in enumerate(steps):
        n = max(new)
        k, v = _kv(g, B, n, n_kv, d, dtype, cuda, i % 2 == 1), _kv(g, B, n, n_kv, d, dtype, cuda)
        for b in range(B):  # what stands behind a sequence's tokens is never read
            k[b, :, new[b]:] = math.nan
            v[b, :, new[b]:] = math.inf
        pool.advance(new)
        kv, vv = pool.append(k, v, want_values=True)
        for b in range(B):
            seqs[b].append(k[b, :, :new[b]].cpu(), v[b, :, :new[b]].cpu())
            assert not kv[b, :, new[b]:].any() and not vv[b, :, new[b]:].any()
            if new[b]:
                rk, rv = (t[:, -new[b]:] for t in seqs[b].values(bs))
                for mine, ref in ((kv, rk), (vv, rv)):
                    err = (mine[b, :, :new[b]].cpu().double() - ref).abs()
                    # the step's and the product's fp32 roundings, then the output's
                    assert (err <= ref.abs() * (2.0 ** -23 + torch.finfo(dtype).eps / 2 * 1.01)).all()
        _check_pages(pool, seqs)
        for b in range(B):  # the open block's tokens, as they came
            o = len(seqs[b]) % bs
            assert torch.equal(pool.tail[b, :, 0, :o].cpu().double(), seqs[b].k[:, len(seqs[b]) - o:])
            assert torch.equal(pool.tail[b, :, 1, :o].cpu().double(), seqs[b].v[:, len(seqs[b]) - o:])
    used = torch.zeros(pool.P, dtype=torch.bool)
    for b in range(B):
        used[pool.table[b, :-(-len(seqs[b]) // bs)].cpu().long()] = True
    for was, now in zip(untouched, (pool.k, pool.v, pool.amax, pool.bounds)):
        assert torch.equal(was.cpu()[~used], now.cpu()[~used])


@pytest.mark.parametrize("dtype,d,bs", [(BF, 128, 64), (F32, 64, 16)])
def test_append_token_by_token_equals_at_once(dtype, d, bs, cuda):
    g = torch.Generator().manual_seed(5)
    n, n_kv = 2 * bs + 5, 2
    k, v = _kv(g, 1, n, n_kv, d, dtype, cuda), _kv(g, 1, n, n_kv, d, dtype, cuda)
    once, each = Pool(cuda, 1, n_kv, d, bs, 4, dtype), Pool(cuda, 1, n_kv, d, bs, 4, dtype)
    once.advance([n])
    once.append(k, v)
    for i in range(n):
        each.advance([1])
        assert each.append(k[:, :, i:i + 1], v[:, :, i:i + 1]) is None
    for a, b in zip(once.state()[:4], each.state()[:4]):
        assert torch.equal(a, b)
    assert torch.equal(once.tail[:, :, :, :n % bs], each.tail[:, :, :, :n % bs])


def test_append_ties_zeros_and_extremes(cuda):
    """Quotients that are exact halves (amax 127 2^e, bf16), pages of zeros,
    an amax on both sides of 2^-80 and near the type's limits, infinities and NaN."""
    bs, d = 16, 32
    rows = torch.arange(bs * d).reshape(bs, d) % 255 - 127
    cases = [rows.double() / 2, torch.zeros(bs, d).double(), torch.full((bs, d), 2.0 ** -80).double(),
             torch.full((bs, d), 2.0 ** -81).double(), rows.double() * 2.0 ** 119, rows.double() * 2.0 ** -86]
    cases[0][0, 0] = 127.0
    special = [rows.double().clone() for _ in range(2)]
    special[0][3, 4], special[1][15, 31] = math.inf, math.nan
    for dtype in (BF, F32):
        for x in cases + special:
            x = x.to(dtype)
            pool = Pool(cuda, 1, 1, d, bs, 2, dtype)
            pool.advance([bs])
            kv, _ = pool.append(x[None, None].to(cuda), x[None, None].to(cuda), want_values=True)
            codes, amax = R.quantize(x)
            pg = int(pool.table[0, 0])
            assert torch.equal(pool.k[pg, 0].cpu().double(), codes) and torch.equal(pool.v[pg, 0].cpu().double(), codes)
            got = float(pool.amax[pg, 0, 0])
            assert got == amax or (math.isnan(got) and math.isnan(amax))
            assert bool(torch.isnan(kv).all()) == (not math.isfinite(amax))


def test_append_leaves_out_blocks_without_a_page(cuda):
    n_kv, d, bs = 1, 32, 16
    g = torch.Generator().manual_seed(1)
    pool = Pool(cuda, 2, n_kv, d, bs, 3, BF)
    pool.table[0, 1] = -1
    pool.table[1, 0] = pool.P + 5
    before = pool.state()
    k, v = _kv(g, 2, 60, n_kv, d, BF, cuda), _kv(g, 2, 60, n_kv, d, BF, cuda)
    pool.advance([40, 60])  # 60 tokens are more than the table's three blocks hold
    kv, vv = pool.append(k, v, want_values=True)
    for b, gone in ((0, range(16, 32)), (1, list(range(0, 16)) + list(range(48, 60)))):
        assert not kv[b, :, list(gone)].any() and not vv[b, :, list(gone)].any()
    for b, blk in ((0, 0), (0, 2), (1, 1), (1, 2)):
        assert kv[b, :, blk * 16:blk * 16 + 8].abs().sum() > 0
    used = {int(pool.table[b, i]) for b, i in ((0, 0), (0, 2), (1, 1), (1, 2))}
    rest = [p for p in range(pool.P) if p not in used]
    for was, now in zip(before[:4], pool.state()[:4]):
        assert torch.equal(was[rest], now[rest])


# ---------------------------------------------------------------- reserve
@pytest.mark.parametrize("B,n,bs,max_blocks,free", [(1, 1, 16, 4, 3), (5, 40, 16, 6, 9), (64, 1, 64, 32, 500),
                                                    (1500, 200, 32, 12, 4000), (33, 100, 16, 8, 0), (2100, 1, 16, 3, 1000)])
def test_reserve_equals_sequential(B, n, bs, max_blocks, free, cuda):
    g = torch.Generator().manual_seed(B)
    for in_place in (False, True):
        lens = torch.randint(0, max_blocks * bs + 1, (B,), generator=g).int()
        new = torch.randint(0, n + 1, (B,), generator=g).int()
        new[B // 2] = -3 if B > 1 else n
        table = torch.randint(0, 99, (B, max_blocks), generator=g).int()
        stack = torch.randperm(free + 5, generator=g).int()
        state = torch.tensor([free, 2], dtype=torch.int32)
        want = R.reserve(lens.tolist(), new.tolist(), table.tolist(), stack.tolist(), state.tolist(), bs)
        L, N, T, S, St = (t.to(cuda) for t in (lens, new, table, stack, state))
        out = (torch.empty_like(L), L, St) if in_place else None
        start, after, st = ops.cache_reserve(L, N, T, S, St, bs, out=out)
        assert start.tolist() == want[0] and after.tolist() == want[1] and st.tolist() == want[2]
        assert T.tolist() == want[3] and torch.equal(S.cpu(), stack)
        if in_place:
            assert after is L and st is St
        else:
            assert torch.equal(L.cpu(), lens) and torch.equal(St.cpu(), state)


@pytest.mark.parametrize("want_values", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_leaves_sequences_without_new_tokens_alone(dtype, want_values, cuda):
    """A sequence whose length stays (within a block, at its edge, empty) keeps
    its pages, bounds and tail, whatever they hold; its values are 0."""
    g = torch.Generator().manual_seed(14)
    lens = [21, 32, 0, 16 * 3 - 1, 40]
    pool = Pool(cuda, 5, 2, 64, 16, 5, dtype, seed=3)
    pool.lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    pool.start = pool.lens.clone()
    pool.start[4] = 38  # the last one gets two tokens
    pool.tail = torch.randn(pool.tail.shape, generator=g).to(dtype).to(cuda)
    before = [t.clone() for t in (pool.k, pool.v, pool.amax, pool.bounds, pool.tail)]
    x = _kv(g, 5, 2, 2, 64, dtype, cuda)
    out = pool.append(x, x, want_values=want_values)
    mine = pool.table[4].long()
    for t, old in zip((pool.k, pool.v, pool.amax, pool.bounds), before):
        t[mine] = old[mine]
        assert torch.equal(t, old)
    assert torch.equal(pool.tail[:4], before[4][:4])
    if want_values:
        assert all(float(o[:4].abs().max()) == 0 and float(o[4].abs().max()) > 0 for o in out)


# ---------------------------------------------------------------- select
SELECTS = [  # dtype, H, n_kv, d, bs, n, lens after the step, top, sink, local
    (BF, 8, 2, 128, 64, 1, [64 * 40, 1, 700], 8, 1, 1),
    (BF, 4, 4, 64, 16, 3, [500, 16, 33], 5, 0, 1),
    (F32, 6, 2, 32, 32, 2, [1000, 64, 2], 9, 2, 3),
    (F32, 33, 1, 96, 16, 1, [900, 15, 17], 4, 1, 2),
    (BF, 32, 2, 64, 16, 5, [5000, 0, 4], 16, 1, 1),
    (BF, 3, 1, 128, 32, 1, [2048, 2049, 31], 33, 4, 4),
]


@pytest.mark.parametrize("case", range(len(SELECTS)))
@pytest.mark.parametrize("flat", [False, True])
def test_select_equals_brute_force(case, flat, cuda):
    """flat: bounds and amax drawn from few values, so that many scores tie."""
    dtype, H, n_kv, d, bs, n, lens, top, sink, local = SELECTS[case]
    g = torch.Generator().manual_seed(case)
    B, mb = len(lens), -(-max(lens) // bs) + 1
    pool = Pool(cuda, B, n_kv, d, bs, mb, dtype)
    if flat:
        pool.bounds = (torch.randint(0, 2, (pool.P, n_kv, 1, 1), generator=g) * torch.tensor([-1, 1]).view(2, 1)).expand(
            pool.P, n_kv, 2, d).to(torch.int8).contiguous().to(cuda)
        pool.amax.fill_(0.75)
    else:
        pool.bounds = pool.bounds.sort(2).values
    pool.lens = torch.tensor(lens, dtype=torch.int32, device=cuda)
    pool.start = torch.tensor([max(0, x - n) for x in lens], dtype=torch.int32, device=cuda)
    pool.table[0, 3 % mb] = -1  # a block without a page is not selected
    q = _kv(g, B, n, H, d, dtype, cuda, strided=True)
    got = pool.select(q, top, sink=sink, local=local).cpu()
    assert got.shape == (B, n, n_kv, top) and got.dtype == torch.int32
    bd, am, tab = pool.bounds.cpu().double(), pool.amax.cpu().double(), pool.table.cpu()
    for b in range(B):
        st = max(0, lens[b] - n)
        for t in range(n):
            if st + t >= lens[b]:
                assert (got[b, t] == -1).all()
                continue
            pages = tab[b, :(st + t) // bs + 1].long()
            for h in range(n_kv):
                x = q[b, h * (H // n_kv):(h + 1) * (H // n_kv), t].cpu().double()
                s = R.select_scores(x, bd[pages.clamp(min=0), h], am[pages.clamp(min=0), h, 0])
                s[pages < 0] = math.nan
                want = R.top_blocks(s, top, sink, local)
                assert got[b, t, h].tolist() == want + [-1] * (top - len(want)), (b, t, h)


def test_select_bound_holds_for_every_key(cuda):
    """The score bounds q8 . k over the block's keys: every block that holds a
    key above the top-th score is listed."""
    g = torch.Generator().manual_seed(3)
    n_kv, d, bs, L = 2, 64, 16, 400
    pool = Pool(cuda, 1, n_kv, d, bs, 25, BF)
    pool.advance([L])
    k, v = _kv(g, 1, L, n_kv, d, BF, cuda), _kv(g, 1, L, n_kv, d, BF, cuda)
    pool.append(k, v)
    pool.start = torch.tensor([L - 1], dtype=torch.int32, device=cuda)
    q = _kv(g, 1, 1, 4, d, BF, cuda)
    pages = pool.table[0].long().cpu()
    for h in range(n_kv):
        x = q[0, 2 * h:2 * h + 2, 0].cpu().double()
        q8 = torch.round(x * 127 / x.abs().max())
        codes = pool.k.cpu()[pages, h].double()
        real = (codes @ q8.T).amax((1, 2)) * pool.amax.cpu()[pages, h, 0].double()
        bound = R.select_scores(x, pool.bounds.cpu()[pages, h].double(), pool.amax.cpu()[pages, h, 0].double())
        assert (real <= bound).all()
        got = pool.select(q, 6)[0, 0, h].tolist()
        assert got == R.top_blocks(bound, 6, 1, 1)


# ---------------------------------------------------------------- attention
ATTENDS = [  # dtype, H, n_kv, d, bs, n, lens after the step
    (BF, 8, 2, 128, 64, 1, [1, 64, 65, 1500, 0]),
    (F32, 8, 2, 128, 64, 1, [1, 63, 300, 7]),
    (BF, 4, 4, 64, 16, 1, [17, 16, 333]),
    (F32, 4, 4, 64, 16, 3, [17, 3, 333, 2]),
    (BF, 32, 1, 64, 32, 4, [700, 4, 33]),
    (F32, 9, 1, 32, 16, 2, [129, 2]),
    (BF, 6, 2, 96, 32, 5, [200, 31, 0]),
    (F32, 40, 1, 96, 64, 1, [90, 1000]),
    (BF, 8, 8, 32, 16, 70, [300, 70, 75]),
    (BF, 16, 2, 128, 64, 19, [200, 1, 64]),
    (F32, 12, 4, 128, 32, 11, [64, 100]),
    # the many-row kernel (64 rows a kv head and more, and a wide table)
    (BF, 4, 1, 64, 32, 16, [500, 16, 65]),
    (BF, 6, 2, 96, 32, 40, [200, 41, 0]),
    (BF, 32, 1, 128, 16, 5, [1000, 5, 64]),
    (BF, 4, 2, 64, 64, 300, [1100, 300, 17]),
    (BF, 3, 1, 32, 32, 33, [65, 2000]),
    (BF, 16, 1, 128, 64, 6, [640, 3000, 6, 0]),
]
MANY_ROWS = len(ATTENDS) - 6  # cases from here on


def _widen(pool, blocks):
    """The table with more columns, without pages."""
    pool.table = torch.nn.functional.pad(pool.table, (0, blocks - pool.table.shape[1]), value=-1).contiguous()


def _filled(case, cuda, seed=0, spread=1.0):
    dtype, H, n_kv, d, bs, n, lens = ATTENDS[case]
    g = torch.Generator().manual_seed(100 + case + seed)
    pool = Pool(cuda, len(lens), n_kv, d, bs, -(-max(lens) // bs) + 1, dtype, seed=case)
    if case >= MANY_ROWS:
        _widen(pool, -(-2 ** 24 // (len(lens) * n * H * bs)))
    k, v = _kv(g, len(lens), max(lens), n_kv, d, dtype, cuda), _kv(g, len(lens), max(lens), n_kv, d, dtype, cuda)
    k = k * spread
    pool.advance(lens)
    pool.append(k, v)
    pool.start = torch.tensor([max(0, x - n) for x in lens], dtype=torch.int32, device=cuda)
    return pool, _kv(g, len(lens), n, H, d, dtype, cuda, strided=True)


def _held(pool, b, length):
    """k, v (n_kv, length, d) float64 as the codes in the pool stand for them."""
    bs = pool.bs
    pages = pool.table[b, :-(-length // bs)].long().cpu().clamp(0, pool.P - 1)
    am = pool.amax.cpu()[pages].double()
    out = []
    for i, c in enumerate((pool.k, pool.v)):
        x = c.cpu()[pages].double() * (am[..., i] / 127)[..., None, None]
        out.append(x.transpose(0, 1).reshape(pool.n_kv, -1, pool.d)[:, :length])
    return out


def _check_attention(pool, q, out, lse, scale, blocks=None, causal=True):
    B, H, n, d = q.shape
    rep = H // pool.n_kv
    start, lens = pool.start.tolist(), pool.lens.tolist()
    assert out.shape == q.shape and out.dtype == q.dtype
    qc, oc, lc = q.cpu().double(), out.cpu().double(), lse.cpu().double()
    for b in range(B):
        fresh = max(0, min(n, lens[b] - start[b]))
        assert not oc[b, :, fresh:].any() and (lc[b, :, fresh:] == -math.inf).all()
        if not fresh:
            continue
        k, v = _held(pool, b, lens[b])
        pos = torch.arange(lens[b])
        for h in range(H):
            seen = (pos[None] <= start[b] + torch.arange(fresh)[:, None]) if causal else torch.ones(fresh, lens[b], dtype=torch.bool)
            page = pool.table[b].cpu()[pos // pool.bs]
            seen = seen & ((page >= 0) & (page < pool.P))
            if blocks is not None:
                listed = torch.zeros(fresh, lens[b], dtype=torch.bool)
                for t in range(fresh):
                    for e in blocks[b, t, h // rep].tolist():
                        if 0 <= e < pool.table.shape[1]:
                            listed[t, e * pool.bs:(e + 1) * pool.bs] = True
                seen = seen & listed
            ref, rl, vmax, reach = R.attend(qc[b, h, :fresh], k[h // rep], v[h // rep], seen, scale)
            tol = R.attention_tolerance(ref, vmax, reach, q.dtype, d, lens[b])
            err = (oc[b, h, :fresh] - ref).abs()
            assert (err <= tol).all(), (b, h, float((err / tol).max()))
            empty = rl == -math.inf
            assert torch.equal(empty, lc[b, h, :fresh] == -math.inf)
            # the lse moves by at most the scores' error and the sum's roundings (2^-20 of 1), then fp32
            lt = (d + 8) * 2.0 ** -23 * reach + 2.0 ** -19 + rl.abs() * 2.0 ** -22
            assert ((lc[b, h, :fresh] - rl).abs()[~empty] <= lt[~empty]).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_over_every_block(case, causal, cuda):
    pool, q = _filled(case, cuda)
    scale = pool.d ** -0.5
    out, lse = pool.attend(q, scale, causal=causal, want_lse=True)
    _check_attention(pool, q, out, lse, scale, causal=causal)
    again = pool.attend(q, scale, causal=causal)
    assert torch.equal(out, again)


@pytest.mark.parametrize("case", range(len(ATTENDS)))
def test_attention_over_listed_blocks(case, cuda):
    """Lists in any order, with holes, entries out of range, blocks behind the
    token, and none at all."""
    pool, q = _filled(case, cuda)
    B, H, n, d = q.shape
    g = torch.Generator().manual_seed(case)
    mb, scale = -(-max(ATTENDS[case][6]) // pool.bs) + 1, d ** -0.5
    for top in (1, 3, 7):
        blocks = torch.stack([torch.randperm(mb + 6, generator=g)[:min(top, mb)] - 3 for _ in range(B * n * pool.n_kv)])
        blocks = torch.nn.functional.pad(blocks, (0, top - blocks.shape[1]), value=-1).view(B, n, pool.n_kv, top)
        blocks[0, 0, 0] = -1
        out, lse = pool.attend(q, scale, blocks=blocks.int().to(cuda), want_lse=True)
        _check_attention(pool, q, out, lse, scale, blocks=blocks)


@pytest.mark.parametrize("case", [0, 1, 4, 9, 12, 15])
def test_attention_skips_blocks_without_a_page(case, cuda):
    pool, q = _filled(case, cuda)
    pool.table[:, 0] = -1
    pool.table[-1, 1] = pool.P
    out, lse = pool.attend(q, 0.2, want_lse=True)
    _check_attention(pool, q, out, lse, 0.2)


@pytest.mark.parametrize("dtype,d,rep", [(BF, 128, 4), (F32, 64, 4), (BF, 64, 100)])
def test_attention_sharp_and_far_scores(dtype, d, rep, cuda):
    """Scores that grow along the cache (the running offset moves all the way),
    a single dominating key, and pages of very different steps, one of zeros."""
    n_kv, bs, L = 1, 16, 400
    g = torch.Generator().manual_seed(9)
    k, v = _kv(g, 1, L, n_kv, d, dtype, cuda), _kv(g, 1, L, n_kv, d, dtype, cuda)
    q = _kv(g, 1, 1, rep, d, dtype, cuda)
    ramp = torch.linspace(-40, 40, L, device=cuda).view(1, 1, L, 1)
    k1 = (q[:, :1, :1] * ramp / (q[:, :1, :1].float() ** 2).sum() * d ** 0.5).to(dtype)
    steps = (2.0 ** torch.randint(-30, 30, (L // bs,), generator=g).double()).float().repeat_interleave(bs).to(cuda)
    v2 = (v.float() * steps.view(1, 1, L, 1)).to(dtype)
    v2[:, :, bs:2 * bs] = 0
    for kk, vv in ((k1, v), (k1.flip(2), v), (k, v2), (k * 30, v), (k * 0, v)):
        pool = Pool(cuda, 1, n_kv, d, bs, L // bs, dtype)
        if rep >= 96:
            _widen(pool, -(-2 ** 24 // (rep * bs)))
        pool.advance([L])
        pool.append(kk.contiguous(), vv)
        pool.start = torch.tensor([L - 1], dtype=torch.int32, device=cuda)
        out, lse = pool.attend(q, d ** -0.5, want_lse=True)
        _check_attention(pool, q, out, lse, d ** -0.5)


@pytest.mark.parametrize("rep", [2, 128])
@pytest.mark.parametrize("bad,value", [("k", math.nan), ("k", math.inf), ("v", math.nan), ("v", -math.inf)])
def test_attention_keeps_nan_and_infinity_where_they_are(bad, value, rep, cuda):
    """A sequence with a page of NaN or infinity or an infinite q gives NaN; the
    others, and stale pages behind a length, do not see it."""
    n_kv, d, bs = 1, 64, 16
    g = torch.Generator().manual_seed(2)
    pool = Pool(cuda, 3, n_kv, d, bs, 4, BF)
    k, v = _kv(g, 3, 40, n_kv, d, BF, cuda), _kv(g, 3, 40, n_kv, d, BF, cuda)
    (k if bad == "k" else v)[1, 0, 20, 3] = value
    pool.advance([40, 40, 40])
    pool.append(k, v)
    pool.amax[pool.table[:, 3].long()] = math.nan  # behind every length
    if rep >= 96:
        _widen(pool, -(-2 ** 24 // (3 * rep * bs)))
    pool.start = pool.lens - 1
    q = _kv(g, 3, 1, rep, d, BF, cuda)
    q[2, 1, 0, 5] = math.inf
    out, lse = pool.attend(q, 0.125, want_lse=True)
    assert torch.isnan(out[1]).all() and torch.isnan(out[2, 1]).all()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[2, 0]).all()
    assert torch.isfinite(lse[0]).all()


def test_attention_long_ragged_batch_splits_evenly(cuda):
    """Many and few units per thread block: outputs equal those of the
    sequences alone up to the joins' order."""
    n_kv, d, bs = 2, 128, 64
    g = torch.Generator().manual_seed(4)
    lens = [9000, 1, 130, 4000, 64, 0, 2500]
    pool = Pool(cuda, len(lens), n_kv, d, bs, -(-max(lens) // bs), BF)
    k, v = _kv(g, len(lens), max(lens), n_kv, d, BF, cuda), _kv(g, len(lens), max(lens), n_kv, d, BF, cuda)
    pool.advance(lens)
    pool.append(k, v)
    pool.start = (pool.lens - 1).clamp(min=0)
    q = _kv(g, len(lens), 1, 8, d, BF, cuda)
    out, lse = pool.attend(q, d ** -0.5, want_lse=True)
    _check_attention(pool, q, out, lse, d ** -0.5)
    for b in range(len(lens)):
        alone = ops.cache_attention(q[b:b + 1], pool.k, pool.v, pool.amax, pool.table[b:b + 1].contiguous(),
                                    pool.start[b:b + 1], pool.lens[b:b + 1], d ** -0.5)
        # the same sums in another grouping: bf16 outputs at most one step apart, and that of the weights' roundings
        assert ((alone[0].float() - out[b].float()).abs() <= 2.0 ** -7 * out[b].float().abs() + 2.0 ** -10).all()


# ---------------------------------------------------------------- together
def test_captured_decode_step(cuda):
    """reserve, append, select and attention recorded once and replayed, with
    in-place lengths: every replay equals the eager operators'."""
    B, H, n_kv, d, bs, mb, top = 3, 4, 2, 64, 16, 8, 3
    g = torch.Generator().manual_seed(6)
    two = []
    for _ in range(2):
        p = Pool(cuda, B, n_kv, d, bs, mb, BF)
        p.free = torch.arange(p.P, dtype=torch.int32, device=cuda).flip(0).contiguous()
        p.count = torch.tensor([p.P, 0], dtype=torch.int32, device=cuda)
        p.table.fill_(-1)
        two.append(p)
    one = torch.ones(B, dtype=torch.int32, device=cuda)
    q, k, v = (torch.zeros(B, h, 1, d, dtype=BF, device=cuda) for h in (H, n_kv, n_kv))

    def step(p):
        ops.cache_reserve(p.lens, one, p.table, p.free, p.count, bs, out=(p.start, p.lens, p.count))
        p.append(k, v)
        blocks = p.select(q, top)
        return p.attend(q, 0.125, blocks=blocks, want_lse=True) + (blocks,)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(two[1])
    torch.cuda.current_stream().wait_stream(side)
    p = two[1]
    p.lens.zero_(), p.table.fill_(-1), p.count.copy_(torch.tensor([p.P, 0]))
    for x, y in zip((p.k, p.v, p.amax, p.bounds, p.tail), two[0].state()):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        held = step(p)
    p.lens.zero_(), p.table.fill_(-1), p.count.copy_(torch.tensor([p.P, 0]))
    for i in range(60):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        want = step(two[0])
        for a, b in zip(held, want):
            assert torch.equal(a, b), i
        assert torch.equal(p.lens, two[0].lens) and torch.equal(p.table, two[0].table)
    assert int(p.lens[0]) == 60 and p.count.tolist() == [p.P - B * 4, 0]
    for a, b in zip(two[0].state(), p.state()):
        assert torch.equal(a, b)
    assert _lib.load().ssa_device_error(1) == 0


def test_attention_many_sums_a_row(cuda):
    """Few units over the whole GPU: a row's partial sums come from tens of
    thread blocks, by one warp a row and by four."""
    for H, n_kv, n, d, dtype in ((2, 1, 1, 64, BF), (4, 2, 1, 128, F32), (8, 1, 90, 64, BF), (32, 1, 64, 32, BF)):
        g = torch.Generator().manual_seed(8)
        L = 9000
        pool = Pool(cuda, 1, n_kv, d, 64, -(-L // 64), dtype)
        pool.advance([L])
        pool.append(_kv(g, 1, L, n_kv, d, dtype, cuda), _kv(g, 1, L, n_kv, d, dtype, cuda))
        pool.start = pool.lens - n
        q = _kv(g, 1, n, H, d, dtype, cuda)
        out, lse = pool.attend(q, d ** -0.5, want_lse=True)
        assert torch.equal(out, pool.attend(q, d ** -0.5))
        few = [0, n - 1] if n > 1 else [0]  # two tokens' rows are enough to compare
        sub = Pool.__new__(Pool)
        sub.__dict__.update(pool.__dict__)
        for t in few:
            sub.start, sub.lens = pool.start + t, pool.start + t + 1
            _check_attention(sub, q[:, :, t:t + 1], out[:, :, t:t + 1], lse[:, :, t:t + 1], d ** -0.5)


def test_many_row_kernel_repeats(cuda):
    """Back to back calls of the many-row kernel, whose warps hand blocks of
    keys to one another: the same bits every time, and no wait that ran out."""
    pool, q = _filled(len(ATTENDS) - 1, cuda)
    want = pool.attend(q, 0.1)
    differ = torch.zeros((), device=cuda)
    for _ in range(300):
        differ += (pool.attend(q, 0.1) != want).any()
    assert float(differ) == 0 and _lib.load().ssa_device_error(1) == 0


def test_many_row_kernel_wait_that_runs_out(cuda):
    """A wait given a single poll gives up: the kernel ends, reports its code and
    leaves the GPU usable."""
    L = _lib.load()
    pool, q = _filled(len(ATTENDS) - 1, cuda)
    want = pool.attend(q, 0.1)
    assert L.ssa_device_error(1) == 0
    L.ssa_debug_set_wait_limit(1)
    try:
        pool.attend(q, 0.1)
        torch.cuda.synchronize()
        assert L.ssa_device_error(1) != 0
    finally:
        L.ssa_debug_set_wait_limit(0)
    assert torch.equal(pool.attend(q, 0.1), want) and L.ssa_device_error(1) == 0


@pytest.mark.parametrize("n", [1, 100])
def test_offsets_beyond_32_bits(n, cuda):
    """Pages whose codes lie past 2^31 bytes, bounds past 2^31 / 32, against the
    same sequences in the first pages."""
    n_kv, d, bs, H, B, L = 16, 128, 64, 32, 2, 200
    P = 2 ** 31 // (n_kv * bs * d) + 40
    g = torch.Generator().manual_seed(12)
    far = Pool.__new__(Pool)
    far.P, far.bs, far.d, far.n_kv, far.B = P, bs, d, n_kv, B
    far.k, far.v = (torch.empty(P, n_kv, bs, d, dtype=torch.int8, device=cuda) for _ in range(2))
    far.bounds = torch.empty(P, n_kv, 2, d, dtype=torch.int8, device=cuda)
    far.amax = torch.empty(P, n_kv, 2, device=cuda)
    far.tail = torch.zeros(B, n_kv, 2, bs, d, dtype=BF, device=cuda)
    far.start, far.lens = (torch.zeros(B, dtype=torch.int32, device=cuda) for _ in range(2))
    far.table = (P - 1 - torch.arange(8, device=cuda)).view(B, 4).int().contiguous()
    near = Pool(cuda, B, n_kv, d, bs, 4, BF)
    k, v = _kv(g, B, L, n_kv, d, BF, cuda), _kv(g, B, L, n_kv, d, BF, cuda)
    q = _kv(g, B, n, H, d, BF, cuda)
    got = []
    for p in (far, near):
        p.advance([L, L - 70])
        p.append(k, v)
        p.start = p.lens - n
        blocks = p.select(q, 3)
        if n > 1:
            _widen(p, -(-2 ** 24 // (B * n * H * bs)))  # the many-row kernel
        whole = p.table[:, :(L - 70) // bs].long()  # pages complete in both sequences: the rest of a page keeps what it held
        got.append((blocks, p.attend(q, 0.1), p.attend(q, 0.1, blocks=blocks), p.k[whole], p.v[whole], p.bounds[whole], p.amax[whole]))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [1, 24])
def test_attention_of_many_sequences(n, cuda):
    """More sequences than a thread block has threads; n = 24 with a wide table
    is the many-row kernel's."""
    B, n_kv, H, d, bs = 700, 1, 3, 32, 16
    g = torch.Generator().manual_seed(13)
    lens = torch.randint(0, 60, (B,), generator=g).tolist()
    pool = Pool(cuda, B, n_kv, d, bs, 4, BF)
    pool.advance(lens)
    pool.append(_kv(g, B, 60, n_kv, d, BF, cuda), _kv(g, B, 60, n_kv, d, BF, cuda))
    pool.start = (pool.lens - n).clamp(min=0)
    if n > 1:
        _widen(pool, 24)
    q = _kv(g, B, n, H, d, BF, cuda)
    out, lse = pool.attend(q, 0.2, want_lse=True)
    _check_attention(pool, q, out, lse, 0.2)


def test_gradients_are_refused(cuda):
    pool, q = _filled(0, cuda)
    want = pool.attend(q, 0.1)
    k = torch.randn(pool.B, pool.n_kv, 1, pool.d, device=cuda, dtype=BF, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradient"):
        pool.attend(q.clone().requires_grad_(), 0.1)
    with pytest.raises(RuntimeError, match="no gradient"):
        pool.append(k, k.detach())
    with pytest.raises(RuntimeError, match="no gradient"):
        pool.append(k.detach(), k)
    with torch.no_grad():
        assert torch.equal(pool.attend(q.clone().requires_grad_(), 0.1), want)


def test_other_stream(cuda):
    pool, q = _filled(0, cuda)
    want = pool.attend(q, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pool.attend(q, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(want, got)
