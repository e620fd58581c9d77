"""The 8-bit block cache in 64 bits, written from its definition: what the
GPU tests of ssa_b200's cache operators are compared with."""
import math

import torch


def quantize(x):
    """Codes (float64 whole numbers) and amax of one page's tokens of one head:
    x (tokens, d). An amax below 2^-80 counts as zero; one that is not finite
    leaves codes 0 and stands for NaN."""
    x = x.double()
    amax = float(x.abs().max()) if not bool(torch.isnan(x).any()) else math.nan
    if not amax >= 2.0 ** -80 and not math.isnan(amax):
        return torch.zeros_like(x), 0.0
    if not math.isfinite(amax):
        return torch.zeros_like(x), amax
    return torch.round(x * 127 / amax), amax  # 127 x is exact in 64 bits, the quotient within 2^-53


class Seq:
    """One sequence's keys and values as they came: k, v (n_kv, tokens, d)."""

    def __init__(self, n_kv, d):
        self.k = torch.zeros(n_kv, 0, d, dtype=torch.float64)
        self.v = torch.zeros(n_kv, 0, d, dtype=torch.float64)

    def append(self, k, v):
        self.k = torch.cat([self.k, k.double().cpu()], 1)
        self.v = torch.cat([self.v, v.double().cpu()], 1)

    def __len__(self):
        return self.k.shape[1]

    def pages(self, bs):
        """[(codes_k, codes_v (n_kv, <= bs, d), amax (n_kv, 2))] of its blocks."""
        out = []
        for p0 in range(0, len(self), bs):
            ck, ak = zip(*[quantize(self.k[h, p0:p0 + bs]) for h in range(self.k.shape[0])])
            cv, av = zip(*[quantize(self.v[h, p0:p0 + bs]) for h in range(self.k.shape[0])])
            out.append((torch.stack(ck), torch.stack(cv), torch.tensor([ak, av], dtype=torch.float64).T))
        return out

    def values(self, bs):
        """k, v (n_kv, tokens, d) as the codes stand for them."""
        ks, vs = [], []
        for ck, cv, am in self.pages(bs):
            ks.append(ck * (am[:, 0] / 127)[:, None, None])
            vs.append(cv * (am[:, 1] / 127)[:, None, None])
        return torch.cat(ks, 1), torch.cat(vs, 1)


def reserve(lens, new, table, free, state, bs):
    """Sequential restatement; returns (start, lens, state, table)."""
    lens, table = [max(0, x) for x in lens], [list(r) for r in table]
    count, refused = state
    start, asked = list(lens), 0
    given = 0
    for b, n in enumerate(new):
        n = max(0, n)
        held, want = -(-lens[b] // bs), -(-(lens[b] + n) // bs)
        if want > len(table[b]):
            refused += 1
            continue
        need = want - held
        if need and asked + need > count:
            refused += 1
            asked += need
            continue
        for j in range(need):
            table[b][held + j] = free[count - 1 - asked - j]
        asked += need
        given += need
        lens[b] += n
    return start, lens, [count - given, refused], table


def select_scores(q, pages_bounds, amax):
    """Scores (blocks,) of one token and kv head: q (rep, d), bounds (blocks,
    2, d), amax (blocks,), all float64."""
    a = q.abs().max()
    q8 = torch.round(q * 127 / a) if a >= 2.0 ** -80 else torch.zeros_like(q)
    s = torch.maximum(q8[None] * pages_bounds[:, None, 0], q8[None] * pages_bounds[:, None, 1]).sum(-1)
    return s.max(1).values * amax


def top_blocks(scores, top, sink, local):
    """Ascending block numbers; scores of blocks without a page are NaN."""
    n = len(scores)
    key = {}
    for i, s in enumerate(scores.tolist()):
        if not math.isnan(s):
            key[i] = math.inf if i < sink or i >= n - local else s
    return sorted(sorted(key, key=lambda i: (-key[i], i))[:top])


def attend(q, k, v, seen, scale):
    """One head's rows: q (rows, d), k, v (keys, d), seen (rows, keys) bool.
    Returns out, lse, and for tolerances max |v| seen and max sum_c |q k|."""
    s = q.double() @ k.T * scale
    s = s.masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(seen, torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None]), torch.zeros_like(s))
    vmax = (seen[..., None] * v.abs()[None]).amax((1, 2)) if k.shape[0] else torch.zeros(q.shape[0], dtype=torch.float64)
    reach = torch.where(seen, q.double().abs() @ k.abs().T * scale, torch.zeros_like(s))
    return p @ v, lse, vmax, reach.amax(-1) if k.shape[0] else torch.zeros(q.shape[0], dtype=torch.float64)


def attention_tolerance(ref, vmax, reach, dtype, d, keys, pieces_join=32):
    """Bound of |out - ref| for (rows, d) rows.

    A score is a chain of d / 16 tensor sums of 16 products and a few fp32
    factors: its error is at most (d + 8) 2^-23 of sum |q k| (natural-log
    units), twice that after the normalisation. A weight is rounded to fp16
    (2^-11; fp32 tensors: to 22 bits, 2^-21 with its remainder's own rounding)
    and 2^x is good to 2^-21. The output is a chain of keys / 64 tensor sums in
    each warp and `pieces_join` joins; each step rounds at 2^-23 of sum p |v|
    <= max |v|. Then one rounding to the output's type."""
    half = torch.finfo(dtype).eps / 2
    weight = 2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -21
    rel = 2 * (d + 8) * 2.0 ** -23 * reach + 2 * (weight + 2.0 ** -21) + (keys / 64 + 16 + pieces_join) * 2.0 ** -23
    return half * ref.abs() * (1 + 2.0 ** -7) + (rel * vmax)[..., None] + 1e-30
