"""Cases of the 8-bit block cache: pages reserved from request lengths, keys
and values appended in 8 bits, blocks selected for each query token, and
attention over all or the selected blocks of the cache.

A cache of one layer is a pool of pages of `bs` tokens: codes int8 (P, n_kv,
bs, d) for keys and values, amax fp32 (P, n_kv, 2) -- a code c stands for
c * amax / 127 -- and bounds int8 (P, n_kv, 2, d), the least and greatest key
code of every channel of a complete page. table (B, max_blocks) maps a
sequence's blocks to pages; tail (B, n_kv, 2, bs, d) keeps the open block's
tokens as they came. start and lens (B,) are the lengths before and after the
current step's tokens."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
TINY = 2.0 ** -80  # a smaller amax counts as zero


# ---------------------------------------------------------------- cases
def listed():
    return [
        # One decoding step of 64 requests: most need no page, some one.
        {"name": "reserve_step", "op": "reserve", "B": 64, "n": 1, "bs": 64, "max_blocks": 512},
        # Admission of 1024 prompts of up to 2048 tokens into small pages, the pool not large enough for all.
        {"name": "reserve_prompts", "op": "reserve", "B": 1024, "n": 2048, "bs": 16, "max_blocks": 512},
        # One token for each of 32 sequences (GQA 32/8, d 128): the decoding step's write.
        {"name": "append_token", "op": "append", "B": 32, "n": 1, "n_kv": 8, "d": 128, "bs": 64, "dtype": "bf16", "past": 8192},
        # Ragged prompts of up to 8192 tokens.
        {"name": "append_prompts", "op": "append", "B": 16, "n": 8192, "n_kv": 8, "d": 128, "bs": 64, "dtype": "bf16", "past": 0},
        # An fp32 model's prompt chunk behind a short past, odd lengths.
        {"name": "append_chunk_fp32", "op": "append", "B": 2, "n": 1023, "n_kv": 8, "d": 64, "bs": 32, "dtype": "fp32", "past": 77},
        # Latency: one token of one sequence chooses 16 of 128 blocks.
        {"name": "select_one", "op": "select", "B": 1, "n": 1, "H": 32, "n_kv": 8, "d": 128, "bs": 64, "dtype": "bf16", "past": 8191, "top": 16},
        # A batch at long context: 64 of 1024 blocks.
        {"name": "select_batch_long", "op": "select", "B": 32, "n": 1, "H": 32, "n_kv": 8, "d": 128, "bs": 32, "dtype": "bf16", "past": 32768, "top": 64},
        # Latency: a short fp32 context.
        {"name": "attend_short_fp32", "op": "attend", "B": 1, "n": 1, "H": 8, "n_kv": 8, "d": 64, "bs": 16, "dtype": "fp32", "past": 333, "top": 0},
        # The ordinary decoding step: 32 ragged sequences of up to 8192 tokens.
        {"name": "attend_batch", "op": "attend", "B": 32, "n": 1, "H": 32, "n_kv": 8, "d": 128, "bs": 64, "dtype": "bf16", "past": 8192, "top": 0},
        # Four draft tokens a sequence on a multi-query model: 128 rows a key head.
        {"name": "attend_mqa_drafts", "op": "attend", "B": 8, "n": 4, "H": 32, "n_kv": 1, "d": 64, "bs": 32, "dtype": "bf16", "past": 8192, "top": 0},
        # A prompt chunk of 256 tokens behind a cached prefix.
        {"name": "attend_chunk", "op": "attend", "B": 2, "n": 256, "H": 32, "n_kv": 8, "d": 128, "bs": 64, "dtype": "bf16", "past": 7936, "top": 0},
        # Selected blocks of a long context: 64 of up to 512 blocks for each of 16 sequences.
        {"name": "attend_blocks_long", "op": "attend", "B": 16, "n": 1, "H": 32, "n_kv": 8, "d": 128, "bs": 64, "dtype": "bf16", "past": 32768, "top": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["reserve", "append", "append", "select", "select", "attend", "attend", "attend", "attend"])
    bs = rng.choice([16, 32, 64])
    if op == "reserve":
        return {"op": op, "B": _log(rng, 1, 1024), "n": _log(rng, 1, 2048), "bs": bs, "max_blocks": rng.choice([257, 512])}
    H, n_kv = rng.choice([(8, 8), (32, 8), (16, 16), (32, 1), (16, 4), (6, 2)])
    c = {"op": op, "n_kv": n_kv, "d": rng.choice([32, 64, 128]), "bs": bs, "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    if op == "append":
        c["n"] = _log(rng, 1, 4096)
        c["B"] = _log(rng, 1, max(1, min(32, (1 << 25) // (c["n"] * n_kv * c["d"]))))
        c["past"] = rng.choice([0, _log(rng, 1, 4096)])
        return c
    c["H"], c["past"] = H, _log(rng, 1, 32768)
    if op == "select":
        c["n"] = _log(rng, 1, 8)
        c["B"] = _log(rng, 1, max(1, min(32, (1 << 28) // (c["past"] * n_kv * c["d"] * c["n"]))))
        c["top"] = rng.choice([8, 16, 33, 64, 128])
        return c
    c["top"] = rng.choice([0, 0, 8, 31, 64])
    c["n"] = _log(rng, 1, 8 if c["top"] else 128)
    keys = max(c["past"], c["top"] * bs * c["n"])
    c["B"] = _log(rng, 1, max(1, min(32, (1 << 26) // (keys * n_kv * c["d"]), (1 << 23) // (c["past"] * c["n"]))))
    return c


# ---------------------------------------------------------------- inputs
def _lengths(g, B, past, dev):
    """Ragged lengths in [past / 2, past], the first one `past` itself."""
    r = torch.rand(B, generator=g, device=dev)
    lens = (past * (0.5 + 0.5 * r)).round().to(torch.int32)
    lens[0] = past
    return lens


def _lens(case, g, dev):
    """Lengths before and after the step's tokens: new tokens are ragged too when there are several."""
    start = _lengths(g, case["B"], case["past"], dev)
    new = torch.full_like(start, case["n"])
    if case["n"] > 1 and case["B"] > 1:
        new = _lengths(g, case["B"], case["n"], dev)
        new[-1] = case["n"] // 3
    return start, (start + new).to(torch.int32)


def _table(case, g, dev):
    nb = (case["past"] + case["n"] + case["bs"] - 1) // case["bs"]
    P = case["B"] * nb + 3
    perm = torch.randperm(P, generator=g, device=dev)[: case["B"] * nb]
    return perm.view(case["B"], nb).to(torch.int32), P


def _codes(g, P, case, dev):
    t = torch.randn(P, case["n_kv"], case["bs"], case["d"], generator=g, device=dev, dtype=torch.bfloat16)
    return t.mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)


def _rows(g, B, n, heads, d, dtype, dev):
    """(B, heads, n, d) view of a projection's (B, n, heads * d) output: channels of unequal size, as keys have."""
    x = torch.randn(B, n, heads * d, generator=g, device=dev)
    w = torch.exp(0.5 * torch.randn(heads * d, generator=g, device=dev))
    return (x * w).to(DTYPES[dtype]).view(B, n, heads, d).transpose(1, 2)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    op = case["op"]
    s = {"op": op, "bs": case["bs"]}
    if op == "reserve":
        B, mb = case["B"], case["max_blocks"]
        new = torch.randint(0, case["n"] + 1, (B,), generator=g, device=dev) if case["n"] > 1 else torch.ones(B, dtype=torch.int64, device=dev)
        past = max(1, (mb - 1) * case["bs"] - case["n"] // 2)  # a few sequences run out of their table's width
        lens = torch.randint(0, past + 1, (B,), generator=g, device=dev)
        held = (lens + case["bs"] - 1) // case["bs"]
        P = int(held.sum()) + max(8, int(0.9 * B * (case["n"] / 2 + case["bs"]) / case["bs"]))
        perm = torch.randperm(P, generator=g, device=dev).to(torch.int32)
        col = torch.arange(mb, device=dev)
        first = held.cumsum(0) - held
        table = torch.where(col < held[:, None], perm[(first[:, None] + col).clamp(max=P - 1)], -1)
        used = int(held.sum())
        s["free"] = torch.cat([perm[used:], perm[:used]]).contiguous()
        s["state"] = torch.tensor([P - used, 0], dtype=torch.int32, device=dev)
        return s | {"lens": lens.to(torch.int32), "new": new.to(torch.int32), "table": table.to(torch.int32).contiguous()}
    B, n, n_kv, d = case["B"], case["n"], case["n_kv"], case["d"]
    s["start"], s["lens"] = _lens(case, g, dev)
    s["table"], P = _table(case, g, dev)
    s["amax"] = torch.exp(0.3 * torch.randn(P, n_kv, 2, generator=g, device=dev)) * 3.5
    if op == "select":
        mid = torch.randn(P, n_kv, d, generator=g, device=dev) * 30
        spread = torch.rand(P, n_kv, 2, d, generator=g, device=dev) * 60
        s["bounds"] = torch.stack([mid - spread[:, :, 0], mid + spread[:, :, 1]], 2).round().clamp(-127, 127).to(torch.int8)
        s["top"] = case["top"]
        return s | {"q": _rows(g, B, n, case["H"], d, case["dtype"], dev)}
    if op == "append":
        s["k"], s["v"] = (_rows(g, B, n, n_kv, d, case["dtype"], dev) for _ in range(2))
        s["k_codes"], s["v_codes"] = (torch.zeros(P, n_kv, case["bs"], d, dtype=torch.int8, device=dev) for _ in range(2))
        s["bounds"] = torch.zeros(P, n_kv, 2, d, dtype=torch.int8, device=dev)
        s["tail"] = torch.randn(B, n_kv, 2, case["bs"], d, generator=g, device=dev).to(DTYPES[case["dtype"]])
        return s
    s["k_codes"], s["v_codes"] = _codes(g, P, case, dev), _codes(g, P, case, dev)
    s["q"] = _rows(g, B, n, case["H"], d, case["dtype"], dev)
    s["scale"] = d ** -0.5
    s["blocks"] = None
    if case["top"]:
        # Distinct blocks in ascending order, as the selection gives them; the token's own among them, -1 behind.
        nb = s["table"].shape[1]
        pos = s["start"][:, None, None].long() + torch.arange(n, device=dev)[None, :, None]
        own_block = (pos // case["bs"]).expand(B, n, n_kv)
        key = torch.rand(B, n, n_kv, nb, generator=g, device=dev)
        col = torch.arange(nb, device=dev)
        key = torch.where(col > own_block[..., None], -1.0, torch.where(col == own_block[..., None], 2.0, key))
        order = key.sort(-1, descending=True).indices[..., : case["top"]]
        taken = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, order, True) & (key >= 0)
        taken &= (pos < s["lens"][:, None, None])[..., None]
        s["blocks"] = _ascending(taken, case["top"])
    return s


# ---------------------------------------------------------------- plain forms
def _ascending(taken, top):
    """Indices of the true entries of the last axis in ascending order, -1 behind, `top` wide."""
    nb = taken.shape[-1]
    idx = torch.where(taken, torch.arange(nb, device=taken.device), nb).sort(-1).values
    idx = torch.nn.functional.pad(idx, (0, max(0, top - nb)), value=nb)[..., :top]
    return torch.where(idx < nb, idx, -1).to(torch.int32)


def _reserve(s):
    lens, new, table, free, bs = s["lens"].long(), s["new"].long(), s["table"], s["free"], s["bs"]
    count = s["state"][0].long()
    held = (lens + bs - 1) // bs
    want = (lens + new + bs - 1) // bs
    wide = want > table.shape[1]
    need = torch.where(wide, 0, want - held)
    upto = need.cumsum(0)
    ok = ~wide & ((need == 0) | (upto <= count))
    given = torch.where(ok, need, 0)
    col = torch.arange(table.shape[1], device=table.device)
    here = ok[:, None] & (col >= held[:, None]) & (col < want[:, None])
    at = count - 1 - ((upto - need)[:, None] + col - held[:, None])
    table.copy_(torch.where(here, free[at.clamp(0, free.numel() - 1)], table))
    after = torch.where(ok, lens + new, lens).to(torch.int32)
    state = torch.stack([count - given.sum(), s["state"][1] + (~ok).sum()]).to(torch.int32)
    return s["lens"], after, state, table


def _quantize(x, amax):
    return torch.where(amax > 0, x.double() * 127 / torch.where(amax > 0, amax, 1.0).double(), 0.0).round().to(torch.int8)


def _append(s):
    k, table, bs = s["k"], s["table"], s["bs"]
    B, n_kv, n, d = k.shape
    dev, P, nb = k.device, s["amax"].shape[0], table.shape[1]
    start, lens = s["start"].long(), s["lens"].long()
    first = start // bs
    nt = (n + bs - 2) // bs + 1  # blocks that n tokens can touch
    pos = first[:, None] * bs + torch.arange(nt * bs, device=dev)
    blk = pos // bs
    page = table.long().gather(1, blk.clamp(max=nb - 1))
    real = (pos < lens[:, None]) & (blk < nb) & (page >= 0) & (page < P) & (lens > start)[:, None]
    page = page.clamp(0, P - 1)
    old = pos < start[:, None]
    b = torch.arange(B, device=dev)[:, None]
    src_new = (pos - start[:, None]).clamp(0, n - 1)
    src_old = pos % bs
    values = []
    bi, ji = real.nonzero(as_tuple=True)
    pg, off = page[bi, ji], src_old[bi, ji]
    done = real.view(B, nt, bs)[:, :, -1]  # complete blocks
    cb, cj = done.nonzero(as_tuple=True)
    cpage = page.view(B, nt, bs)[cb, cj, 0]
    touched = real.view(B, nt, bs)[:, :, 0]
    tb, tj = touched.nonzero(as_tuple=True)
    tpage = page.view(B, nt, bs)[tb, tj, 0]
    isopen = real & ~old & (blk == (lens // bs)[:, None])
    ob, oj = isopen.nonzero(as_tuple=True)
    isnew = (real & ~old).nonzero(as_tuple=True)
    for i, (x, codes) in enumerate(((s["k"], s["k_codes"]), (s["v"], s["v_codes"]))):
        xn = x.permute(0, 2, 1, 3)[b, src_new]               # (B, nt*bs, n_kv, d)
        xo = s["tail"][:, :, i].permute(0, 2, 1, 3)[b, src_old]
        full = torch.where(real[..., None, None], torch.where(old[..., None, None], xo, xn), 0).float()
        amax = full.abs().view(B, nt, bs, n_kv, d).amax((2, 4))  # (B, nt, n_kv)
        amax = torch.where(amax < TINY, 0.0, amax)
        each = amax.repeat_interleave(bs, 1)[..., None]
        c = _quantize(full, each)
        codes[pg, :, off] = c[bi, ji]
        s["amax"][tpage, :, i] = amax[tb, tj]
        if i == 0:
            cc = c.view(B, nt, bs, n_kv, d)[cb, cj]
            s["bounds"][cpage, :, 0] = cc.amin(1)
            s["bounds"][cpage, :, 1] = cc.amax(1)
        s["tail"][ob, :, i, src_old[ob, oj]] = xn[ob, oj]
        out = torch.zeros(B, n, n_kv, d, dtype=x.dtype, device=dev)
        out[isnew[0], src_new[isnew]] = (c.float() * (each / 127))[isnew].to(x.dtype)
        values.append(out.permute(0, 2, 1, 3))
    return values[0], values[1], s["amax"], s["k_codes"], s["v_codes"], s["bounds"], s["tail"]


def _select(s, sink=1, local=1):
    q, bs, top = s["q"], s["bs"], s["top"]
    B, H, n, d = q.shape
    table, P = s["table"].long(), s["bounds"].shape[0]
    n_kv, nb = s["bounds"].shape[1], table.shape[1]
    x = q.view(B, n_kv, H // n_kv, n, d).permute(0, 3, 1, 2, 4).float()  # (B, n, n_kv, rep, d)
    a = x.abs().amax((3, 4), keepdim=True)
    q8 = _quantize(x, a).float()
    page = table.clamp(0, P - 1)
    lo, hi = (s["bounds"][:, :, i][page].float().permute(0, 2, 3, 1)[:, None] for i in (0, 1))  # (B, 1, n_kv, d, nb)
    dot = (q8.clamp(min=0) @ hi + q8.clamp(max=0) @ lo).amax(3)          # (B, n, n_kv, nb): whole numbers, exact
    score = dot.double() * s["amax"][:, :, 0][page].permute(0, 2, 1)[:, None].double()
    pos = s["start"].long()[:, None] + torch.arange(n, device=q.device)
    here = torch.where(pos < s["lens"][:, None], pos // bs + 1, 0)[..., None, None]
    col = torch.arange(nb, device=q.device)
    score = torch.where((col < sink) | (col >= here - local), math.inf, score)
    score = torch.where(col < here, score, -math.inf)
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    taken = torch.zeros_like(score, dtype=torch.bool).scatter_(-1, order, True) & (col < here)
    return _ascending(taken, top)


def _softmax_rows(score, v):
    """Weighted rows of v and the log of the weights' sum; a row without a finite score is 0 and -inf."""
    m = score.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(score - m)
    total = e.sum(-1, keepdim=True)
    return (e @ v) / torch.where(total > 0, total, 1.0), (m + torch.log(total))[..., 0]


def _attend(s):
    q, bs, table = s["q"], s["bs"], s["table"].long()
    B, H, n, d = q.shape
    P, n_kv = s["amax"].shape[:2]
    rep, dev = H // n_kv, q.device
    pos = s["start"].long()[:, None] + torch.arange(n, device=dev)
    limit = torch.where(pos < s["lens"][:, None], pos + 1, 0)            # (B, n) keys that a token sees
    x = q.view(B, n_kv, rep, n, d).float() * s["scale"]
    if s["blocks"] is None:
        page = table.clamp(0, P - 1)
        k, v = (c[page].float() * (s["amax"][:, :, i][page] / 127)[..., None, None] for i, c in enumerate((s["k_codes"], s["v_codes"])))
        k, v = (t.permute(0, 2, 1, 3, 4).reshape(B, n_kv, -1, d) for t in (k, v))
        score = x.reshape(B, n_kv, rep * n, d) @ k.transpose(-1, -2)
        score = score.view(B, n_kv, rep, n, -1)
        key = torch.arange(k.shape[2], device=dev)
        score = torch.where(key < limit[:, None, None, :, None], score, -math.inf)
        out, lse = _softmax_rows(score.view(B, n_kv, rep * n, -1), v)
        out = out.view(B, H, n, d)
    else:
        blocks = s["blocks"].long()                                      # (B, n, n_kv, T)
        page = table[:, None, None].expand(-1, n, n_kv, -1).gather(-1, blocks.clamp(0, table.shape[1] - 1)).clamp(0, P - 1)
        kv = torch.arange(n_kv, device=dev)[:, None]
        k, v = (c[page, kv].float() * (s["amax"][page, kv][..., i] / 127)[..., None, None] for i, c in enumerate((s["k_codes"], s["v_codes"])))
        k, v = (t.flatten(3, 4) for t in (k, v))                         # (B, n, n_kv, T*bs, d)
        score = x.permute(0, 3, 1, 2, 4) @ k.transpose(-1, -2)           # (B, n, n_kv, rep, T*bs)
        key = (blocks[..., None] * bs + torch.arange(bs, device=dev)).flatten(3)
        seen = (key >= 0) & (key < limit[:, :, None, None])
        out, lse = _softmax_rows(torch.where(seen[..., None, :], score, -math.inf), v)
        out = out.permute(0, 2, 3, 1, 4).reshape(B, H, n, d)
        lse = lse.permute(0, 2, 3, 1)
    return out.to(q.dtype), lse.reshape(B, H, n)


def run(s):
    op = s["op"]
    if not own:
        return {"reserve": _reserve, "append": _append, "select": _select, "attend": _attend}[op](s)
    from ssa_b200 import ops
    if op == "reserve":
        start, lens, state = ops.cache_reserve(s["lens"], s["new"], s["table"], s["free"], s["state"], s["bs"])
        return start, lens, state, s["table"]
    if op == "append":
        k, v = ops.cache_append(s["k"], s["v"], s["k_codes"], s["v_codes"], s["amax"], s["bounds"], s["tail"], s["table"], s["start"],
                                s["lens"], want_values=True)
        return k, v, s["amax"], s["k_codes"], s["v_codes"], s["bounds"], s["tail"]
    if op == "select":
        return ops.cache_select(s["q"], s["bounds"], s["amax"], s["table"], s["start"], s["lens"], s["top"], s["bs"])
    return ops.cache_attention(s["q"], s["k_codes"], s["v_codes"], s["amax"], s["table"], s["start"], s["lens"], s["scale"],
                               blocks=s["blocks"], want_lse=True)


# ---------------------------------------------------------------- work and 64-bit values
def work(case):
    B, n, bs, op = case["B"], case["n"], case["bs"], case["op"]
    if op == "reserve":  # lengths in and out, a table entry and a free page's number for each page
        return {"bytes": 20 * B + 8 * B * max(1, n // 2) / bs, "flops": 0}
    n_kv, d, size = case["n_kv"], case["d"], DTYPES[case["dtype"]].itemsize
    # Ragged lengths average three quarters of the longest.
    tokens = B * n if n == 1 or B == 1 else n * (0.75 * (B - 2) + 1 + 1 / 3)
    if op == "append":  # tokens in, their codes and values out, a page's amax and bounds
        elements = 2 * tokens * n_kv * d
        return {"bytes": elements * (2 * size + 1) + tokens / bs * n_kv * (8 + 2 * d), "flops": 4 * elements}
    H, past = case["H"], case["past"] if B == 1 else case["past"] * (0.75 * (B - 1) + 1) / B
    rows = tokens * H * d * size
    if op == "select":
        pages = (past + bs - 1) // bs
        return {"bytes": B * pages * n_kv * (2 * d + 4) + rows + tokens * n_kv * case["top"] * 4, "flops": tokens * pages * H * 4 * d}
    keys = min(case["top"] * bs, past + 1) if case["top"] else past + n / 2
    # Without a list every key of a sequence is read once, with one each token's own blocks are.
    read = tokens * keys if case["top"] else B * (past + n)
    return {"bytes": read * n_kv * (2 * d + 8 / bs) + 2 * rows + tokens * H * 4, "flops": 4 * tokens * keys * H * d}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("reserve", "select"):
        return None  # whole numbers only
    bs, table = s["bs"], s["table"].long()
    start, lens = s["start"].tolist(), s["lens"].tolist()
    if s["op"] == "append":
        B, n_kv, n, d = s["k"].shape
        vals = [torch.zeros(B, n_kv, n, d, dtype=torch.float64, device="cuda") for _ in range(2)]
        amax = s["amax"].double()
        for b in range(B):
            lo = start[b] // bs * bs
            for i, x in enumerate((s["k"], s["v"])):
                if lens[b] == start[b]:
                    continue
                seq = torch.cat([s["tail"][b, :, i, : start[b] - lo], x[b, :, : lens[b] - start[b]]], 1).double()
                pad = -seq.shape[1] % bs
                blocks = torch.nn.functional.pad(seq, (0, 0, 0, pad)).view(n_kv, -1, bs, d)
                top = blocks.abs().flatten(2).amax(-1)
                step = top[..., None, None] / 127
                held = torch.round(blocks / top[..., None, None].clamp(min=1e-300) * 127) * step
                vals[i][b, :, : lens[b] - start[b]] = held.view(n_kv, -1, d)[:, start[b] - lo: lens[b] - lo]
                amax[table[b, lo // bs: lo // bs + top.shape[1]], :, i] = top.T
        return vals[0], vals[1], amax, None, None, None, None
    q = s["q"].double()
    B, H, n, d = q.shape
    n_kv = s["amax"].shape[1]
    rep = H // n_kv
    out = torch.zeros(B, H, n, d, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, n), -math.inf, dtype=torch.float64, device="cuda")
    for b in range(B):
        if s["blocks"] is None:
            if lens[b] == start[b]:
                continue
            pages = table[b, : (lens[b] + bs - 1) // bs]
            k, v = ((c[pages].double() * (s["amax"][pages][..., i].double() / 127)[..., None, None]).transpose(0, 1).reshape(n_kv, -1, d)
                    for i, c in enumerate((s["k_codes"], s["v_codes"])))
            fresh = lens[b] - start[b]
            at = q[b, :, :fresh].reshape(n_kv, rep, fresh, d) * s["scale"]
            score = torch.einsum("grtd,gkd->grtk", at, k[:, : lens[b]])
            later = torch.arange(lens[b], device="cuda")[None] > start[b] + torch.arange(fresh, device="cuda")[:, None]
            score.masked_fill_(later, -math.inf)
            out[b, :, :fresh] = torch.einsum("grtk,gkd->grtd", score.softmax(-1), v[:, : lens[b]]).reshape(H, fresh, d)
            lse[b, :, :fresh] = score.logsumexp(-1).reshape(H, fresh)
            continue
        for t in range(lens[b] - start[b]):
            for h in range(n_kv):
                blocks = s["blocks"][b, t, h].long()
                blocks = blocks[blocks >= 0]
                pages = table[b, blocks]
                k, v = ((c[pages, h].double() * (s["amax"][pages, h, i].double() / 127)[:, None, None]).reshape(-1, d)
                        for i, c in enumerate((s["k_codes"], s["v_codes"])))
                seen = (blocks[:, None] * bs + torch.arange(bs, device="cuda")).reshape(-1) <= start[b] + t
                score = q[b, h * rep: (h + 1) * rep, t] @ k[seen].T * s["scale"]
                out[b, h * rep: (h + 1) * rep, t] = score.softmax(-1) @ v[seen]
                lse[b, h * rep: (h + 1) * rep, t] = score.logsumexp(-1)
    return out, lse
