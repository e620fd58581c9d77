"""Serving: BlockCache, SparseAttention.step / prefill and SparseTransformer's
cached steps, against the model computed in 64 bits over the values that the
cache holds, and as a captured CUDA graph."""
import math

import pytest
import torch

import cache_ref as R
from ssa_b200 import BlockCache, SSAConfig, SparseAttention, SparseTransformer

pytestmark = pytest.mark.gpu

CFG = dict(num_neighbors=64, num_hash_rounds=4, max_num_hashes=8, window_size=4, num_global_tokens=2, causal=True)


def _model(dt, dev, H=4, n_kv=2, d_model=256, layers=2, vocab=50):
    torch.manual_seed(0)
    return SparseTransformer(SSAConfig(d_model=d_model, num_heads=H, num_kv_heads=n_kv, **CFG), layers, vocab).to(dev, dt).eval()


def _attention_reference(attn, x, cache, layer, blocks=None):
    """SparseAttention.step in 64 bits: the projections as the model computes
    them (its own type), attention over the values the cache holds."""
    B, n, _ = x.shape
    q = attn._split_q(attn.Wq(x)).double().cpu()
    k, v = (t.double().cpu() for t in cache.values(layer))
    start, lens = cache.start.tolist(), cache.lens.tolist()
    out = torch.zeros(B, n, attn.H, attn.d_head, dtype=torch.float64)
    for b in range(B):
        for t in range(lens[b] - start[b]):
            for h in range(attn.H):
                seen = torch.arange(k.shape[2]) <= start[b] + t
                if blocks is not None:
                    on = torch.zeros(cache.max_blocks, dtype=torch.bool)
                    on[[e for e in blocks[b, t, h // attn.kv_rep].tolist() if e >= 0]] = True
                    seen = seen & on.repeat_interleave(cache.block_size)
                g = h // attn.kv_rep
                out[b, t, h] = R.attend(q[b, h, t:t + 1], k[b, g], v[b, g], seen[None], attn.scale)[0][0]
    return out.reshape(B, n, -1) @ attn.Wo.weight.double().cpu().T


@pytest.mark.parametrize("dt,top", [(torch.bfloat16, None), (torch.bfloat16, 3), (torch.float32, None), (torch.float32, 4)])
def test_attention_step_equals_reference(dt, top, cuda):
    attn = _model(dt, cuda).layers[0].attn
    cache = BlockCache(3, 2, 64, 200, block_size=16, top_blocks=top, dtype=dt)
    g = torch.Generator().manual_seed(1)
    for n, new in ((60, [60, 1, 33]), (1, [1, 1, 1]), (5, [5, 0, 2]), (1, [1, 1, 1])):
        x = torch.randn(3, n, 256, generator=g).to(cuda, dt)
        cache.reserve(torch.tensor(new, dtype=torch.int32, device=cuda))
        out = attn.step(x, cache)
        blocks = None
        if top is not None:
            sink, local = attn.cached_blocks(16)
            assert (sink, local) == (1, 2)
            q = attn._split_q(attn.Wq(x))
            blocks = cache.select(q, sink=sink, local=local).cpu()
        ref = _attention_reference(attn, x, cache, 0, blocks)
        # the attention's and the projection's roundings to the model's type (half a step each), the
        # weights' 2^-11, and the projection's own sum of 256 products: against the row's norm
        eps = torch.finfo(dt).eps / 2
        tol = 4 * eps + (2.0 ** -11 if dt == torch.bfloat16 else 256 * 2.0 ** -24)
        for b in range(3):
            d = (out[b, :new[b]].double().cpu() - ref[b, :new[b]]).norm()
            assert d <= tol * ref[b, :new[b]].norm() + 1e-12, (b, float(d))
    assert cache.lens.tolist() == [67, 3, 37] and cache.refused() == 0


def test_transformer_prefill_and_steps(cuda):
    """A prompt over the sparse graph equals `forward`; single tokens and four
    at once fill the same cache."""
    m = _model(torch.bfloat16, cuda, layers=3)
    ids = torch.randint(0, 50, (2, 90), device=cuda)
    cache = m.new_cache(2, 128, block_size=32)
    with torch.no_grad():
        ref, _ = m(ids)
    out = m.prefill(ids, cache)
    assert torch.equal(out, ref)  # the same kernels on the same values
    nxt = torch.randint(0, 50, (2, 4), device=cuda)
    for t in range(4):
        y = m.step(nxt[:, t:t + 1], cache)
    assert y.shape == (2, 1, 256) and torch.isfinite(y.float()).all() and cache.lens.tolist() == [94, 94]
    # the same four tokens in one step: the last row sees the same cache
    again = m.new_cache(2, 128, block_size=32)
    m.prefill(ids, again)
    z = m.step(nxt, again)
    assert z.shape == (2, 4, 256) and again.lens.tolist() == [94, 94]
    for a, b in zip(cache._layers[0], again._layers[0]):
        # layer 0's keys and values do not depend on attention: its cache is the same, bit for bit
        assert torch.equal(a, b)


def test_release_and_refusal(cuda):
    m = _model(torch.bfloat16, cuda, layers=1)
    cache = m.new_cache(3, 64, block_size=16, num_blocks=6)
    x = torch.randint(0, 50, (3, 32), device=cuda)
    m.step(x, cache)
    assert cache.lens.tolist() == [32, 32, 32] and cache.state.tolist() == [0, 0]
    y = m.step(x[:, :1], cache)  # no page left: nothing is stored, nothing breaks
    assert cache.lens.tolist() == [32, 32, 32] and cache.refused() == 3 and torch.isfinite(y.float()).all()
    cache.release(torch.tensor([False, True, False]))
    assert cache.lens.tolist() == [32, 0, 32] and cache.state.tolist() == [2, 3]
    want = m.new_cache(3, 64, block_size=16)
    m.step(x, want, torch.tensor([0, 20, 0], dtype=torch.int32, device=cuda))
    got = m.step(x, cache, torch.tensor([0, 20, 0], dtype=torch.int32, device=cuda))
    assert cache.lens.tolist() == [32, 20, 32]
    k, v = cache.values()
    kw, vw = want.values()
    assert torch.equal(k[1], kw[1]) and torch.equal(v[1], vw[1])
    assert torch.isfinite(got[1, :20].float()).all()
    pages = cache.table[cache.table >= 0].tolist()
    assert sorted(pages) == list(range(6))


def test_captured_model_step(cuda):
    """A whole model step, block selection included, as one CUDA graph."""
    m = _model(torch.bfloat16, cuda, layers=2)
    ids = torch.randint(0, 50, (2, 70), device=cuda)
    eager, cap = (m.new_cache(2, 256, block_size=16, top_blocks=4) for _ in range(2))
    m.prefill(ids, eager), m.prefill(ids, cap)
    tok = torch.randint(0, 50, (2, 1), device=cuda)
    one = torch.ones(2, dtype=torch.int32, device=cuda)
    kept = [t.clone() for t in (cap.lens, cap.start, cap.state, cap.table, cap.k_codes, cap.v_codes, cap.amax, cap.bounds, cap.tail)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        m.step(tok, cap, one)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        held = m.step(tok, cap, one)
    for t, k in zip((cap.lens, cap.start, cap.state, cap.table, cap.k_codes, cap.v_codes, cap.amax, cap.bounds, cap.tail), kept):
        t.copy_(k)
    for _ in range(40):
        want = m.step(tok, eager, one)
        graph.replay()
        assert torch.equal(held, want)
        tok.copy_((want.float().sum(-1) * 7).long().abs() % 50)
    assert cap.lens.tolist() == [110, 110] and torch.equal(cap.table, eager.table)


def test_step_refusals(cuda):
    m = _model(torch.bfloat16, cuda, layers=1)
    cache = m.new_cache(2, 64, block_size=16)
    q = torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16, device=cuda)
    with pytest.raises(ValueError, match="block budget"):
        cache.select(q)
    with pytest.raises(ValueError):
        cache.select(q, top=1, sink=1, local=1)
    with pytest.raises(ValueError, match="k_codes"):
        cache.append(torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16, device=cuda),
                     torch.zeros(2, 3, 1, 64, dtype=torch.bfloat16, device=cuda))
    with pytest.raises(ValueError, match="tail"):
        cache.append(torch.zeros(2, 2, 1, 64, device=cuda), torch.zeros(2, 2, 1, 64, device=cuda))
    with pytest.raises(ValueError, match="differ"):
        cache.append(torch.zeros(2, 2, 1, 64, device=cuda), torch.zeros(2, 2, 2, 64, device=cuda))
    with pytest.raises(ValueError, match="blocks"):
        cache.attend(q, 1.0, blocks=torch.zeros(2, 1, 2, 3, dtype=torch.int64, device=cuda))
    with pytest.raises(ValueError, match="divisible"):
        cache.attend(q[:, :3], 1.0)
    with pytest.raises(ValueError, match="table"):
        cache.attend(q[:1], 1.0)
    with pytest.raises(NotImplementedError, match="float32 or bfloat16"):
        cache.attend(q.half(), 1.0)
    with pytest.raises(RuntimeError, match="gradient"):
        cache.attend(q.requires_grad_(), 1.0)
    with pytest.raises(ValueError, match="new_lens"):
        cache.reserve(torch.ones(2, dtype=torch.int64, device=cuda))
    with pytest.raises(ValueError):
        cache.release(torch.ones(3, dtype=torch.bool))
    full = SparseAttention(SSAConfig(d_model=256, num_heads=4, num_kv_heads=2, **{**CFG, "causal": False})).to(cuda, torch.bfloat16)
    with pytest.raises(ValueError, match="causal"):
        full.step(torch.zeros(2, 1, 256, dtype=torch.bfloat16, device=cuda), cache)
    none = cache.attend(q[:, :, :0].detach(), 1.0)
    assert none.shape == (2, 4, 0, 64)
