"""Prompts in a cache that has no room for all of them, of unequal lengths,
and beside sequences that are already decoding."""
import pytest
import torch

from ssa_b200 import SSAConfig, SparseTransformer
from test_gpu_serving import CFG, _model

pytestmark = pytest.mark.gpu


def _ids(g, B, N, dev):
    return torch.randint(0, 50, (B, N), generator=g).to(dev)


def _forward(m, ids):
    with torch.no_grad():
        return m(ids)[0]


def _without_attention(m, ids):
    """The model's rows where attention gives zeros."""
    with torch.no_grad():
        x = m.embed(ids)
        for layer in m.layers:
            a = layer.attn.Wo(torch.zeros_like(x))
            x = x + a + layer.ff(layer.norm2(x + a))
        return m.norm(x)


def _state(cache):
    return [t.clone() for t in (cache.k_codes, cache.v_codes, cache.amax, cache.bounds, cache.tail, cache.table, cache.lens)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_refused_prompts_have_zero_attention(dt, cuda):
    m, g = _model(dt, cuda), torch.Generator().manual_seed(1)
    ids = _ids(g, 3, 40, cuda)
    cache = m.new_cache(3, 64, block_size=16, num_blocks=7)  # 40 tokens are three blocks: the third sequence gets none
    out = m.prefill(ids, cache)
    assert cache.lens.tolist() == [40, 40, 0] and cache.refused() == 1
    assert torch.equal(out[:2], _forward(m, ids)[:2])
    assert torch.equal(out[2], _without_attention(m, ids)[2])
    narrow = m.new_cache(3, 32, block_size=16)  # a table too narrow for any of them
    assert torch.equal(m.prefill(ids, narrow), _without_attention(m, ids))
    assert narrow.lens.tolist() == [0, 0, 0] and narrow.refused() == 3


def test_prompts_of_unequal_lengths(cuda):
    m, g = _model(torch.bfloat16, cuda), torch.Generator().manual_seed(2)
    ids, lens = _ids(g, 4, 70, cuda), [70, 1, 0, 33]
    cache = m.new_cache(4, 128, block_size=16)
    out = m.prefill(ids, cache, torch.tensor(lens, dtype=torch.int32, device=cuda))
    want, none = _forward(m, ids), _without_attention(m, ids)
    assert cache.lens.tolist() == lens and cache.refused() == 0
    for b, n in enumerate(lens):
        assert torch.equal(out[b, n:], none[b, n:]), b
        if n >= 2:  # the two global tokens are real: the rows' neighbors are those of the padded batch
            assert torch.equal(out[b, :n], want[b, :n]), b
    whole = m.new_cache(4, 128, block_size=16)
    m.prefill(ids, whole)
    k, v = (t.cpu() for t in cache.values())
    kw, vw = (t.cpu() for t in whole.values())
    for b, n in enumerate(lens):  # complete blocks of tokens equal those of the whole rows'; nothing behind
        full = n // 16 * 16
        assert torch.equal(k[b, :, :full], kw[b, :, :full]) and torch.equal(v[b, :, :full], vw[b, :, :full])
        assert not k[b, :, n:].any() and not v[b, :, n:].any()
    nxt = m.step(_ids(g, 4, 1, cuda), cache)
    assert torch.isfinite(nxt.float()).all() and cache.lens.tolist() == [n + 1 for n in lens]


@pytest.mark.parametrize("indices", [None, [0, 40, 3]])
def test_padding_is_never_attended(indices, cuda):
    """Global tokens may lie in a row's padding: what stands there changes nothing."""
    torch.manual_seed(0)
    cfg = SSAConfig(d_model=256, num_heads=4, num_kv_heads=2, **{**CFG, "global_token_indices": indices})
    m, g = SparseTransformer(cfg, 3, 50).to(cuda, torch.bfloat16).eval(), torch.Generator().manual_seed(6)
    ids, lens = _ids(g, 5, 60, cuda), [60, 1, 2, 39, 41]
    new = torch.tensor(lens, dtype=torch.int32, device=cuda)
    got = []
    for _ in range(2):
        cache = m.new_cache(5, 64, block_size=16)
        got.append([m.prefill(ids, cache, new), *cache.values(0), *cache.values(2)])
        for b, n in enumerate(lens):
            ids[b, n:] = (ids[b, n:] + 7) % 50
    for b, n in enumerate(lens):
        assert torch.equal(got[0][0][b, :n], got[1][0][b, :n]), b
    for a, b in zip(got[0][1:], got[1][1:]):
        assert torch.equal(a, b)


def test_prompt_beside_decoding_sequences(cuda):
    m, g = _model(torch.bfloat16, cuda), torch.Generator().manual_seed(3)
    cache = m.new_cache(3, 128, block_size=16)
    m.prefill(_ids(g, 3, 50, cuda), cache)
    for _ in range(3):
        m.step(_ids(g, 3, 1, cuda), cache)
    cache.release(torch.tensor([False, True, False]))
    before = _state(cache)
    ids = _ids(g, 3, 44, cuda)
    out = m.prefill(ids, cache, torch.tensor([0, 44, 0], dtype=torch.int32, device=cuda))
    assert cache.lens.tolist() == [53, 44, 53] and cache.refused() == 0
    assert torch.equal(out[1], _forward(m, ids)[1])
    live = cache.table[[0, 2], :4].flatten().long()
    for was, now in zip(before[:4], _state(cache)[:4]):
        assert torch.equal(was[:, live], now[:, live])
    assert torch.equal(before[4][:, [0, 2]], cache.tail[:, [0, 2]]) and torch.equal(before[5][[0, 2]], cache.table[[0, 2]])
    alone = m.new_cache(3, 128, block_size=16)
    m.prefill(ids, alone)
    for a, b in zip(cache.values(1), alone.values(1)):
        assert torch.equal(a[1], b[1])


def test_prompts_do_not_go_behind_tokens(cuda):
    """A sequence that has tokens takes no prompt: it stays as it is and is counted."""
    m, g = _model(torch.bfloat16, cuda), torch.Generator().manual_seed(4)
    cache = m.new_cache(3, 128, block_size=16)
    m.prefill(_ids(g, 3, 20, cuda), cache, torch.tensor([20, 0, 5], dtype=torch.int32, device=cuda))
    before = _state(cache)
    ids = _ids(g, 3, 30, cuda)
    out = m.prefill(ids, cache)
    assert cache.lens.tolist() == [20, 30, 5] and cache.refused() == 2
    assert torch.equal(out[1], _forward(m, ids)[1])
    for b in (0, 2):
        assert torch.equal(out[b], _without_attention(m, ids)[b])
        pages = cache.table[b, :2][:2 if b == 0 else 1].long()
        for was, now in zip(before[:4], _state(cache)[:4]):
            assert torch.equal(was[:, pages], now[:, pages])
        assert torch.equal(before[4][:, b], cache.tail[:, b])
    m.prefill(ids, cache, torch.zeros(3, dtype=torch.int32, device=cuda))
    assert cache.lens.tolist() == [20, 30, 5] and cache.refused() == 2


def test_prefill_refusals(cuda):
    m, g = _model(torch.bfloat16, cuda), torch.Generator().manual_seed(5)
    cache = m.new_cache(2, 64, block_size=16)
    ids = _ids(g, 2, 8, cuda)
    for bad in (torch.ones(3, dtype=torch.int32, device=cuda), torch.ones(2, device=cuda), torch.ones(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="new_lens"):
            m.prefill(ids, cache, bad)
    for layer in m.layers:
        layer.attn.config.causal = False
    with pytest.raises(ValueError, match="causal"):
        m.prefill(ids, cache, torch.ones(2, dtype=torch.int32, device=cuda))
    assert cache.lens.tolist() == [0, 0] and cache.refused() == 0
