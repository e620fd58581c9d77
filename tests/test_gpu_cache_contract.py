"""What a step promises beside its values: fp32 weights where the config asks
for them, refusals that leave the cache as it was, and no silent tangents."""
import pytest
import torch
from torch.autograd import forward_ad

import cache_ref as R
from ssa_b200 import BlockCache, SSAConfig, SparseAttention, SparseTransformer, ops
from test_gpu_serving import CFG, _model

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("top", [None, 3])
def test_step_with_fp32_weights(top, cuda):
    """config.fp32_attn_weights: two tokens of nearly the same weight whose values
    nearly cancel. Weights of 11 bits leave up to 2^-12 of the values each; the
    output has to be right to 2^-19 of them and its own rounding."""
    torch.manual_seed(0)
    cfg = SSAConfig(d_model=128, num_heads=1, **{**CFG, "fp32_attn_weights": True})
    attn = SparseAttention(cfg).to(cuda, torch.bfloat16)
    eye = torch.eye(128, dtype=torch.bfloat16, device=cuda)
    with torch.no_grad():
        for w in (attn.Wq, attn.Wk, attn.Wv, attn.Wo):
            w.weight.copy_(eye)
        attn.Wk.weight[64:] = 0  # scores are of the first half
    g = torch.Generator().manual_seed(2)
    for _ in range(8):
        x = torch.zeros(1, 3, 128)
        x[0, :, :64] = 0.1 * torch.randn(3, 64, generator=g)
        far = 8 * torch.randn(64, generator=g)
        x[0, 0, 64:], x[0, 1, 64:] = far, -far
        cache = BlockCache(1, 1, 128, 64, block_size=16, top_blocks=top, dtype=torch.bfloat16)
        cache.reserve(3)
        out = attn.step(x.to(cuda, torch.bfloat16), cache)[0, 2].double().cpu()
        k, v = (t[0, 0, :3].double().cpu() for t in cache.values())
        q = x[0, 2].to(torch.bfloat16).double()
        ref, _, vmax, reach = R.attend(q[None], k, v, torch.ones(1, 3, dtype=torch.bool), attn.scale)
        ref, vmax, reach = ref[0], float(vmax[0]), float(reach[0])
        # weights to 2^-21 with the exponential's 2^-21 and the scores' error; bf16 output, and Wo's rounding of it
        tol = 2 * 2.0 ** -8 * ref.abs() + (2 * 136 * 2.0 ** -23 * reach + 2.0 ** -19) * vmax
        err = (out - ref).abs()
        assert (err <= tol).all(), float((err / tol).max())
        assert ref.abs().max() > 0


def _snapshot(cache):
    return [t.clone() for t in (cache.lens, cache.start, cache.state, cache.table, cache.k_codes, cache.v_codes, cache.amax,
                                cache.bounds, cache.tail)]


def test_a_refused_step_leaves_the_cache(cuda):
    """What step and prefill can refuse they refuse before a page is taken."""
    m = _model(torch.bfloat16, cuda)
    ids = torch.randint(0, 50, (2, 5), device=cuda)
    mk = lambda **kw: BlockCache(**{**dict(batch=2, num_kv_heads=2, head_dim=64, max_tokens=64, num_layers=2, block_size=16), **kw})  # noqa: E731
    wide = {**CFG, "global_token_indices": [0, 100]}  # seven leading blocks of 16 are always attended
    far = SparseTransformer(SSAConfig(d_model=256, num_heads=4, num_kv_heads=2, **wide), 2, 50).to(cuda, torch.bfloat16).eval()
    full = SparseTransformer(SSAConfig(d_model=256, num_heads=4, num_kv_heads=2, **{**CFG, "causal": False}), 2, 50).to(
        cuda, torch.bfloat16).eval()
    for model, cache, what in ((m, mk(batch=3), "batch"), (m, mk(num_kv_heads=1), "num_kv_heads"), (m, mk(head_dim=32), "head_dim"),
                               (m, mk(num_layers=1), "num_layers"), (far, mk(top_blocks=8), "top_blocks"), (full, mk(), "causal")):
        before = _snapshot(cache)
        calls = [lambda: model.step(ids, cache)]
        if what not in ("top_blocks", "causal"):
            calls.append(lambda: model.prefill(ids, cache))
        for call in calls:
            with pytest.raises(ValueError, match=what):
                call()
        for a, b in zip(before, _snapshot(cache)):
            assert torch.equal(a, b), what
    far.step(ids, mk(top_blocks=9))


def test_a_cache_of_another_type_is_refused(cuda):
    """The type is the projections': under autocast its, else the weights'."""
    m = _model(torch.float32, cuda)
    ids = torch.randint(0, 50, (2, 5), device=cuda)
    for dt, auto in ((torch.bfloat16, False), (torch.float32, True)):
        cache = BlockCache(2, 2, 64, 64, num_layers=2, block_size=16, dtype=dt)
        with torch.autocast("cuda", torch.bfloat16, enabled=auto), pytest.raises(ValueError, match="dtype"):
            m.step(ids, cache)
        assert cache.lens.tolist() == [0, 0] and int(cache.state[0]) == cache.num_blocks
    cache = BlockCache(2, 2, 64, 64, num_layers=2, block_size=16, dtype=torch.bfloat16)
    with torch.autocast("cuda", torch.bfloat16):
        m.prefill(ids, cache)
        out = m.step(ids[:, :1], cache)
    assert cache.lens.tolist() == [6, 6] and torch.isfinite(out).all()


def test_tangents_are_refused(cuda):
    """A dual tensor's tangent is not dropped without a word, under no_grad either."""
    cache = BlockCache(1, 2, 64, 64, block_size=16)
    x = torch.randn(1, 2, 3, 64, device=cuda, dtype=torch.bfloat16)
    cache.reserve(3)
    cache.append(x, x)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (torch.enable_grad, torch.no_grad):
            with grad():
                for call in (lambda: cache.append(dual, x), lambda: cache.append(x, dual), lambda: cache.attend(dual, 0.1)):
                    with pytest.raises(RuntimeError, match="no gradient"):
                        call()
        plain = forward_ad.unpack_dual(dual).primal
        assert torch.equal(cache.attend(plain, 0.1), cache.attend(x, 0.1))
        assert ops.cache_select(dual, cache.bounds[0], cache.amax[0], cache.table, cache.start, cache.lens, 2, 16).dtype == torch.int32
    assert torch.equal(cache.attend(dual, 0.1), cache.attend(x, 0.1))  # the level is over: no tangent
