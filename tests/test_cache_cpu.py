"""CPU-side checks of the block cache: the C ABI's refusals (none reaches a
launch), the operators' refusals, and the restatement the GPU tests use."""
import ctypes
import math

import pytest
import torch

import cache_ref as R
from ssa_b200 import _lib, ops

ONE = ctypes.c_void_p(1 << 20)  # aligned, never dereferenced: every call below is refused before a launch


def _params(**kw):
    p = _lib.CacheParams()
    base = dict(B=2, H=4, n_kv=2, n=1, d=64, dtype=1, block_size=16, max_blocks=4, num_pages=9, top=3, sink=1, local=1,
                causal=1, scale=0.125, q_sb=256, q_sh=64, q_sn=256, k_sb=128, k_sh=64, k_sn=128, v_sb=128, v_sh=64,
                v_sn=128, o_sb=256, o_sh=64, o_sn=256)
    for k, v in {**base, **kw}.items():
        setattr(p, k, v)
    return p


def _append(p, k=ONE, table=ONE, values=(None, None), tail=ONE):
    return _lib.load().ssa_cache_append(p, k, ONE, ONE, ONE, ONE, ONE, tail, table, ONE, ONE, *values, None)


def _select(p, q=ONE, out=ONE):
    return _lib.load().ssa_cache_select(p, q, ONE, ONE, ONE, ONE, ONE, out, None)


def _attn(p, ws=ONE, nbytes=0, blocks=None, out=ONE):
    return _lib.load().ssa_cache_attn(p, ONE, ONE, ONE, ONE, ONE, ONE, ONE, blocks, out, None, ws, nbytes, None)


@pytest.mark.parametrize("change,code", [
    (dict(B=0), 1), (dict(n=0), 1), (dict(n_kv=0), 1), (dict(max_blocks=0), 1), (dict(num_pages=0), 1), (dict(dtype=2), 1),
    (dict(d=48), 2), (dict(d=256), 2), (dict(block_size=8), 2), (dict(block_size=128), 2), (dict(block_size=17), 2),
    (dict(max_blocks=1 << 27), 2)])
def test_abi_refuses_geometry(change, code):
    p = _params(**change)
    assert _append(p) == code
    assert _select(p) == code
    assert _attn(p) == code
    assert _lib.load().ssa_last_error()


def test_abi_refuses_arguments():
    L = _lib.load()
    assert L.ssa_cache_append(None, *[ONE] * 10, None, None, None) == _lib.SSA_ERR_INVALID
    assert _append(_params(), k=None) == _lib.SSA_ERR_INVALID
    assert _append(_params(), k=ctypes.c_void_p((1 << 20) + 2)) == _lib.SSA_ERR_UNSUPPORTED
    assert _append(_params(), table=None) == _lib.SSA_ERR_INVALID
    assert _append(_params(), tail=None) == _lib.SSA_ERR_INVALID
    assert _append(_params(), values=(ONE, None)) == _lib.SSA_ERR_INVALID
    assert _append(_params(k_sn=63)) == _lib.SSA_ERR_UNSUPPORTED
    assert _append(_params(v_sh=-64)) == _lib.SSA_ERR_INVALID
    assert _select(_params(H=3)) == _lib.SSA_ERR_INVALID
    for bad in (dict(top=1), dict(local=0), dict(sink=-1), dict(sink=3), dict(top=0)):
        assert _select(_params(**bad)) == _lib.SSA_ERR_INVALID, bad
    assert _select(_params(), out=None) == _lib.SSA_ERR_INVALID
    assert _select(_params(max_blocks=1 << 20)) == _lib.SSA_ERR_UNSUPPORTED
    assert _attn(_params(H=5)) == _lib.SSA_ERR_INVALID
    assert _attn(_params(), out=None) == _lib.SSA_ERR_INVALID
    assert _attn(_params(top=0), blocks=ONE, nbytes=1 << 30) == _lib.SSA_ERR_INVALID
    need = L.ssa_cache_attn_workspace_size(_params(), 0)
    assert need > 0 and _attn(_params(), nbytes=need - 1) == _lib.SSA_ERR_WORKSPACE
    assert _attn(_params(), ws=None, nbytes=need) == _lib.SSA_ERR_WORKSPACE
    assert L.ssa_cache_attn_workspace_size(None, 0) == 0
    r = [2, 4, 16, 9] + [ctypes.c_void_p((1 << 20) + 64 * i) for i in range(8)] + [None]
    assert L.ssa_cache_reserve(*[0] + r[1:]) == _lib.SSA_ERR_INVALID
    assert L.ssa_cache_reserve(*r[:4], None, *r[5:]) == _lib.SSA_ERR_INVALID
    assert L.ssa_cache_reserve(*r[:9], r[4], *r[10:]) == _lib.SSA_ERR_INVALID  # start_out is lens
    assert L.ssa_cache_reserve(2, 1 << 27, 16, 9, *r[4:]) == _lib.SSA_ERR_UNSUPPORTED


def test_ops_refuse_cpu_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    t = torch.zeros(2, 4, dtype=torch.int32)
    x = torch.zeros(2, 2, 1, 64)
    c = torch.zeros(9, 2, 16, 64, dtype=torch.int8)
    am, bd, tail = torch.zeros(9, 2, 2), torch.zeros(9, 2, 2, 64, dtype=torch.int8), torch.zeros(2, 2, 2, 16, 64)
    for call in (lambda: ops.cache_reserve(i, i, t, i, i, 16), lambda: ops.cache_append(x, x, c, c, am, bd, tail, t, i, i),
                 lambda: ops.cache_select(x, bd, am, t, i, i, 2, 16), lambda: ops.cache_attention(x, c, c, am, t, i, i, 1.0)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_quantize_reference():
    codes, amax = R.quantize(torch.tensor([[127.0, 63.5, 62.5, -0.5, 0.25, -127.0]]))
    assert amax == 127 and codes.tolist() == [[127, 64, 62, 0, 0, -127]]
    assert R.quantize(torch.full((2, 2), 2.0 ** -81))[1] == 0
    assert math.isnan(R.quantize(torch.tensor([[1.0, math.nan]]))[1])


def test_reserve_reference():
    start, lens, state, table = R.reserve([0, 16, 5], [17, 1, 11], [[9] * 2, [9] * 2, [9] * 2], [1, 2, 3], [3, 0], 16)
    assert (start, lens, state) == ([0, 16, 5], [17, 17, 16], [0, 0])
    assert table == [[3, 2], [9, 1], [9, 9]]
    assert R.reserve([0, 0, 16], [17, 16, 0], [[9] * 2] * 3, [1, 2], [1, 0], 16)[1:3] == ([0, 0, 16], [1, 2])


def test_block_cache_refusals():
    from ssa_b200 import BlockCache
    for bad, err in ((dict(batch=0), ValueError), (dict(block_size=24), NotImplementedError), (dict(head_dim=48), NotImplementedError),
                     (dict(dtype=torch.float16), NotImplementedError), (dict(top_blocks=0), ValueError), (dict(device="cpu"), RuntimeError)):
        kw = {**dict(batch=1, num_kv_heads=1, head_dim=64, max_tokens=64), **bad}
        with pytest.raises(err):
            BlockCache(**kw)


def test_cached_blocks():
    import warnings
    from ssa_b200 import SSAConfig, SparseAttention
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        for kw, want in ((dict(num_global_tokens=2, window_size=8), (1, 2)), (dict(num_global_tokens=0, window_size=0), (0, 1)),
                         (dict(num_global_tokens=33, window_size=16), (3, 2)),
                         (dict(global_token_indices=[0, 40], window_size=17), (3, 3)),
                         (dict(global_token_indices=[], window_size=1), (0, 2))):
            attn = SparseAttention(SSAConfig(d_model=64, num_heads=2, num_neighbors=64, **kw))
            assert attn.cached_blocks(16) == want, kw
