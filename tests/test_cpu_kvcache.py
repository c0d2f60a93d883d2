"""Refusals of the cache operators and of qknorm_rope, on the host: nothing touches a device."""
import ctypes as C

import pytest
import torch

from deepx_b200 import _native as N


def cache(**kw):
    f = dict(k=4096, v=8192 << 20, k_scale=64, v_scale=128, pages=4, kv_heads=2, page_tokens=16, head_dim=64, format=N.CACHE_I8)
    f.update(kw)
    return N.KvCache(*f.values())


def seqs(**kw):
    f = dict(starts=64, lens=128, table=256, batch=2, table_cols=3, rows=5)
    f.update(kw)
    return N.KvSeqs(*f.values())


FAR = 1 << 45  # addresses that overlap nothing and are never followed: every call below is refused or has nothing to do


def write(dtype=N.F32, k=FAR, ks=128, v=FAR * 2, vs=128, s=None, c=None):
    return N.lib.dx_kvcache_write(dtype, k, ks, v, vs, s or seqs(), c or cache(), None, None)


def read(dtype=N.F32, k=FAR, ks=128, v=FAR * 2, vs=128, s=None, c=None):
    return N.lib.dx_kvcache_read(dtype, s or seqs(), c or cache(), k, ks, v, vs, None, None)


def attend(dtype=N.BF16, q=FAR, qs=256, heads=4, s=None, c=None, scale=0.125, max_new=0, window=0, out=FAR * 2, os=256, ws=None, ws_bytes=0):
    return N.lib.dx_kvcache_attention(dtype, q, qs, heads, s or seqs(), c or cache(), scale, max_new, window, out, os, ws, ws_bytes, None, None)


CACHES = [(dict(format=2), N.E_DTYPE), (dict(format=-1), N.E_DTYPE), (dict(page_tokens=8), N.E_SHAPE), (dict(page_tokens=48), N.E_SHAPE),
          (dict(page_tokens=512), N.E_SHAPE), (dict(head_dim=0), N.E_SHAPE), (dict(head_dim=24), N.E_SHAPE), (dict(head_dim=272), N.E_SHAPE),
          (dict(kv_heads=0), N.E_SHAPE), (dict(pages=-1), N.E_SHAPE), (dict(k=None), N.E_ARG), (dict(v_scale=None), N.E_ARG), (dict(k=4100), N.E_ARG)]
SEQS = [(dict(batch=-1), N.E_SHAPE), (dict(rows=-1), N.E_SHAPE), (dict(rows=1 << 31), N.E_SHAPE), (dict(table_cols=1 << 30), N.E_SHAPE),
        (dict(starts=None), N.E_ARG), (dict(lens=None), N.E_ARG), (dict(table=None), N.E_ARG)]


@pytest.mark.parametrize("call", [write, read, attend])
def test_descriptors_are_checked(call):
    for kw, code in CACHES:
        if kw == dict(head_dim=272) or kw.get("kv_heads") == 0:
            continue
        assert call(c=cache(**kw)) == code, kw
    assert call(c=cache(head_dim=272), **({"qs": 4096, "os": 4096} if call is attend else {"ks": 4096, "vs": 4096})) == N.E_SHAPE
    assert call(c=cache(kv_heads=0)) == N.E_SHAPE
    for kw, code in SEQS:
        assert call(s=seqs(**kw)) == code, kw
    assert call(s=seqs(rows=0)) == N.OK and call(s=seqs(batch=0)) == N.OK  # nothing to do


@pytest.mark.parametrize("call", [write, read])
def test_rows_are_checked(call):
    assert call(dtype=N.F64) == N.E_DTYPE and call(dtype=N.I32) == N.E_DTYPE
    assert call(ks=127) == N.E_SHAPE and call(vs=0) == N.E_SHAPE
    assert call(k=None) == N.E_ARG and call(v=None) == N.E_ARG
    assert call(k=4096 + 16) == N.E_ALIAS and call(v=(8192 << 20) - 64) == N.E_ALIAS


def test_attention_arguments_are_checked():
    assert attend(dtype=N.F32) == N.E_DTYPE and attend(dtype=N.I8) == N.E_DTYPE
    assert attend(heads=3) == N.E_SHAPE and attend(heads=0) == N.E_SHAPE
    assert attend(qs=255) == N.E_SHAPE and attend(os=128) == N.E_SHAPE
    for bad in (0.0, -1.0, float("nan"), float("inf"), 1e-60):
        assert attend(scale=bad) == N.E_ARG, bad
    assert attend(max_new=-1) == N.E_ARG and attend(window=-1) == N.E_ARG
    assert attend(q=None) == N.E_ARG and attend(out=None) == N.E_ARG
    assert attend(out=FAR + 64) == N.E_ALIAS and attend(out=4096) == N.E_ALIAS
    assert attend(s=seqs(rows=(1 << 31) - 1)) == N.E_SHAPE  # rows of a key head's group beyond 32 bits


def test_attention_workspace_is_checked():
    need = N.lib.dx_kvcache_attention_workspace_bytes(N.BF16, 4, seqs(), cache(), 0)
    assert need > 0
    assert N.lib.dx_kvcache_attention_workspace_bytes(N.BF16, 4, seqs(rows=0), cache(), 0) == 0
    assert N.lib.dx_kvcache_attention_workspace_bytes(N.BF16, 4, seqs(), cache(format=7), 0) == 0
    assert attend() == N.E_WORKSPACE and attend(ws=FAR * 4, ws_bytes=need - 1) == N.E_WORKSPACE
    assert attend(ws=FAR * 4 + 64, ws_bytes=need) == N.E_ARG


def rope(dtype=N.F32, q=FAR, qs=256, qh=4, k=FAR * 2, ks=128, kh=2, tokens=3, dim=64, norm=1, eps=1e-6, inv=64, rotated=64, pos_dtype=N.I32, pos=64, qo=FAR * 3,
         qos=256, ko=FAR * 4, kos=128):
    return N.lib.dx_qknorm_rope(dtype, q, qs, qh, k, ks, kh, tokens, dim, norm, None, None, eps, inv, rotated, 0, pos_dtype, pos, qo, qos, ko, kos, None)


def test_rope_arguments_are_checked():
    assert rope(dtype=N.F64) == N.E_DTYPE and rope(dtype=N.I8) == N.E_DTYPE and rope(pos_dtype=N.F32) == N.E_DTYPE
    assert rope(dim=0) == N.E_SHAPE and rope(dim=513, qs=4096, ks=4096) == N.E_SHAPE
    assert rope(rotated=66) == N.E_SHAPE and rope(rotated=3) == N.E_SHAPE and rope(rotated=-2) == N.E_SHAPE
    assert rope(tokens=-1) == N.E_SHAPE and rope(qh=-1) == N.E_SHAPE
    assert rope(qs=255) == N.E_SHAPE and rope(kos=127) == N.E_SHAPE
    assert rope(eps=-1.0) == N.E_ARG and rope(eps=float("nan")) == N.E_ARG
    assert rope(q=None) == N.E_ARG and rope(ko=None) == N.E_ARG and rope(inv=None) == N.E_ARG and rope(pos=None) == N.E_ARG
    assert rope(tokens=0) == N.OK and rope(qh=0, kh=0) == N.OK
    assert rope(qo=FAR + 4) == N.E_ALIAS            # shifted over its own input
    assert rope(qo=FAR, qos=512) == N.E_ALIAS       # the same start, another stride
    assert rope(ko=FAR) == N.E_ALIAS                # keys over the queries
    # columns of one packed row: keys' output where the queries' input is
    assert rope(qs=512, k=FAR + 256 * 4, ks=512, qo=FAR, qos=512, ko=FAR + 255 * 4, kos=512) == N.E_ALIAS


def test_tensorfunc_checks():
    from deepx_b200 import tensorfunc as TF
    K = torch.zeros(5, 2, 64)
    with pytest.raises(ValueError, match="no CPU path"):
        TF.kvcache_write(K, K, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32),
                         torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.ones(4, 2), torch.ones(4, 2))
    with pytest.raises(ValueError, match="no CPU path"):
        TF.qknorm_rope(K, K, None, None, torch.zeros(32), torch.zeros(5, dtype=torch.int32), None, False, K, K)
    assert C.sizeof(N.KvCache) == 72 and C.sizeof(N.KvSeqs) == 48  # the header's structures
