"""Attention over the 8-bit cache where its numbers lie far apart: keys and queries near the ends of float32, values of very different
scales, pages behind a window.  Plain implementations in 64 bits and the bounds: kvcache_plain.py."""
import pytest
import torch

import kvcache_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def TF():
    from deepx_b200 import tensorfunc
    return tensorfunc


def attend(TF, b, Q, scale, window=0, max_new=0, table=None):
    from deepx_b200 import _native as N
    Out = torch.full_like(Q, 3.0)
    TF.kvcache_attention(Q, *b.cache(), b.starts, b.length, b.table if table is None else table, scale, max_new, window, Out, b.flag)
    N.check(N.lib.dx_kvcache_status(None))
    return Out


def check(TF, b, Q, scale, window=0, max_new=0):
    want, bound = P.attention_rows(b, Q, scale, window)
    got = attend(TF, b, Q, scale, window, max_new)
    assert int(b.flag) == 0
    last = b.host_starts[-1]
    got, want, bound = got[:last].double(), want[:last], bound[:last]
    bound = bound + P.half_step(Q.dtype) * (want.abs() + bound) + torch.finfo(Q.dtype).tiny
    off = (got - want).abs()
    assert torch.isfinite(got).all()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound).max()):.3f} of the bound"


def zero_keys(b, seq, column, scale):
    at = int(b.host_table[seq, column])
    b.k.view(torch.uint8)[at] = 0
    b.ks[at] = scale


# ---- keys of zero and far from one ---------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("size", [1e-15, 1e-18, 1e-30, 1e-38])
@pytest.mark.parametrize("empty", [2.0**-126, 0.0])
def test_small_queries_over_keys_of_zero(TF, dim, window, size, empty):
    """Pages of zero keys (the smallest scale; never written: scale zero) on the diagonal and in front of it, and rows of tiny queries:
    their scores are zero, not no number, whichever kernel is taken."""
    lens, new = [200, 150], [130, 130]
    b = P.Batch(31, lens, new, 1, dim, 16, "int8").fill(lens, (-8, -4))
    for column in (1, 6, 9):  # tokens 16-31, 96-111, 144-159
        zero_keys(b, 0, column, empty)
        zero_keys(b, 1, min(column, 8), empty)
    Q = b.rand(b.rows, 2, dim, dtype=torch.bfloat16) * size
    for hint in (130, 0):
        check(TF, b, Q, dim ** -0.5, window, hint)
    new1 = P.Batch(32, [200], [1], 1, dim, 16, "int8").fill([200], (-8, -4))
    zero_keys(new1, 0, 12, empty)
    check(TF, new1, new1.rand(1, 2, dim, dtype=torch.bfloat16) * size, dim ** -0.5, window, 1)


@pytest.mark.parametrize("new", [1, 130])
@pytest.mark.parametrize("exponent", [-105, -120])
def test_small_keys_under_large_queries(TF, new, exponent):
    """Keys of scales below 2^-100 that the queries make up for: scores of ordinary size."""
    lens = [300]
    b = P.Batch(33, lens, [new], 1, 64, 32, "int8").fill(lens, (exponent - 1, exponent))
    b.vs[b.host_table.flatten()] = 2.0**-6
    Q = (b.rand(b.rows, 4, 64) * 2.0**(-exponent - 6)).bfloat16()
    check(TF, b, Q, 0.125, max_new=new)


@pytest.mark.parametrize("new", [1, 130])
def test_tiny_scale_of_float16_queries(TF, new):
    lens = [300]
    b = P.Batch(34, lens, [new], 1, 128, 16, "e4m3").fill(lens, (-8, -4))
    zero_keys(b, 0, 3, 2.0**-126)
    zero_keys(b, 0, 18, 2.0**-126)
    check(TF, b, b.rand(b.rows, 4, 128, dtype=torch.float16), 1e-36, max_new=new)
