"""Norm and rotation of queries and keys on the GPU against a plain implementation in 64 bits."""
import pytest
import torch

import kvcache_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def TF():
    from deepx_b200 import tensorfunc
    return tensorfunc


def check(got, x, weight, inv, positions, eps, interleaved):
    """The norm: a float32 sum of dim squares (dim/32 + 6 additions one after the other in a lane and over lanes, each 2^-24; half of
    it after the root), a division, a root and two products: below (dim/64 + 10) * 2^-24.  The rotation: sine and cosine are off by
    2^-22 (the fraction of a turn, at most 1/2, is rounded to float32: 2^-25 turns = 2^-22.3; the function: 2^-24), two products and a sum
    2^-23 of the pair's size.  Then one rounding."""
    want, size = P.rope(x, weight, inv, positions, eps, interleaved)
    work = size * ((x.shape[-1] / 64 + 10) * 2.0**-24 + 2.0**-22 + 2.0**-23)
    bound = work + P.half_step(x.dtype) * (want.abs() + work) + torch.finfo(x.dtype).tiny
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound).max()):.3f} of the bound"


def inputs(dtype, tokens, qh, kh, dim, rotated, seed=0):
    g = torch.Generator().manual_seed(seed + tokens + dim)
    dt = P.FLOATS[dtype]
    Q, K = ((torch.randn(tokens, h, dim, generator=g) * 3).to(dt).cuda() for h in (qh, kh))
    qw, kw = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dt).cuda() for _ in "qk")
    inv = (10000.0 ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / max(rotated, 1))).float().cuda()
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g).int().cuda()
    return Q, K, qw, kw, inv, pos


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,qh,kh,dim,rotated", [(1, 1, 1, 128, 128), (5, 32, 8, 128, 128), (33, 14, 2, 64, 64), (7, 3, 1, 96, 96), (9, 4, 4, 256, 64),
                                                      (3, 5, 2, 80, 32), (4, 2, 1, 512, 512), (6, 3, 2, 7, 4), (2, 1, 1, 1, 0), (8, 6, 0, 64, 0),
                                                      (11, 2, 2, 72, 48), (300, 2, 1, 16, 16), (10, 2, 3, 100, 20), (4, 1, 2, 48, 36), (5, 3, 1, 8, 8)])
def test_norm_and_rotation(TF, dtype, interleaved, tokens, qh, kh, dim, rotated):
    Q, K, qw, kw, inv, pos = inputs(dtype, tokens, qh, kh, dim, rotated)
    for eps, a, b in ((1e-6, qw, kw), (1e-5, None, kw), (None, None, None)):
        Qo, Ko = torch.empty_like(Q), torch.empty_like(K)
        TF.qknorm_rope(Q, K, a, b, inv, pos, eps, interleaved, Qo, Ko)
        check(Qo, Q, a, inv, pos, eps, interleaved)
        check(Ko, K, b, inv, pos, eps, interleaved)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_far_and_negative_positions(TF, dtype):
    Q, K, qw, kw, inv, _ = inputs(dtype, 8, 4, 2, 128, 128)
    pos = torch.tensor([0, 1, -1, 2**31 - 1, 10**7 + 1, 12345678901, -(10**10), 2**40 + 1], device="cuda")
    Qo, Ko = torch.empty_like(Q), torch.empty_like(K)
    TF.qknorm_rope(Q, K, qw, kw, inv, pos, 1e-6, False, Qo, Ko)
    # float64 angles of 10^12: the product's rounding is 2^-53 * 2^40 = 2^-13 of a radian there, in the plain form too
    near = pos.abs() < 2**31
    check(Qo[near], Q[near], qw, inv, pos[near], 1e-6, False)
    check(Ko[near], K[near], kw, inv, pos[near], 1e-6, False)
    assert torch.isfinite(Qo).all()


@pytest.mark.parametrize("first", [0, 1, 4, 8])
def test_in_place_in_a_packed_projection(TF, first):
    """Queries and keys as columns of the rows [q | k | v] of one projection, aligned and not; the values stay."""
    for dtype in (torch.bfloat16, torch.float32):
        g = torch.Generator().manual_seed(first)
        buf = torch.randn(19, first + (6 + 2 + 2) * 64, generator=g).to(dtype).cuda()
        before = buf.clone()
        heads = buf[:, first:].unflatten(1, (10, 64))
        Q, K = heads[:, :6], heads[:, 6:8]
        q, k = Q.clone(), K.clone()
        w = torch.rand(64, generator=g).to(dtype).cuda()
        inv = (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().cuda()
        pos = torch.arange(19, device="cuda")
        TF.qknorm_rope(Q, K, w, w, inv, pos, 1e-6, False, Q, K)
        check(Q, q, w, inv, pos, 1e-6, False)
        check(K, k, w, inv, pos, 1e-6, False)
        assert torch.equal(buf[:, :first], before[:, :first]) and torch.equal(buf[:, first + 512:], before[:, first + 512:])


def test_rows_of_zeros_and_infinities(TF):
    """A head of zeros stays zero (eps divides); one infinite element spoils its own head alone."""
    Q, K, qw, kw, inv, pos = inputs("bfloat16", 4, 4, 2, 64, 64)
    Q[1, 2] = 0
    clean, out, Ko = torch.empty_like(Q), torch.empty_like(Q), torch.empty_like(K)
    TF.qknorm_rope(Q, K, qw, kw, inv, pos, 1e-6, False, clean, Ko)
    assert not clean[1, 2].any()
    Q[2, 1, 5] = float("inf")
    TF.qknorm_rope(Q, K, qw, kw, inv, pos, 1e-6, False, out, Ko)
    out[2, 1] = clean[2, 1]
    assert torch.equal(out, clean)


def test_no_tokens_no_heads(TF):
    Q, K, qw, kw, inv, pos = inputs("bfloat16", 0, 4, 2, 64, 64)
    TF.qknorm_rope(Q, K, qw, kw, inv, pos, 1e-6, False, torch.empty_like(Q), torch.empty_like(K))


def test_weights_and_rotation_on_another_stream(TF):
    Q, K, qw, kw, inv, pos = inputs("bfloat16", 64, 32, 8, 128, 128)
    want_q, want_k = torch.empty_like(Q), torch.empty_like(K)
    TF.qknorm_rope(Q, K, qw, kw, inv, pos, 1e-6, False, want_q, want_k)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    Qo, Ko = torch.empty_like(Q), torch.empty_like(K)
    with torch.cuda.stream(st):
        TF.qknorm_rope(Q, K, qw, kw, inv, pos, 1e-6, False, Qo, Ko)
    torch.cuda.synchronize()
    assert torch.equal(Qo, want_q) and torch.equal(Ko, want_k)
