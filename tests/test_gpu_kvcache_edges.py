"""Attention over the 8-bit cache where its numbers lie far apart: keys and queries near the ends of float32, values of very different
scales, pages behind a window.  Plain implementations in 64 bits and the bounds: kvcache_plain.py."""
import pytest
import torch

import kvcache_plain as P
from test_gpu_qknorm import check as check_rope

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


# ---- values of pages whose scales lie far apart ------------------------------------------------------------------
def apart(seed, lens, new, heads, dim, page, fmt, exponents, gap, favoured):
    """A batch whose pages have the value scales 2^exponents[column % len]; keys such that a query of ones scores `gap` (natural
    logarithm; up to twice that) less on every page but the columns of `favoured`."""
    b = P.Batch(seed, lens, new, heads, dim, page, fmt).fill(lens)
    plus, minus = (0x01, 0xFF) if fmt == "int8" else (0x38, 0xB8)  # the codes of 1 and -1
    for i, n in enumerate(lens):
        for c in range(-(-n // page)):
            at = int(b.host_table[i, c])
            b.k.view(torch.uint8)[at] = plus if c % len(exponents) in favoured else minus
            b.ks[at] = gap / 2 / dim / 0.125
            b.vs[at] = 2.0 ** exponents[c % len(exponents)]
    b.ks.copy_(torch.ldexp(torch.ones_like(b.ks), torch.frexp(b.ks.nan_to_num(1.0))[1]))
    return b


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 3, 140])
@pytest.mark.parametrize("exponents,favoured", [
    ((0, -26), (1,)), ((-26, 0), (0,)), ((0, -40), (1,)), ((-24, 10, -24), (0,)), ((30, -90), (1,)), ((-126, 20), (0,)), ((100, -126), (1,)),
    ((-10, -126, -10), (1,)), ((-6, -8, -30, -7), (2, 3)), ((-126,), (0,)), ((110,), (0,)), ((-126, -100), (0,))])
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 128)])
def test_values_of_scales_far_apart(TF, fmt, new, exponents, favoured, page, dim):
    """A row keeps the bits of the page it weighs, whatever scale the pages beside it have."""
    lens = [600, 333]
    for gap in (60.0, 6.0):
        b = apart(35 + page, lens, [new, new], 1, dim, page, fmt, exponents, gap, favoured)
        check(TF, b, torch.ones(b.rows, 4, dim, dtype=torch.bfloat16, device="cuda"), 0.125, max_new=new)
        check(TF, b, b.rand(b.rows, 4, dim, dtype=torch.bfloat16), 0.125, max_new=new)


@pytest.mark.parametrize("new", [1, 140])
def test_written_values_of_scales_far_apart(TF, new):
    """The same through kvcache_write: a token of 10^9 in a history of values of 10^-3, behind every row's attention or before it."""
    lens, dim, page = [500], 64, 16
    for where in (5, 250, 350, 499):
        b = P.Batch(36, lens, lens, 1, dim, page, "int8")
        K, V = b.rand(500, 1, dim), b.rand(500, 1, dim) * 1e-3
        V[where] *= 1e12
        K[where] = -4.0
        TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
        b.new, b.host_starts, b.rows = [new], [0, new], new
        b.starts = torch.tensor([0, new], dtype=torch.int32, device="cuda")
        Q = torch.full((new, 2, dim), 3.0, device="cuda").bfloat16()
        check(TF, b, Q, 0.125, max_new=new)


@pytest.mark.parametrize("new", [1, 4, 140])
@pytest.mark.parametrize("power", [20, 24, 27, 40, 80])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_of_scales_far_apart_under_huge_scores(TF, new, power, dim):
    """Scores of about 2^power, the same for every token of half of the pages and far below on the others: each of those tokens has
    the same weight, whatever its page's value scale is, and no bit of a scale is lost beside the score.  Weights are exact here but for
    their rounding to 16 bits and the exponential's 2^-21: 2^-11 + 2^-15 of the mean |v|, as in kvcache_plain.attention_rows, and its
    fixed term of the largest scale among pages of one weight."""
    lens, page = [900, 500], 16
    exponents = (-6, -3, -30, -7, -12, -3, -20, -5, -6)
    b = apart(43, lens, [new, new], 1, dim, page, "int8", exponents, 1.0, (0, 2, 4, 6, 8))
    b.ks[b.host_table.flatten()] = 2.0 ** (power - 20)
    Q = (torch.randint(4, 8, (b.rows, 4, dim), generator=b.g).cuda() * 2.0**18).bfloat16()  # the products and their sums are exact
    out = attend(TF, b, Q, 1.0 / dim, max_new=new).double()
    assert int(b.flag) == 0
    for i, n in enumerate(lens):
        v = b.history(b.v, b.vs, i)[:, 0]
        token = torch.arange(n, device="cuda")
        chosen = (token // page) % len(exponents) % 2 == 0
        for t in range(new):
            use = v[: n - new + t + 1][chosen[: n - new + t + 1]]
            want, size = use.mean(0), use.abs().mean(0)
            bound = size * (2.0**-11 + 2.0**-15 + n * 2.0**-23) + 2.0**-30 * 127 * 2.0**-6
            off = (out[b.host_starts[i] + t] - want).abs()
            assert bool((off <= bound + P.half_step(torch.bfloat16) * (want.abs() + bound)).all())


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 4, 140])
@pytest.mark.parametrize("exponents", [(0, -6, -5), (0,), (-6, 0, 0), (0, 100, -126)])
def test_values_of_scale_zero(TF, fmt, new, exponents):
    """Pages of value scale zero (never written) have their share of the sum and add nothing, whatever their codes are; exponent 0 stands for one."""
    lens, page = [500, 33 + new], 16
    b = P.Batch(45, lens, [new, new], 1, 64, page, fmt).fill(lens, (-7, -5))
    for i, n in enumerate(lens):
        for c in range(-(-n // page)):
            e = exponents[c % len(exponents)]
            b.vs[int(b.host_table[i, c])] = 2.0**e if e else 0.0
    check(TF, b, b.rand(b.rows, 4, 64, dtype=torch.bfloat16), 0.125, max_new=new)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [4, 140])
@pytest.mark.parametrize("size", [float("inf"), 1e30, 1e7])
def test_rows_beside_one_of_huge_scores(TF, fmt, new, size):
    """A row of huge or infinite queries does not harm the rows beside it (some of a warp may then be rounded in another order)."""
    lens = [300, 40 + new]
    for dim in (64, 128):
        b = P.Batch(46, lens, [new, new], 1, dim, 16, fmt).fill(lens, (-9, -4))
        Q = b.rand(b.rows, 4, dim, dtype=torch.bfloat16)
        bad = Q.clone()
        bad[1, 2] = size
        bad[new + 2, 0] = -size
        out = attend(TF, b, bad, 0.125, max_new=new).double()
        want, bound = P.attention_rows(b, Q, 0.125)
        for row, head in ((1, 2), (new + 2, 0)):
            out[row, head] = want[row, head]
        assert bool(((out - want).abs() <= bound + P.half_step(Q.dtype) * (want.abs() + bound)).all()) and int(b.flag) == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("new", [1, 4, 140])
def test_scales_that_are_no_powers_of_two(TF, fmt, new):
    """A cache that another program made: scales of any positive float, a few of them powers of two.  A scale may lie below its power of two
    by up to half, the largest weight then 2^5 times: twice the fixed term, so twice the bound."""
    for spread in (1.0, 12.0):
        lens = [700, 90 + new]
        b = P.Batch(44, lens, [new, new], 2, 96, 16, fmt).fill(lens, (-9, -7))
        for scales in (b.ks, b.vs):
            u = torch.rand(scales.shape, generator=b.g).cuda()
            scales.copy_(torch.where(u < 0.2, scales, scales * torch.exp2(u * 2 - 1)))
        b.vs *= torch.exp2((torch.rand(b.vs.shape, generator=b.g).cuda() - 0.5) * spread)
        Q = b.rand(b.rows, 6, 96, dtype=torch.bfloat16)
        want, bound = P.attention_rows(b, Q, 0.1)
        off = (attend(TF, b, Q, 0.1, max_new=new).double() - want).abs()
        bound = 2 * bound
        assert bool((off <= bound + P.half_step(Q.dtype) * (want.abs() + bound)).all()) and int(b.flag) == 0


@pytest.mark.parametrize("new", [1, 5, 140])
def test_rows_do_not_depend_on_pages_they_do_not_see(TF, new):
    """What stands in the pages in front of a row's window and behind the row (its scales too) does not change one bit of it."""
    lens, window = [400], 48
    b = P.Batch(37, lens, [new], 1, 64, 16, "e4m3").fill(lens, (-30, -2))
    Q = b.rand(b.rows, 4, 64, dtype=torch.bfloat16)
    clean = attend(TF, b, Q, 0.125, window, new)
    first = max(0, 400 - new - window + 1) // 16
    for c in range(first):
        at = int(b.host_table[0, c])
        b.vs[at], b.ks[at] = 2.0 ** (c % 40), 2.0**-100
    assert torch.equal(clean, attend(TF, b, Q, 0.125, window, new)) and int(b.flag) == 0
    # rows in front of the last page: its scale is not theirs
    if new > 16:
        b.vs[int(b.host_table[0, 24])] = 2.0**60  # tokens 384-399
        out = attend(TF, b, Q, 0.125, window, new)
        check_rows = new - 16
        want, bound = P.attention_rows(b, Q, 0.125, window)
        want, bound = want[:check_rows], bound[:check_rows]
        off = (out[:check_rows].double() - want).abs()
        assert bool((off <= bound + P.half_step(Q.dtype) * (want.abs() + bound) + torch.finfo(Q.dtype).tiny).all())


@pytest.mark.parametrize("fmt,exponent", [("int8", 120), ("e4m3", 118)])
@pytest.mark.parametrize("lens,new,q_heads,dim", [([3000], [1], 4, 64), ([3000], [150], 4, 64), ([40000], [1], 2, 128), ([900, 700, 650], [1, 1, 1], 12, 128),
                                                  ([900], [1], 2, 256)])
def test_values_near_the_end_of_float32(TF, fmt, exponent, lens, new, q_heads, dim):
    """Averages of values near float32's largest, in one part and joined out of few and of many: nothing on the way is larger than they are."""
    b = P.Batch(39, lens, new, 1, dim, 16, fmt).fill(lens, (-9, -8))
    b.vs[b.host_table.flatten()] = 2.0**exponent
    v = b.v.view(torch.uint8)
    v &= 0x7F  # positive, up to the largest code
    if fmt == "e4m3":
        v[v == 0x7F] = 0x7E
    check(TF, b, b.rand(b.rows, q_heads, dim, dtype=torch.bfloat16), 0.05, max_new=max(new))


# ---- pages behind a window ------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page,q_heads,dim", [(16, 4, 64), (32, 4, 128), (16, 8, 256), (64, 20, 96), (128, 2, 64)])
@pytest.mark.parametrize("window,lens,new", [(1, [500, 64, 3], [1, 1, 1]), (100, [500, 333, 129], [1, 2, 4]), (33, [700, 256], [1, 16]),
                                             (17, [700, 300, 5], [300, 100, 5]), (129, [900, 400], [130, 260])])
def test_pages_behind_the_window_are_not_looked_at(TF, fmt, page, q_heads, dim, window, lens, new):
    """Pages in front of every row's window may have been given back: their table entries are of no page, the pages' bytes and scales
    anything; no flag, and not one bit of the result is another."""
    b = P.Batch(38 + page, lens, new, 2, dim, page, fmt).fill(lens)
    Q = b.rand(b.rows, 2 * q_heads, dim, dtype=torch.bfloat16)
    for hint in (max(new), 0):
        want = attend(TF, b, Q, dim ** -0.5, window, hint)
        table = b.table.clone()
        for i, (n, m) in enumerate(zip(lens, new)):
            for c in range(max(0, n - m - window + 1) // page):
                table[i, c] = (-1, b.pages, 2**31 - 1, -2**31)[c % 4]
        got = attend(TF, b, Q, dim ** -0.5, window, hint, table)
        assert int(b.flag) == 0
        assert torch.equal(got, want)
    b.table = table
    check(TF, b, Q, dim ** -0.5, window, max(new))
    # the page that the first row's window begins in is looked at
    i = 0
    c = max(0, lens[i] - new[i] - window + 1) // page
    table = b.table.clone()
    table[i, c] = -1
    attend(TF, b, Q, dim ** -0.5, window, max(new), table)
    assert int(b.flag) == 1


# ---- columns of one buffer ------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("first", [0, 1])
def test_outputs_beside_one_another_in_one_buffer(TF, dtype, first):
    """Keys and values read into columns of the same rows, queries and keys turned into such columns, an output beside its queries: what a
    packed projection's buffer is used for.  The columns between stay as they were."""
    dt, lens, new = P.FLOATS[dtype], [70, 9], [64, 9]
    b = P.Batch(40, lens, new, 2, 64, 16, "int8").fill(lens)
    b.table = b.host_table.int().cuda()
    buf = torch.full((b.rows, first + 600), 7.0, dtype=dt, device="cuda")

    def columns(at, heads):
        return buf[:, first + at: first + at + heads * 64].unflatten(1, (heads, 64))

    K, V = (torch.empty(b.rows, 2, 64, dtype=dt, device="cuda") for _ in "kv")
    TF.kvcache_read(*b.cache(), *b.seqs(), K, V, b.flag)
    TF.kvcache_read(*b.cache(), *b.seqs(), columns(320, 2), columns(128, 2), b.flag)
    assert torch.equal(columns(320, 2), K) and torch.equal(columns(128, 2), V)
    inv = (10000.0 ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().cuda()
    pos = torch.arange(b.rows, device="cuda")
    Q = b.rand(b.rows, 4, 64, dtype=dt)
    TF.qknorm_rope(Q, K, None, None, inv, pos, 1e-6, False, columns(0, 4), columns(320, 2))
    check_rope(columns(0, 4), Q, None, inv, pos, 1e-6, False)  # another kernel off 16-byte boundaries: other bits than that of whole tensors
    check_rope(columns(320, 2), K, None, inv, pos, 1e-6, False)
    if dt != torch.float32:
        out, turned = torch.empty_like(Q), columns(0, 4).clone()
        TF.kvcache_attention(turned, *b.cache(), *b.seqs(), 0.125, 64, 0, out, b.flag)
        TF.kvcache_attention(columns(0, 4), *b.cache(), *b.seqs(), 0.125, 64, 0, columns(256, 4), b.flag)
        assert torch.equal(columns(256, 4), out) and torch.equal(columns(0, 4), turned)
    assert bool((buf[:, :first] == 7).all()) and bool((buf[:, first + 512:] == 7).all())


def test_overlapping_outputs_are_an_error(TF):
    b = P.Batch(41, [20], [20], 1, 64, 16, "int8").fill([20])
    K = torch.zeros(20, 1, 64, device="cuda")
    inv, pos = torch.zeros(32, device="cuda"), torch.arange(20, device="cuda")
    with pytest.raises(Exception, match="overlap"):
        TF.kvcache_read(*b.cache(), *b.seqs(), K, K)
    with pytest.raises(Exception, match="overlap"):
        TF.kvcache_write(K, K, *b.seqs(), b.k, b.k, b.ks, b.vs)
    with pytest.raises(Exception, match="overlap"):
        TF.qknorm_rope(K, K.clone(), None, None, inv, pos, 1e-6, False, K, K)


# ---- head sizes above 128 that are no power of two ---------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dim", [144, 208, 240])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_large_head_sizes(TF, fmt, dim, page):
    """Written, read back and attended: single tokens, few and many rows, few parts and many, a window."""
    for lens, new in (([1, 300, 17], [1, 1, 1]), ([130, 70], [130, 33]), ([9000], [1]), ([0, 2, 600], [3, 1, 5])):
        b = P.Batch(42 + dim, lens, new, 2, dim, page, fmt, extra_rows=1).fill([max(0, n - m) for n, m in zip(lens, new)], (-9, -3))
        K, V = b.rand(b.rows, 2, dim, dtype=torch.bfloat16), b.rand(b.rows, 2, dim, dtype=torch.bfloat16)
        want = P.write(b, K, V)
        TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
        for got, w in zip(b.cache(), want):
            assert torch.equal(got.cpu().view(torch.uint8), w.view(torch.uint8))
        R, S = torch.full_like(K, 7.0), torch.full_like(V, 7.0)
        TF.kvcache_read(*b.cache(), *b.seqs(), R, S, b.flag)
        for got, codes, scales in ((R, b.k, b.ks), (S, b.v, b.vs)):
            for i, (n, m) in enumerate(zip(lens, new)):
                at = b.host_starts[i] + max(0, m - n)
                assert torch.equal(got[at: b.host_starts[i] + m], b.history(codes, scales, i)[max(0, n - m):].to(K.dtype))
        for window in (0, 50):
            check(TF, b, b.rand(b.rows, 6, dim, dtype=torch.bfloat16), dim ** -0.5, window, max(new))
