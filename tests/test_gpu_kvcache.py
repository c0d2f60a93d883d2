"""The 8-bit key/value cache on the GPU: writing, reading back and attention, against plain implementations in 64 bits
(kvcache_plain.py), where they can go wrong: empty and one-token sequences, pages that end inside a tile, rows that see no
key, stale bytes, bad tables, strides, other streams, captured graphs, offsets beyond 32 bits."""
import pytest
import torch

import kvcache_plain as P

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def TF():
    from deepx_b200 import tensorfunc
    return tensorfunc


def same_bits(a, b, what):
    a, b = a.cpu(), b.cpu()
    if a.element_size() == 1:
        a, b = a.view(torch.uint8), b.view(torch.uint8)
    else:
        a, b = a.view(torch.int32), b.view(torch.int32)
    assert torch.equal(a, b), f"{what}: {int((a != b).sum())} of {a.numel()} differ"


# ---- write ---------------------------------------------------------------------------------------------------
# (lens, new): one token each into empty, partly filled and full pages; prompts over several pages; sequences without new
# tokens; more new tokens than the sequence holds; an empty one
WRITES = [
    ([1], [1]),
    ([16, 17, 33, 64, 65], [1, 1, 1, 1, 1]),
    ([5, 0, 40, 130], [5, 0, 0, 129]),
    ([100, 3, 257], [37, 7, 200]),
]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,new", WRITES)
@pytest.mark.parametrize("page,heads,dim", [(16, 2, 64), (64, 3, 80), (128, 1, 128), (32, 1, 16)])
def test_write(TF, dtype, fmt, lens, new, page, heads, dim):
    b = P.Batch(len(lens) * page + dim, lens, new, heads, dim, page, fmt, extra_rows=3)
    b.fill([max(0, n - m) for n, m in zip(lens, new)], (-9, -3))
    K, V = (b.rand(b.rows, heads, dim) * s for s in (3.0, 0.01))
    K, V = K.to(P.FLOATS[dtype]), V.to(P.FLOATS[dtype])
    want = P.write(b, K, V)
    TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
    for g, w, name in zip(b.cache(), want, ("k", "v", "k_scale", "v_scale")):
        same_bits(g, w, name)
    assert int(b.flag) == 0


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_scale_grows_falls_and_repeats(TF, fmt):
    """Token by token into one page: the scale follows the largest value so far; a page begun anew forgets it; the same write
    twice changes nothing."""
    page, dim = 16, 32
    b = P.Batch(3, [16], [1], 1, dim, page, fmt, extra_cols=0)
    sizes = [1e-3, 5.0, 2e-4, 5.0, 300.0, 0.0, 448.0, 127.0, 128.0, 1e-30, 1e4, 1.0, 2.0, 3.0, 60000.0, 4.0]
    for t, size in enumerate(sizes):
        b.lens, b.length = [t + 1], torch.tensor([t + 1], dtype=torch.int32, device="cuda")
        K = b.rand(1, 1, dim).clamp(-1, 1) * size
        K[0, 0, 0] = size
        want = P.write(b, K, -K)
        for _ in range(2):
            TF.kvcache_write(K, -K, *b.seqs(), *b.cache(), b.flag)
            for g, w in zip(b.cache(), want):
                same_bits(g, w, f"token {t}")
    b.lens, b.length = [1], torch.tensor([1], dtype=torch.int32, device="cuda")
    K = b.rand(1, 1, dim) * 1e-3
    want = P.write(b, K, K)
    TF.kvcache_write(K, K, *b.seqs(), *b.cache(), b.flag)
    for g, w in zip(b.cache(), want):
        same_bits(g, w, "begun anew")
    assert float(b.ks.nan_to_num().max()) < 1e-3


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_of_what_is_not_finite(TF, fmt):
    b = P.Batch(4, [20], [20], 1, 16, 32, fmt)
    K, V = b.rand(20, 1, 16), b.rand(20, 1, 16)
    K[3, 0, 5], K[4, 0, 6], K[7, 0, 7] = float("inf"), -float("inf"), float("nan")
    V[:] = float("inf")
    want = P.write(b, K, V)
    TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
    for g, w, name in zip(b.cache(), want, ("k", "v", "k_scale", "v_scale")):
        same_bits(g, w, name)
    assert int(b.flag) == 4
    assert float(b.vs[int(b.host_table[0, 0])]) == 2.0**-126


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_write_smallest_and_largest_values(TF, fmt):
    """Subnormal inputs, float32's largest, zeros: the scale stays a normal power of two."""
    for value in (0.0, 1e-45, 1e-40, 1.1754944e-38, 3.4e38, torch.finfo(torch.float32).max):
        b = P.Batch(5, [4], [4], 1, 16, 16, fmt)
        K = torch.full((4, 1, 16), value, device="cuda")
        K[1] *= 0.5
        want = P.write(b, K, K)
        TF.kvcache_write(K, K, *b.seqs(), *b.cache(), b.flag)
        for g, w in zip(b.cache(), want):
            same_bits(g, w, f"value {value}")


def test_write_from_a_packed_projection_and_unaligned(TF):
    """K and V as column ranges of one projection's rows, also where no 16-byte load is possible."""
    for first in (0, 1, 3):
        b = P.Batch(6, [70, 9], [64, 9], 2, 48, 32, "int8")
        b.fill([6, 0])
        buf = b.rand(b.rows, 5 * 96 + first, dtype=torch.bfloat16)
        K, V = (buf[:, first + c * 96: first + (c + 1) * 96].unflatten(1, (2, 48)) for c in (2, 4))
        want = P.write(b, K, V)
        TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
        for g, w in zip(b.cache(), want):
            same_bits(g, w, f"first column {first}")


def test_write_ragged_batch_of_many(TF):
    """One long prompt among many single tokens: chunks with many first tokens, and more sequences than a block has threads."""
    new = [1] * 150 + [700] + [1, 0, 2] * 30
    lens = [n + 7 * i % 90 for i, n in enumerate(new)]
    b = P.Batch(7, lens, new, 1, 32, 16, "e4m3")
    b.fill([n - m for n, m in zip(lens, new)])
    K, V = b.rand(b.rows, 1, 32), b.rand(b.rows, 1, 32)
    want = P.write(b, K, V)
    TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
    for g, w in zip(b.cache(), want):
        same_bits(g, w, "ragged")


# ---- read ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,new,page,heads,dim", [([1], [1], 16, 1, 16), ([100, 0, 33], [100, 0, 33], 32, 3, 80), ([5, 300], [9, 250], 64, 2, 128),
                                                     ([513, 7], [1, 7], 256, 1, 256)])
def test_read(TF, dtype, fmt, lens, new, page, heads, dim):
    b = P.Batch(8, lens, new, heads, dim, page, fmt, extra_rows=2).fill(lens, (-30, 10))
    K, V = (torch.full((b.rows, heads, dim), 7.0, dtype=P.FLOATS[dtype], device="cuda") for _ in "kv")
    TF.kvcache_read(*b.cache(), *b.seqs(), K, V, b.flag)
    assert int(b.flag) == 0
    for got, codes, scales in ((K, b.k, b.ks), (V, b.v, b.vs)):
        want = torch.full((b.rows, heads, dim), 7.0, dtype=torch.float64, device="cuda")
        for i, (n, m) in enumerate(zip(lens, new)):
            h = b.history(codes, scales, i)
            want[b.host_starts[i]: b.host_starts[i] + m] = 0.0
            want[b.host_starts[i] + max(0, m - n): b.host_starts[i] + m] = h[max(0, n - m):]
        assert torch.equal(got, want.to(P.FLOATS[dtype]))


# ---- attention -----------------------------------------------------------------------------------------------
def check_attention(TF, b, Q, scale, window=0, max_new=0, Out=None):
    want, bound = P.attention(b, Q, scale, window)
    filler = torch.full(Q.shape, 3.0, dtype=Q.dtype, device=Q.device)
    if Out is None:
        Out = filler.clone()
    else:
        Out.copy_(filler)
    TF.kvcache_attention(Q, *b.cache(), *b.seqs(), scale, max_new, window, Out, b.flag)
    from deepx_b200 import _native as N
    N.check(N.lib.dx_kvcache_status(None))
    assert int(b.flag) == 0
    last = b.host_starts[-1]
    assert torch.equal(Out[last:], filler[last:]), "rows behind the last sequence changed"
    got = Out[:last].double()
    bound = bound[:last] + P.half_step(Q.dtype) * (want[:last].abs() + bound[:last]) + torch.finfo(Q.dtype).tiny
    off = (got - want[:last]).abs()
    assert torch.isfinite(got).all()
    assert bool((off <= bound).all()), f"off by up to {float((off / bound).max()):.3f} of the bound"
    return Out


DECODES = [  # (lens, new)
    ([1], [1]),
    ([0, 1, 2, 15, 16, 17, 63, 64, 65], [1] * 9),
    ([1000, 129, 5], [1, 1, 1]),
    ([300, 2, 40], [4, 3, 2]),  # rows in front of position 0 among them: see no key
    ([77, 0, 31], [0, 0, 1]),
]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,new", DECODES)
@pytest.mark.parametrize("page,q_heads,kv_heads,dim", [(64, 8, 2, 128), (16, 7, 1, 64), (32, 3, 3, 96), (128, 20, 1, 16), (256, 4, 2, 256), (64, 40, 1, 80)])
def test_attention_of_few_rows(TF, dtype, fmt, lens, new, page, q_heads, kv_heads, dim):
    b = P.Batch(len(lens) + page, lens, new, kv_heads, dim, page, fmt, extra_rows=2).fill(lens)
    Q = b.rand(b.rows, q_heads, dim, dtype=P.FLOATS[dtype])
    check_attention(TF, b, Q, dim ** -0.5, max_new=max(new))


@pytest.mark.parametrize("dtype,fmt", [("float16", "int8"), ("bfloat16", "e4m3"), ("bfloat16", "int8"), ("float16", "e4m3")])
@pytest.mark.parametrize("lens,new", [([200], [200]), ([130, 129, 128], [130, 129, 128]), ([700, 90, 3], [301, 90, 5]), ([513, 257, 1, 0], [40, 257, 1, 2]), ([2000], [150])])
@pytest.mark.parametrize("page,q_heads,kv_heads,dim", [(64, 8, 2, 128), (16, 7, 1, 64), (32, 3, 3, 96), (256, 4, 2, 256), (128, 6, 1, 112), (64, 2, 2, 16)])
def test_attention_of_prompts(TF, dtype, fmt, lens, new, page, q_heads, kv_heads, dim):
    b = P.Batch(len(lens) * 7 + page, lens, new, kv_heads, dim, page, fmt, extra_rows=1).fill(lens)
    Q = b.rand(b.rows, q_heads, dim, dtype=P.FLOATS[dtype])
    for hint in (max(new), 0, 1):
        check_attention(TF, b, Q, dim ** -0.5, max_new=hint)


@pytest.mark.parametrize("window", [1, 5, 16, 100, 129, 4096])
@pytest.mark.parametrize("lens,new", [([500, 64, 3], [1, 1, 1]), ([500, 64, 3], [300, 64, 2])])
def test_attention_window(TF, window, lens, new):
    b = P.Batch(9, lens, new, 2, 64, 32, "int8").fill(lens)
    check_attention(TF, b, b.rand(b.rows, 6, 64, dtype=torch.bfloat16), 0.125, window, max(new))


@pytest.mark.parametrize("new", [1, 200])
def test_attention_scales_far_apart(TF, new):
    """Pages whose scales differ by many powers of two, pages of zeros (the smallest scale), a scale of any float."""
    lens = [1500]
    b = P.Batch(10, lens, [new], 1, 128, 16, "e4m3").fill(lens, (-20, -2))
    b.vs[b.host_table[0, 3].item()] = 2.0**-126
    b.ks[b.host_table[0, 5].item()] = 2.0**-126
    b.vs[b.host_table[0, 7].item()] = 0.3
    b.ks[b.host_table[0, 8].item()] = 0.0007
    check_attention(TF, b, b.rand(b.rows, 4, 128, dtype=torch.float16), 0.02, max_new=new)


@pytest.mark.parametrize("new", [1, 150])
def test_attention_of_large_and_small_queries(TF, new):
    """bfloat16 queries beyond float16's range, zero rows, rows of one large element; scores that saturate the softmax."""
    lens = [400]
    b = P.Batch(11, lens, [new], 1, 64, 64, "int8").fill(lens, (-7, -7))
    for size in (1e-30, 1e6, 1e30):
        Q = b.rand(b.rows, 4, 64, dtype=torch.bfloat16) * size
        Q[:, 1] = 0
        Q[:, 2, 1:] *= 1e-3
        check_attention(TF, b, Q, 0.125 / size, max_new=new)
    check_attention(TF, b, b.rand(b.rows, 4, 64, dtype=torch.bfloat16), 3.0, max_new=new)


@pytest.mark.parametrize("new", [1, 130])
def test_attention_strides(TF, new):
    """Queries as columns of a packed projection, outputs as columns of a wider buffer, also off 16-byte boundaries."""
    for first in (0, 1):
        lens = [new + 20, new]
        b = P.Batch(12, lens, [new, new], 2, 64, 16, "int8").fill(lens)
        buf = b.rand(b.rows, 600 + first, dtype=torch.bfloat16)
        Q = buf[:, first: first + 256].unflatten(1, (4, 64))
        Out = torch.zeros(b.rows, 300 + first, dtype=torch.bfloat16, device="cuda")
        check_attention(TF, b, Q, 0.125, max_new=new, Out=Out[:, first: first + 256].unflatten(1, (4, 64)))
        assert not Out[:, :first].any() and not Out[:, first + 256:].any()


def test_attention_row_of_no_number_stays_alone(TF):
    """A query that is not a number makes its own row so, no other."""
    for new in (4, 140):
        lens = [300]
        b = P.Batch(13, lens, [new], 1, 64, 64, "e4m3").fill(lens)
        Q = b.rand(b.rows, 4, 64, dtype=torch.bfloat16)
        clean, out = torch.empty_like(Q), torch.empty_like(Q)
        TF.kvcache_attention(Q, *b.cache(), *b.seqs(), 0.125, new, 0, clean)
        bad = Q.clone()
        bad[1, 2, 3] = float("nan")
        TF.kvcache_attention(bad, *b.cache(), *b.seqs(), 0.125, new, 0, out)
        assert torch.isnan(out[1, 2]).all()
        out[1, 2] = clean[1, 2]
        assert torch.equal(out, clean)


@pytest.mark.parametrize("q_heads,kv_heads,dim,page", [(14, 2, 64, 16), (8, 2, 128, 64)])
def test_attention_of_a_mixed_batch(TF, q_heads, kv_heads, dim, page):
    """Prompts, prompts continued and single tokens in one call: items of one tile of rows and of two in the same block, many of each."""
    lens = [5000, 700, 3000, 900, 64, 2500, 4000, 1, 1300, 2222, 650, 3333]
    new = [1, 700, 300, 1, 64, 37, 500, 1, 19, 1, 650, 128]
    b = P.Batch(25, lens, new, kv_heads, dim, page, "e4m3", extra_rows=1).fill(lens)
    check_attention(TF, b, b.rand(b.rows, q_heads, dim, dtype=torch.bfloat16), dim ** -0.5, max_new=700)


@pytest.mark.parametrize("dim,group", [(128, 4), (64, 8), (96, 1), (64, 1)])
def test_attention_of_many_short_sequences(TF, dim, group):
    """Short sequences with few new tokens each, without a hint of how few, so that they go the prompts' way too: rows that see nothing,
    one tile of rows or hardly any of it, a step or two of keys; and with the hint, the other way."""
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 128, 200, 129, 31] * 4
    new = [2, 1, 3, 1, 16, 5, 1, 2, 33, 1, 64, 4, 0] * 4
    b = P.Batch(26, lens, new, 2, dim, 16, "int8", extra_rows=3).fill(lens)
    Q = b.rand(b.rows, 2 * group, dim, dtype=torch.float16)
    for hint in (0, max(new)):
        check_attention(TF, b, Q, dim ** -0.5, max_new=hint)


@pytest.mark.parametrize("dim,new", [(128, 8), (128, 9), (64, 16), (64, 17), (96, 8), (80, 9)])
def test_attention_where_the_ways_part(TF, dim, new):
    """Four rows for each new token: the last number that goes the way of few rows, the first that goes the prompts' way."""
    lens = [500, 40, new]
    b = P.Batch(27, lens, [new] * 3, 1, dim, 64, "e4m3").fill(lens)
    check_attention(TF, b, b.rand(b.rows, 4, dim, dtype=torch.bfloat16), dim ** -0.5, max_new=new)


def test_attention_many_sequences(TF):
    """More sequences than a block has threads, of very different lengths, some empty."""
    lens = [(37 * i) % 211 for i in range(700)]
    lens[333] = 9000
    new = [1 if i % 5 else 0 for i in range(700)]
    b = P.Batch(14, lens, new, 1, 64, 64, "int8", extra_cols=0).fill(lens)
    check_attention(TF, b, b.rand(b.rows, 2, 64, dtype=torch.bfloat16), 0.125, max_new=1)


def test_attention_same_bits_every_time(TF):
    lens, new = [5000, 700, 1], [1, 300, 1]
    b = P.Batch(15, lens, new, 2, 128, 64, "e4m3").fill(lens)
    Q = b.rand(b.rows, 8, 128, dtype=torch.bfloat16)
    outs = []
    for _ in range(4):
        out = torch.empty_like(Q)
        TF.kvcache_attention(Q, *b.cache(), *b.seqs(), 0.09, 300, 0, out)
        outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


def test_long_cache_offsets_beyond_32_bits(TF):
    """Pages at byte offsets above 2^32: written, read back and attended."""
    heads, dim, page = 8, 128, 256
    pages = (5 << 30) // (heads * dim * page)
    lens, new = [700, 300], [700, 1]
    b = P.Batch(16, lens, new, heads, dim, page, "int8", extra_cols=0)
    b.pages = pages
    b.host_table = torch.tensor([[pages - 1, pages - 2, 3], [pages - 3, pages - 5, 0]])
    b.table = b.host_table.int().cuda()
    b.k, b.v = (torch.zeros(pages, heads, page, dim, dtype=torch.int8, device="cuda") for _ in "kv")
    b.ks, b.vs = (torch.ones(pages, heads, device="cuda") for _ in "kv")
    b.fill(lens)
    K, V = b.rand(b.rows, heads, dim, dtype=torch.bfloat16), b.rand(b.rows, heads, dim, dtype=torch.bfloat16)
    TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
    RK, RV = torch.empty_like(K), torch.empty_like(V)
    TF.kvcache_read(*b.cache(), *b.seqs(), RK, RV, b.flag)
    assert float((RK.float() - K.float()).abs().max()) < 0.05 and float((RV.float() - V.float()).abs().max()) < 0.05
    check_attention(TF, b, b.rand(b.rows, 16, dim, dtype=torch.bfloat16), dim ** -0.5, max_new=700)


# ---- bad tables, lengths and starts ----------------------------------------------------------------------------
@pytest.mark.parametrize("new", [1, 140])
def test_bad_pages_are_masked_and_flagged(TF, new):
    lens = [200, 150]
    b = P.Batch(17, lens, [new, new], 2, 64, 16, "int8").fill(lens)
    Q = b.rand(b.rows, 4, 64, dtype=torch.bfloat16)
    bad = b.table.clone()
    for i, (s, c) in enumerate(((0, 2), (1, 0), (1, 8))):
        bad[s, c] = (-1, b.pages, 2**31 - 1)[i]
    out = torch.empty_like(Q)
    TF.kvcache_attention(Q, *b.cache(), b.starts, b.length, bad, 0.125, new, 0, out, b.flag)
    assert int(b.flag) == 1 and torch.isfinite(out).all()
    # the sequence whose masked page lies in front of every row's window is untouched by it
    clean = torch.empty_like(Q)
    TF.kvcache_attention(Q, *b.cache(), b.starts, b.length, b.table, 0.125, new, 0, clean)
    assert not torch.equal(out, clean)
    # written tokens of a bad page are dropped, its reads are zero
    before = b.k.clone()
    K = b.rand(b.rows, 2, 64)
    all_bad = torch.full_like(b.table, b.pages)
    TF.kvcache_write(K, K, b.starts, b.length, all_bad, *b.cache(), b.flag)
    assert torch.equal(before, b.k)
    R, S = torch.ones_like(K), torch.ones_like(K)
    TF.kvcache_read(*b.cache(), b.starts, b.length, all_bad, R, S, b.flag)
    assert not R.any() and not S.any()
    TF.kvcache_attention(Q, *b.cache(), b.starts, b.length, all_bad, 0.125, new, 0, out, b.flag)
    assert not out.any()


@pytest.mark.parametrize("new", [1, 140])
def test_bad_starts_and_lengths_are_flagged(TF, new):
    lens = [200, 150]
    b = P.Batch(18, lens, [new, new], 1, 64, 16, "int8").fill(lens)
    Q, K = b.rand(b.rows, 4, 64, dtype=torch.bfloat16), b.rand(b.rows, 1, 64)
    big = 2**31 - 1
    for starts, length in (([0, new, big], lens), ([-5, new, 2 * new], lens), ([new, 0, 2 * new], lens), ([0, new, 2 * new], [big, 150]),
                           ([0, new, 2 * new], [200, -7]), ([-big, big, big], [big, big]), ([big, -big, 0], [0, 0])):
        s, n = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (starts, length))
        for call in (lambda f: TF.kvcache_attention(Q, *b.cache(), s, n, b.table.clamp(max=b.pages - 1), 0.125, new, 0, torch.empty_like(Q), f),
                     lambda f: TF.kvcache_read(*b.cache(), s, n, b.table.clamp(max=b.pages - 1), K.clone(), K.clone(), f),
                     lambda f: TF.kvcache_write(K, K, s, n, b.table.clamp(max=b.pages - 1), *b.cache(), f)):
            flag = torch.zeros(1, dtype=torch.int32, device="cuda")
            call(flag)
            assert int(flag) & 2, (starts, length)


def test_empty_calls(TF):
    b = P.Batch(19, [0, 0], [0, 0], 1, 64, 16, "int8")
    Q, K = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(0, 1, 64, device="cuda")
    TF.kvcache_attention(Q, *b.cache(), *b.seqs(), 0.125, 0, 0, torch.empty_like(Q))
    TF.kvcache_write(K, K, *b.seqs(), *b.cache())
    TF.kvcache_read(*b.cache(), *b.seqs(), K, K.clone())


# ---- streams and graphs ----------------------------------------------------------------------------------------
def test_captured_step_replays_with_other_lengths(TF):
    """A decode step (write, attention) captured once and replayed as the sequences grow; two such graphs and eager calls of the
    same operators in between, each with scratch of its own."""
    heads, dim, page, steps = 2, 64, 16, 40
    graphs = []
    for seed in (20, 21):
        lens = [3000, 1, 15]
        b = P.Batch(seed, lens, [1, 1, 1], heads, dim, page, "int8", extra_cols=steps // page + 2).fill(lens)
        b.table = b.host_table.int().cuda()
        K, V = b.rand(3, heads, dim), b.rand(3, heads, dim)
        Q, Out = b.rand(3, 8, dim, dtype=torch.bfloat16), torch.empty(3, 8, dim, dtype=torch.bfloat16, device="cuda")

        def step(b=b, K=K, V=V, Q=Q, Out=Out):
            TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
            TF.kvcache_attention(Q, *b.cache(), *b.seqs(), 0.125, 1, 0, Out, b.flag)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, b, K, V, Q, Out, torch.cuda.Stream()))
    for t in range(steps):
        torch.cuda.synchronize()
        for graph, b, K, V, Q, Out, _ in graphs:
            b.lens = [n + 1 for n in b.lens]
            b.length += 1
            K.copy_(b.rand(3, heads, dim))
            V.copy_(b.rand(3, heads, dim))
            Q.copy_(b.rand(3, 8, dim, dtype=torch.bfloat16))
        torch.cuda.synchronize()
        for graph, *_, stream in graphs:  # both at once
            with torch.cuda.stream(stream):
                graph.replay()
        eager = torch.empty_like(graphs[0][5])
        torch.cuda.synchronize()
        for graph, b, K, V, Q, Out, _ in graphs:
            if t % 13 == 0:
                want, bound = P.attention(b, Q, 0.125)
                off = (Out.double() - want).abs()
                assert bool((off <= bound + P.half_step(Q.dtype) * (want.abs() + bound)).all())
            TF.kvcache_attention(Q, *b.cache(), *b.seqs(), 0.125, 1, 0, eager, b.flag)
            assert torch.equal(eager, Out) and int(b.flag) == 0


def test_calls_on_two_streams_at_once(TF):
    batches = []
    for seed in (22, 23):
        lens, new = [4000, 900, 33], [1, 1, 1]
        b = P.Batch(seed, lens, new, 2, 128, 64, "e4m3").fill(lens)
        Q = b.rand(3, 8, 128, dtype=torch.bfloat16)
        want = torch.empty_like(Q)
        TF.kvcache_attention(Q, *b.cache(), *b.seqs(), 0.09, 1, 0, want)
        batches.append((b, Q, want, torch.empty_like(Q), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(30):
        for b, Q, want, out, st in batches:
            with torch.cuda.stream(st):
                TF.kvcache_attention(Q, *b.cache(), *b.seqs(), 0.09, 1, 0, out)
    torch.cuda.synchronize()
    for b, Q, want, out, st in batches:
        assert torch.equal(out, want)


# ---- the operators together ------------------------------------------------------------------------------------
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_layer_attention_prompt_then_tokens(TF, fmt):
    """What serving does: a prompt in two chunks and then tokens one by one, queries and keys normed and rotated in place, written
    to the cache, attended.  Each step's attention is held to the cache as it stands; the cache at the end to the keys and values
    in 64 bits.  That bound: a code is off by half a step of its page's scale when written and half a step of the new scale each
    time it has grown (twofold at least): s/2 + s/4 + ... < s, and s <= 2 * largest / 127; e4m3 half a step is 2^-4 of the value, and
    2^-10 s below the smallest normal code, s <= 2 * largest / 448; the rotation's own bfloat16 rounding comes on top."""
    torch.manual_seed(1)
    q_heads, heads, dim, page, total = 8, 2, 64, 16, 150
    dev = "cuda"
    b = P.Batch(24, [total], [1], heads, dim, page, fmt)
    b.table = b.host_table.int().to(dev)
    inv = (10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).float().to(dev)
    qw, kw = (1 + 0.1 * torch.randn(dim)).bfloat16().to(dev), (1 + 0.1 * torch.randn(dim)).bfloat16().to(dev)
    QKV = torch.randn(total, q_heads + 2 * heads, dim).bfloat16().to(dev)
    positions = torch.arange(total, device=dev, dtype=torch.int32)
    t = 0
    for n in (64, 30) + (1,) * (total - 94):
        x = QKV[t: t + n].clone()
        Q, K, V = x[:, :q_heads], x[:, q_heads: q_heads + heads], x[:, q_heads + heads:]
        TF.qknorm_rope(Q, K, qw, kw, inv, positions[t: t + n], 1e-6, False, Q, K)
        t += n
        b.lens, b.new, b.host_starts = [t], [n], [0, n]
        b.starts = torch.tensor([0, n], dtype=torch.int32, device=dev)
        b.length = torch.tensor([t], dtype=torch.int32, device=dev)
        TF.kvcache_write(K, V, *b.seqs(), *b.cache(), b.flag)
        check_attention(TF, b, Q, dim ** -0.5, max_new=n)
    k, _ = P.rope(QKV[:, q_heads: q_heads + heads], kw, inv, positions, 1e-6, False)
    v = QKV[:, q_heads + heads:].double()
    for want, codes, scales in ((k, b.k, b.ks), (v, b.v, b.vs)):
        largest = float(want.abs().max())
        off = (b.history(codes, scales, 0) - want).abs()
        own = 2 * largest / 127 if fmt == "int8" else want.abs() * 2.0**-4 + 2.0**-10 * 2 * largest / 448
        assert bool((off <= own + want.abs() * 2.0**-7).all())
