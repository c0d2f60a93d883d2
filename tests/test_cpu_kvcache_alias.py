"""Memory that a call of the cache operators or of qknorm_rope would write and that another of its arguments uses too: refused on the host.
Addresses are made up; every call below is refused before anything follows one."""
import pytest

from deepx_b200 import _native as N

A = 1 << 44  # one place for each argument, far from the others
PLACES = ["k", "v", "kc", "vc", "ks", "vs", "starts", "lens", "table", "flag", "q", "out", "ws", "qo", "ko", "qw", "kw", "inv", "pos"]
ROWS, HEADS, DIM, PAGES, PAGE, BATCH, COLS = 5, 2, 64, 4, 16, 2, 3
STRIDE = HEADS * DIM


def places(**moved):
    at = {name: A * (i + 1) for i, name in enumerate(PLACES)}
    at.update(moved)
    return at


def descriptors(at):
    return (N.KvSeqs(at["starts"], at["lens"], at["table"], BATCH, COLS, ROWS),
            N.KvCache(at["kc"], at["vc"], at["ks"], at["vs"], PAGES, HEADS, PAGE, DIM, N.CACHE_I8))


def write(at, stride=STRIDE):
    s, c = descriptors(at)
    return N.lib.dx_kvcache_write(N.F32, at["k"], stride, at["v"], stride, s, c, at["flag"], None)


def read(at, stride=STRIDE, v_stride=None):
    s, c = descriptors(at)
    return N.lib.dx_kvcache_read(N.F32, s, c, at["k"], stride, at["v"], v_stride or stride, at["flag"], None)


def attend(at, ws_bytes=0, q_stride=4 * DIM, out_stride=4 * DIM):
    s, c = descriptors(at)
    return N.lib.dx_kvcache_attention(N.BF16, at["q"], q_stride, 4, s, c, 0.125, 0, 0, at["out"], out_stride, at["ws"], ws_bytes, at["flag"], None)


def rope(at, q_stride=4 * DIM, k_stride=2 * DIM):
    return N.lib.dx_qknorm_rope(N.F32, at["q"], q_stride, 4, at["k"], k_stride, 2, ROWS, DIM, 1, at["qw"], at["kw"], 1e-6, at["inv"], DIM, 0, N.I32,
                                at["pos"], at["qo"], q_stride, at["ko"], k_stride, None)


CODES = PAGES * HEADS * PAGE * DIM
SCALES, ROW_BYTES = PAGES * HEADS * 4, ((ROWS - 1) * STRIDE + STRIDE) * 4


@pytest.mark.parametrize("a,b,size", [("kc", "vc", CODES), ("ks", "vs", SCALES), ("kc", "ks", CODES), ("vc", "ks", CODES), ("kc", "vs", CODES), ("kc", "k", CODES),
                                      ("vc", "v", CODES), ("k", "ks", ROW_BYTES), ("v", "vs", ROW_BYTES), ("kc", "starts", CODES), ("vc", "lens", CODES), ("kc", "table", CODES),
                                      ("starts", "ks", 4 * (BATCH + 1)), ("lens", "vs", 4 * BATCH), ("table", "ks", 4 * BATCH * COLS), ("kc", "flag", CODES), ("vs", "flag", SCALES),
                                      ("k", "flag", ROW_BYTES), ("lens", "flag", 4 * BATCH)])
def test_write(a, b, size):
    for offset in (0, size // 32 * 16, (size - 1) // 16 * 16):  # the start, the middle, the last sixteen bytes
        assert write(places(**{b: places()[a] + offset})) == N.E_ALIAS, offset


@pytest.mark.parametrize("a,b,size", [("k", "v", ROW_BYTES), ("v", "k", ROW_BYTES), ("kc", "k", CODES), ("vc", "v", CODES), ("k", "ks", ROW_BYTES), ("v", "vs", ROW_BYTES),
                                      ("k", "starts", ROW_BYTES), ("v", "lens", ROW_BYTES), ("k", "table", ROW_BYTES), ("v", "flag", ROW_BYTES), ("kc", "flag", CODES), ("table", "flag", 4 * BATCH * COLS)])
def test_read(a, b, size):
    for offset in (0, size // 32 * 16, (size - 1) // 16 * 16):
        assert read(places(**{b: places()[a] + offset})) == N.E_ALIAS, offset


def test_read_into_columns_of_one_buffer():
    """K and V beside one another in the rows of a buffer are fine (the GPU tests call that); a column in common, or rows of two strides
    among one another, are not."""
    k = places()["k"]
    assert read(places(v=k + (STRIDE - 1) * 4), 2 * STRIDE) == N.E_ALIAS
    assert read(places(v=k + (STRIDE + 1) * 4), 2 * STRIDE) == N.E_ALIAS
    assert read(places(v=k + STRIDE * 4), 2 * STRIDE, 2 * STRIDE + 1) == N.E_ALIAS
    # starts between two rows would be fine; over a row's end it is not
    assert read(places(starts=k + (2 * STRIDE + STRIDE - 1) * 4), 2 * STRIDE) == N.E_ALIAS


OUT_BYTES = ROWS * 4 * DIM * 2


@pytest.mark.parametrize("a,b,size", [("out", "q", OUT_BYTES), ("q", "out", OUT_BYTES), ("kc", "out", CODES), ("out", "vc", OUT_BYTES), ("out", "ks", OUT_BYTES), ("out", "vs", OUT_BYTES),
                                      ("out", "starts", OUT_BYTES), ("out", "lens", OUT_BYTES), ("out", "table", OUT_BYTES), ("out", "flag", OUT_BYTES), ("q", "flag", OUT_BYTES),
                                      ("starts", "flag", 4 * (BATCH + 1))])
def test_attention(a, b, size):
    assert attend(places()) == N.E_WORKSPACE  # what is asked next: nothing overlaps
    for offset in (0, size // 32 * 16, (size - 1) // 16 * 16):
        assert attend(places(**{b: places()[a] + offset})) == N.E_ALIAS, offset


def test_attention_workspace():
    s, c = descriptors(places())
    need = N.lib.dx_kvcache_attention_workspace_bytes(N.BF16, 4, s, c, 0)
    ws = places()["ws"]
    for name in ("q", "out", "kc", "vc", "ks", "vs", "starts", "lens", "table", "flag"):
        for offset in (0, need // 512 * 256, (need - 1) // 256 * 256):
            assert attend(places(**{name: ws + offset}), need) == N.E_ALIAS, (name, offset)


@pytest.mark.parametrize("a,b,size", [("qo", "ko", ROWS * 4 * DIM * 4), ("ko", "qo", ROWS * 2 * DIM * 4), ("qo", "k", ROWS * 4 * DIM * 4), ("ko", "q", ROWS * 2 * DIM * 4),
                                      ("qo", "qw", ROWS * 4 * DIM * 4), ("ko", "qw", ROWS * 2 * DIM * 4), ("qo", "kw", ROWS * 4 * DIM * 4), ("qo", "inv", ROWS * 4 * DIM * 4),
                                      ("ko", "pos", ROWS * 2 * DIM * 4)])
def test_rope(a, b, size):
    for offset in (0, size // 32 * 16, (size - 1) // 16 * 16):
        assert rope(places(**{b: places()[a] + offset})) == N.E_ALIAS, offset


def test_rope_columns():
    """In place in a packed projection, but for one column that both outputs have."""
    q = places()["q"]
    assert rope(places(qo=q, k=q + 4 * DIM * 4, ko=q + (4 * DIM - 1) * 4), 8 * DIM, 8 * DIM) == N.E_ALIAS
    assert rope(places(ko=places()["qo"] + 4 * DIM * 4 - 4), 8 * DIM, 8 * DIM) == N.E_ALIAS
    assert rope(places(qo=q, qw=q + 8 * DIM * 4), 8 * DIM, 2 * DIM) == N.E_ALIAS  # a weight in the second row
