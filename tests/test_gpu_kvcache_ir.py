"""The cache operators as deepxIR ops: an executor runs a layer's attention line by line and as a compiled program, with the
results of the direct calls; what does not fit is an error reply."""
import numpy as np
import pytest
import torch

import kvcache_plain as P
from helpers import to_np

pytestmark = pytest.mark.gpu
PAGE, HEADS, Q_HEADS, DIM, BATCH, COLS = 16, 2, 8, 64, 3, 8


@pytest.fixture()
def ex():
    from deepx_b200.executor import Executor
    e = Executor(0)
    yield e
    e.close()


def t(dtype, name):
    return f"tensor<{dtype}>:{name}"


CACHE = ", ".join([t("int8", "kc"), t("int8", "vc"), t("float32", "ks"), t("float32", "vs")])
SEQS = ", ".join([t("int32", "starts"), t("int32", "lens"), t("int32", "table")])


def layer(fmt, max_new, dtype="bfloat16"):
    return [
        f"qknorm_rope({t(dtype, 'q')}, {t(dtype, 'k')}, {t(dtype, 'qw')}, {t(dtype, 'kw')}, {t('float32', 'inv')}, {t('int32', 'pos')}, var<float32>:1e-6, "
        f"var<bool>:false)->({t(dtype, 'q')}, {t(dtype, 'k')})",
        f"kvcache_write({t(dtype, 'k')}, {t(dtype, 'v')}, {SEQS}, var<string>:{fmt})->({CACHE})",
        f"kvcache_attention({t(dtype, 'q')}, {CACHE}, {SEQS}, var<float32>:0.125, var<int32>:{max_new}, var<int32>:0, var<string>:{fmt})->({t(dtype, 'out')})",
        f"kvcache_read({CACHE}, {SEQS}, var<string>:{fmt})->({t(dtype, 'rk')}, {t(dtype, 'rv')})",
    ]


def inputs(rows, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16()  # noqa: E731
    return {"q": r(rows, Q_HEADS, DIM), "k": r(rows, HEADS, DIM), "v": r(rows, HEADS, DIM), "qw": 1 + 0.1 * r(DIM), "kw": 1 + 0.1 * r(DIM),
            "inv": (10000.0 ** (-torch.arange(0, DIM, 2, dtype=torch.float64) / DIM)).float()}


def seqs(lens, new):
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, new)]).astype(np.int32)
    return starts, np.asarray(lens, np.int32), pos


def put(ex, name, x):
    a = to_np(x) if isinstance(x, torch.Tensor) else x
    if ex.ptr(name):
        ex.upload(name, a)
    else:
        ex.put(name, a)


def make(ex, lens, new, seed=0):
    starts, n, pos = seqs(lens, new)
    for name, x in {**inputs(int(starts[-1]), seed), "starts": starts, "lens": n, "pos": pos}.items():
        put(ex, name, x)
    table = np.random.default_rng(1).permutation(BATCH * COLS).reshape(BATCH, COLS).astype(np.int32)
    put(ex, "table", table)
    for name in ("kc", "vc"):
        ex.put(name, np.zeros((BATCH * COLS, HEADS, PAGE, DIM), np.int8))
    for name in ("ks", "vs"):
        ex.put(name, np.zeros((BATCH * COLS, HEADS), np.float32))
    rows = int(starts[-1])
    ex.new("out", "bfloat16", (rows, Q_HEADS, DIM))
    ex.new("rk", "bfloat16", (rows, HEADS, DIM))
    ex.new("rv", "bfloat16", (rows, HEADS, DIM))
    return table


def direct(fmt, table, lens, new, x, cache):
    """The same through the Python functions; `cache` is changed in place."""
    from deepx_b200 import tensorfunc as TF
    starts, n, pos = (torch.from_numpy(a).cuda() for a in seqs(lens, new))
    x = {k: v.cuda() for k, v in x.items()}
    TF.qknorm_rope(x["q"], x["k"], x["qw"], x["kw"], x["inv"], pos, 1e-6, False, x["q"], x["k"])
    tab = torch.from_numpy(table).cuda()
    TF.kvcache_write(x["k"], x["v"], starts, n, tab, *cache)
    out, rk, rv = torch.empty_like(x["q"]), torch.empty_like(x["k"]), torch.empty_like(x["v"])
    TF.kvcache_attention(x["q"], *cache, starts, n, tab, 0.125, max(new), 0, out)
    TF.kvcache_read(*cache, starts, n, tab, rk, rv)
    return {"out": out, "rk": rk, "rv": rv}


def fresh_cache(fmt):
    shape = (BATCH * COLS, HEADS, PAGE, DIM)
    return [torch.zeros(shape, dtype=torch.int8, device="cuda").view(P.FORMATS[fmt]) for _ in "kv"] + [torch.zeros(shape[:2], device="cuda") for _ in "kv"]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("lens,new", [([70, 3, 40], [70, 3, 40]), ([1, 1, 1], [1, 1, 1])])
def test_lines_give_what_the_calls_give(ex, fmt, lens, new):
    table = make(ex, lens, new)
    for line in layer(fmt, max(new)):
        ex.run(line)
    want = direct(fmt, table, lens, new, inputs(sum(new), 0), fresh_cache(fmt))
    for name, w in want.items():
        assert np.array_equal(np.asarray(ex.download(name)).view(np.uint16), to_np(w).view(np.uint16)), name


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_compiled_step_replays_as_sequences_grow(ex, fmt):
    """A decode step as one compiled program, replayed with new inputs and lengths in the same tensors."""
    lens, new = [40, 1, 17], [1, 1, 1]
    cache = fresh_cache(fmt)
    table = make(ex, lens, new)
    prog = ex.compile("\n".join(layer(fmt, 1)))  # runs once
    direct(fmt, table, lens, new, inputs(3, 0), cache)
    for step in range(1, 30):
        lens = [n + 1 for n in lens]
        starts, n, pos = seqs(lens, new)
        x = inputs(3, step)
        for name in ("q", "k", "v"):
            put(ex, name, x[name])
        put(ex, "lens", n)
        put(ex, "pos", pos)
        prog.run()
        ex.sync()
        x["qw"], x["kw"] = inputs(3, 0)["qw"], inputs(3, 0)["kw"]
        want = direct(fmt, table, lens, new, x, cache)
        for name, w in want.items():
            assert np.array_equal(np.asarray(ex.download(name)).view(np.uint16), to_np(w).view(np.uint16)), (step, name)


def test_what_does_not_fit_is_an_error_reply(ex):
    make(ex, [5, 5, 5], [1, 1, 1])
    good = layer("int8", 1)
    for bad, text in ((good[1].replace("string>:int8", "string>:int4"), "format"), (good[2].replace("float32>:0.125", "float32>:-1"), "scale"),
                      (good[1].replace(t("int32", "lens"), t("int32", "starts")), "starts is"), (good[2].replace(t("bfloat16", "out"), t("bfloat16", "rk")), "queries"),
                      (good[3].replace(t("float32", "ks"), t("float32", "inv")), "scales"), (good[0].replace(t("int32", "pos"), t("int32", "table")), "positions"),
                      (good[1].replace(t("bfloat16", "k") + ",", t("bfloat16", "q") + ","), "keys and values")):
        status, reply = ex.reply(bad)
        assert status != 0 and text in reply, (bad, reply)
    for line in good:
        ex.run(line)
