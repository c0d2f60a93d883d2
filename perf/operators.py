"""Cases and plain forms of the operators around the 8-bit key/value cache: qknorm_rope, kvcache_write, kvcache_read and
kvcache_attention.

``own`` false: ``run`` computes an operator with elementary torch operations in 32 bits (rotation angles in 64);
``own`` true: it makes the call a user makes of ``deepx_b200.tensorfunc``.  Both take the state of ``prepare``: the inputs,
the pages of the cache and the output buffers.

The cache holds pages of ``page`` tokens, ``[pages, kv_heads, page, head_dim]`` codes of 8 bits and one float32 scale for each
page and head.  New tokens are packed rows; ``starts`` says where each sequence's rows begin, ``lens`` how many tokens it
holds with them, ``table`` which pages they are in.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
LARGEST = {"int8": 127.0, "e4m3": 448.0}


# ---- cases -----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user, one new token, a short conversation: the smallest call, all latency
        attention("attention: 1 x 1 token of 1500", 1, 1, 1, 1500, 1500, 32, 8, 128, 64, "bf16", "int8"),
        # a batch of users in decode, histories of every length
        attention("attention: 64 x 1 token of 300-8192", 64, 1, 1, 300, 8192, 32, 8, 128, 64, "bf16", "e4m3"),
        # one user with a very long document: few rows, the work has to be split along the cache
        attention("attention: 1 x 1 token of 262100", 1, 1, 1, 262100, 262100, 32, 8, 128, 128, "f16", "int8"),
        # the prompt of two new users at once: bound by the tensor cores and the exponentials
        attention("attention: 2 x 4096 tokens, prompt", 2, 4096, 4096, 4096, 4096, 32, 8, 128, 64, "bf16", "int8"),
        # prompts continued and decoded in one batch, a small model of 14 heads (seven share a key head) and small pages
        attention("attention: 12 x 1-700 tokens of 5000", 12, 1, 700, 700, 5000, 14, 2, 64, 16, "bf16", "e4m3"),
        # queries and keys of a decode batch: the smallest call
        rope("qknorm_rope: 64 tokens", 64, 32, 8, 128, 128, False, True, "bf16"),
        # a prompt of 16384 tokens
        rope("qknorm_rope: 16384 tokens", 16384, 32, 8, 128, 128, False, True, "bf16"),
        # an odd number of tokens in float32, pairs side by side, half of the head rotated, no norm
        rope("qknorm_rope: 4099 tokens f32", 4099, 14, 2, 64, 32, True, False, "f32"),
        # the keys and values of a decode batch
        write("kvcache_write: 64 x 1 token", 64, 1, 1, 100, 2000, 8, 128, 64, "bf16", "int8"),
        # the keys and values of four prompts
        write("kvcache_write: 4 x 5000-8192 tokens", 4, 5000, 8192, 8192, 10000, 8, 128, 64, "bf16", "e4m3"),
        # a short history read back
        read("kvcache_read: 1 x 700 tokens", 1, 700, 700, 700, 700, 8, 128, 16, "bf16", "int8"),
        # long histories read back, small heads
        read("kvcache_read: 8 x 3000-9000 tokens", 8, 3000, 9000, 9000, 9000, 8, 64, 128, "f16", "e4m3"),
    ]


def attention(name, batch, new_lo, new_hi, len_lo, len_hi, q_heads, kv_heads, dim, page, dtype, code, window=0):
    return {"name": name, "op": "attention", "batch": batch, "new_lo": new_lo, "new_hi": new_hi, "len_lo": len_lo, "len_hi": len_hi,
            "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "code": code, "window": window}


def rope(name, tokens, q_heads, kv_heads, dim, rotated, interleaved, norm, dtype):
    return {"name": name, "op": "rope", "tokens": tokens, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "rotated": rotated,
            "interleaved": interleaved, "norm": norm, "dtype": dtype}


def write(name, batch, new_lo, new_hi, len_lo, len_hi, kv_heads, dim, page, dtype, code):
    return {"name": name, "op": "write", "batch": batch, "new_lo": new_lo, "new_hi": new_hi, "len_lo": len_lo, "len_hi": len_hi,
            "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype, "code": code}


def read(name, batch, new_lo, new_hi, len_lo, len_hi, kv_heads, dim, page, dtype, code):
    return dict(write(name, batch, new_lo, new_hi, len_lo, len_hi, kv_heads, dim, page, dtype, code), op="read")


def log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49))))))


def draw(rng):
    kind = rng.choice(["decode", "decode", "prompt", "mixed", "rope", "write", "read"])
    dtype, code = rng.choice(["bf16", "f16"]), rng.choice(["int8", "e4m3"])
    page, dim = rng.choice([16, 32, 64, 128]), rng.choice([64, 96, 128])
    q_heads, kv_heads = rng.choice([(32, 8), (14, 2), (16, 16), (8, 1), (24, 8)])
    if kind == "rope":
        tokens = log_int(rng, 1, 16384)
        rotated = rng.choice([dim, dim // 2])
        c = rope("", tokens, q_heads, kv_heads, dim, rotated, rng.random() < 0.3, rng.random() < 0.8, rng.choice(["bf16", "f16", "f32"]))
    elif kind in ("write", "read"):
        batch = log_int(rng, 1, 64)
        new_hi = log_int(rng, 1, max(1, 32768 // batch))
        new_lo = rng.randint(1, new_hi)
        len_hi = new_hi + log_int(rng, 1, 3000)
        c = (write if kind == "write" else read)("", batch, new_lo, new_hi, new_hi, len_hi, kv_heads, dim, page, rng.choice(["bf16", "f16", "f32"]), code)
    elif kind == "decode":
        batch = log_int(rng, 1, 64)
        most = int(2.5e8 / (batch * kv_heads * dim))
        len_hi = log_int(rng, 16, min(262144, most))
        window = log_int(rng, 100, 4000) if rng.random() < 0.2 else 0
        c = attention("", batch, 1, rng.choice([1, 1, 2, 4]), rng.randint(4, len_hi), len_hi, q_heads, kv_heads, dim, page, dtype, code, window)
    elif kind == "prompt":
        batch = rng.choice([1, 2])
        new = log_int(rng, 100, 4000 if batch == 1 else 2500)
        len_hi = new + rng.choice([0, 0, rng.randint(1, 1500)])
        c = attention("", batch, rng.randint(new // 2, new), new, len_hi, len_hi, q_heads, kv_heads, dim, page, dtype, code)
    else:
        batch = rng.randint(2, 12)
        new_hi = log_int(rng, 20, 700)
        c = attention("", batch, 1, new_hi, new_hi, new_hi + log_int(rng, 100, 4000), q_heads, kv_heads, dim, page, dtype, code)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------------------------------
def sizes(case):
    """(lens, new tokens) of each sequence: the same for every seed, so that the work is."""
    g = torch.Generator().manual_seed(1)
    b = case["batch"]
    new = torch.randint(case["new_lo"], case["new_hi"] + 1, (b,), generator=g)
    # lengths spread evenly over their logarithm, the longest among them
    u = torch.rand(b, generator=g, dtype=torch.float64)
    u[0] = 1.0
    lens = (case["len_lo"] * (case["len_hi"] / case["len_lo"]) ** u).round().long().clamp(max=case["len_hi"])
    return torch.maximum(lens, new).tolist(), new.tolist()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = {"case": case}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    d = case["dim"]
    if case["op"] == "rope":
        t = case["tokens"]
        channel = torch.exp(0.5 * randn(d))  # some channels are larger than others
        s["q"], s["k"] = (randn(t, case["q_heads"], d) * channel).to(dtype), (randn(t, case["kv_heads"], d) * channel).to(dtype)
        s["q_weight"], s["k_weight"] = (1 + 0.2 * randn(d)).to(dtype), (1 + 0.2 * randn(d)).to(dtype)
        s["inv_freq"] = 500000.0 ** (-torch.arange(0, case["rotated"], 2, device=dev, dtype=torch.float64) / case["rotated"])
        s["inv_freq"] = s["inv_freq"].float()
        s["positions"] = torch.randint(0, 131072, (t,), generator=g, device=dev).int()
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        return s

    lens, new = sizes(case)
    h, page, b = case["kv_heads"], case["page"], case["batch"]
    cols = -(-max(lens) // page)
    pages = b * cols + 3
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    total = starts[-1]
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    s["table"] = torch.randperm(pages, generator=g, device=dev)[: b * cols].reshape(b, cols).int()
    s["max_len"], s["max_new"], s["total"] = max(lens), max(new), total
    codes = CODES[case["code"]]
    for x in ("k", "v"):
        if case["code"] == "int8":
            s[x + "_cache"] = torch.randint(-127, 128, (pages, h, page, d), generator=g, device=dev, dtype=torch.int8)
        else:  # every finite value of the format
            bits = torch.randint(0, 254, (pages, h, page, d), generator=g, device=dev, dtype=torch.uint8)
            s[x + "_cache"] = torch.where(bits >= 127, bits + 1, bits).view(codes)
        # scales of earlier tokens: values of about one in size
        e = torch.randint(0, 2, (pages, h), generator=g, device=dev)
        s[x + "_scale"] = torch.ldexp(torch.ones(pages, h, device=dev), e - (6 if case["code"] == "int8" else 7))
    if case["op"] == "attention":
        q = case["q_heads"]
        s["scale"] = d ** -0.5
        s["q"] = randn(total, q, d).to(dtype)
        s["out"] = torch.empty(total, q, d, device=dev, dtype=dtype)
    elif case["op"] == "write":
        channel = torch.exp(0.5 * randn(h, d))
        s["k"], s["v"] = (randn(total, h, d) * channel).to(dtype), randn(total, h, d).to(dtype)
    else:
        s["k"], s["v"] = (torch.empty(total, h, d, device=dev, dtype=dtype) for _ in "kv")
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        return {"rope": own_rope, "write": own_write, "read": own_read, "attention": own_attention}[op](s, case)
    return {"rope": plain_rope, "write": plain_write, "read": plain_read, "attention": plain_attention}[op](s, case)


def own_rope(s, case):
    from deepx_b200 import tensorfunc as TF

    norm = (s["q_weight"], s["k_weight"], 1e-6) if case["norm"] else (None, None, None)
    TF.qknorm_rope(s["q"], s["k"], norm[0], norm[1], s["inv_freq"], s["positions"], norm[2], case["interleaved"], s["q_out"], s["k_out"])
    return s["q_out"], s["k_out"]


def own_write(s, case):
    from deepx_b200 import tensorfunc as TF

    cache = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    TF.kvcache_write(s["k"], s["v"], s["starts"], s["lens"], s["table"], *cache)
    return cache


def own_read(s, case):
    from deepx_b200 import tensorfunc as TF

    TF.kvcache_read(s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["starts"], s["lens"], s["table"], s["k"], s["v"])
    return s["k"], s["v"]


def own_attention(s, case):
    from deepx_b200 import tensorfunc as TF

    TF.kvcache_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["starts"], s["lens"], s["table"], s["scale"],
                         s["max_new"], case["window"], s["out"])
    return s["out"]


# ---- plain forms -----------------------------------------------------------------------------------------------------------
def plain_rope(s, case):
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float(), angle.sin().float()
    r = case["rotated"]

    def one(x, weight):
        y = x.float()
        if case["norm"]:
            y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * weight.float()
        if case["interleaved"]:
            a, b = y[..., 0:r:2], y[..., 1:r:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., : r // 2], y[..., r // 2 : r]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((turned, y[..., r:]), -1).to(x.dtype)

    return one(s["q"], s["q_weight"]), one(s["k"], s["k_weight"])


def rows(s, case):
    """Of each packed row: its sequence, its place among the sequence's new tokens, its position, page and slot."""
    row = torch.arange(s["total"], device=s["starts"].device)
    seq = torch.searchsorted(s["starts"][1:].long(), row, right=True)
    nth = row - s["starts"].long()[seq]
    position = nth + (s["lens"] - s["starts"][1:] + s["starts"][:-1]).long()[seq]
    return seq, nth, position, s["table"].long()[seq, position // case["page"]], position % case["page"]


def power_of_two(amax, code):
    """The least power of two, 2^-126 at least, in whose units amax is within the codes' range."""
    _, e = torch.frexp(amax / LARGEST[code])  # one too high at the border, and right above and below it
    e = e - (torch.ldexp(torch.ones_like(amax) * LARGEST[code], e - 1) >= amax).int()
    return torch.ldexp(torch.ones_like(amax), e.clamp(min=-126))


def rounded(x, code):
    return x.round().clamp(-127, 127).to(torch.int8) if code == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn)


def plain_write(s, case):
    code, page = case["code"], case["page"]
    seq, nth, position, where, slot = rows(s, case)
    first = (s["lens"] - s["starts"][1:] + s["starts"][:-1]).long()  # each sequence's first new position
    begun = s["table"].long()[torch.arange(case["batch"], device=first.device), first // page]  # the page it is in
    earlier = torch.arange(page, device=first.device)[None, :] < (first % page)[:, None]  # that page's earlier tokens
    for x in ("k", "v"):
        new, cache, scale = s[x].float(), s[x + "_cache"], s[x + "_scale"]
        amax = torch.zeros_like(scale).index_reduce_(0, where, new.abs().amax(-1), "amax")
        kept = torch.zeros_like(scale)
        kept[begun] = scale[begun] * earlier.any(-1, keepdim=True)
        grown = torch.maximum(power_of_two(amax, code), kept)
        old = cache[begun].float()
        again = rounded(old * (scale[begun] / grown[begun])[..., None, None], code)
        bits = cache.view(torch.uint8)
        bits[begun] = torch.where(earlier[:, None, :, None], again.view(torch.uint8), cache[begun].view(torch.uint8))
        bits[where, :, slot] = rounded(new / grown[where][..., None], code).view(torch.uint8)
        scale[where] = grown[where]
    return s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def plain_read(s, case):
    _, _, _, where, slot = rows(s, case)
    for x in ("k", "v"):
        s[x].copy_(s[x + "_cache"][where, :, slot].float() * s[x + "_scale"][where][..., None])
    return s["k"], s["v"]


def plain_attention(s, case):
    seq, nth, position, _, _ = rows(s, case)
    b, n, length, page, d = case["batch"], s["max_new"], s["max_len"], case["page"], case["dim"]
    kv, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    place = torch.arange(length, device=seq.device)
    where, slot = s["table"].long()[:, place // page], (place % page).expand(b, length)

    def history(x):  # [batch, kv head, token, dim]
        return (s[x + "_cache"][where, :, slot].float() * s[x + "_scale"][where][..., None]).transpose(1, 2)

    q = torch.zeros(b, n, kv, group, d, device=seq.device)
    q[seq, nth] = s["q"].float().view(-1, kv, group, d)
    at = (s["lens"] - s["starts"][1:] + s["starts"][:-1]).long()[:, None] + torch.arange(n, device=seq.device)  # [batch, new]
    seen = place <= at[..., None]
    if case["window"]:
        seen &= place > at[..., None] - case["window"]
    score = torch.matmul(q.permute(0, 2, 1, 3, 4).reshape(b, kv, n * group, d) * s["scale"], history("k").transpose(2, 3))
    score.view(b, kv, n, group, length).masked_fill_(~seen[:, None, :, None, :], -torch.inf)
    score -= score.amax(-1, keepdim=True)
    score.exp_()
    total = score.sum(-1, keepdim=True)
    o = torch.matmul(score, history("v")) / total
    o = o.view(b, kv, n, group, d).permute(0, 2, 1, 3, 4)[seq, nth]
    return o.reshape(-1, case["q_heads"], d).to(s["q"].dtype)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------
def work(case):
    d = case["dim"]
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    if case["op"] == "rope":
        values = case["tokens"] * (case["q_heads"] + case["kv_heads"]) * d
        return {"bytes": 2 * values * size + 4 * case["tokens"] + 2 * d * size + 2 * case["rotated"], "flops": 10 * values}
    lens, new = sizes(case)
    h, page = case["kv_heads"], case["page"]
    if case["op"] in ("write", "read"):
        values = 2 * sum(new) * h * d
        touched = sum((n - 1) // page - (n - m) // page + 1 for n, m in zip(lens, new))
        return {"bytes": values * (size + 1) + 8 * touched * h + 4 * touched + 8 * case["batch"], "flops": 2 * values}
    window = case["window"]
    keys = pairs = 0
    for n, m in zip(lens, new):
        first = n - m
        low = max(0, first - window + 1) if window else 0
        keys += n - low
        if window:
            full = max(0, n - max(first, window - 1))  # rows that see `window` keys
            short = m - full
            pairs += full * window + short * (2 * first + short + 1) // 2
        else:
            pairs += m * (2 * first + m + 1) // 2
    rows_ = sum(new) * case["q_heads"]
    return {"bytes": 2 * keys * h * d + 2 * rows_ * d * size + 8 * -(-keys // page) * h + 4 * -(-keys // page) + 8 * case["batch"],
            "flops": 4 * d * pairs * case["q_heads"]}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return exact_rope(s, case)
    lens, new = sizes(case)
    table, page = s["table"].tolist(), case["page"]
    if case["op"] == "write":
        for x in ("k", "v"):
            exact_write(s, case, x, lens, new, table)
        # int8 codes are whole numbers and have no nearer value
        codes = [None if case["code"] == "int8" else s[x].double() for x in ("k_cache", "v_cache")]
        return codes[0], codes[1], s["k_scale"].double(), s["v_scale"].double()

    def history(x, b, lo, hi):  # [token, kv head, dim] of the tokens lo..hi of sequence b
        at = torch.tensor(table[b][lo // page : (hi - 1) // page + 1], device="cuda", dtype=torch.long)
        whole = s[x + "_cache"][at].double() * s[x + "_scale"][at].double()[:, :, None, None]
        flat = whole.permute(0, 2, 1, 3).reshape(-1, case["kv_heads"], case["dim"])
        return flat[lo % page : lo % page + hi - lo]

    if case["op"] == "read":
        return tuple(torch.cat([history(x, b, lens[b] - new[b], lens[b]) for b in range(case["batch"])]) for x in ("k", "v"))
    out, row = [], 0
    group = case["q_heads"] // case["kv_heads"]
    for b, (n, m) in enumerate(zip(lens, new)):
        low = max(0, n - m - case["window"] + 1) if case["window"] else 0
        k, v = history("k", b, low, n), history("v", b, low, n)
        key = torch.arange(low, n, device="cuda")[None, :]
        at = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = key > at
        if case["window"]:
            hidden |= key <= at - case["window"]
        heads = []
        for h in range(case["q_heads"]):
            a = s["q"][row : row + m, h].double() @ k[:, h // group].T * case["dim"] ** -0.5
            a = torch.softmax(a.masked_fill(hidden, float("-inf")), -1)
            heads.append(a @ v[:, h // group])
        out.append(torch.stack(heads, 1))
        row += m
    return torch.cat(out)


def exact_rope(s, case):
    r, out = case["rotated"], []
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(s["positions"].double(), s["inv_freq"].double()))[:, None]
    for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])):
        y = x.double()
        if case["norm"]:
            y = y * torch.rsqrt(torch.mean(y ** 2, -1, keepdim=True) + 1e-6) * w.double()
        y = y.clone()
        pairs = y[..., :r].unflatten(-1, (r // 2, 2)) if case["interleaved"] else y[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        y[..., :r] = z.flatten(-2) if case["interleaved"] else z.transpose(-1, -2).flatten(-2)
        out.append(y)
    return tuple(out)


def exact_write(s, case, x, lens, new, table):
    """Page by page; the codes of a page come from all its tokens' values, the earlier ones as the cache holds them."""
    page, code, row = case["page"], case["code"], 0
    cache, scale = s[x + "_cache"], s[x + "_scale"]
    for b, (n, m) in enumerate(zip(lens, new)):
        value = s[x][row : row + m].double()
        row += m
        for c in range((n - m) // page, (n - 1) // page + 1):
            at, lo, hi = table[b][c], max(n - m, c * page), min(n, (c + 1) * page)
            fresh = value[lo - (n - m) : hi - (n - m)].transpose(0, 1)  # [head, token, dim]
            amax = fresh.abs().amax((1, 2))
            units = torch.div(amax, torch.full_like(amax, LARGEST[code]))  # a division by a number would be a product with its reciprocal
            part, least = torch.frexp(units)  # units = part * 2^least with part in [0.5, 1)
            least = torch.clamp(least - (part == 0.5).int(), min=-126)
            new_scale = torch.ldexp(torch.ones_like(amax), least)
            if lo > c * page:
                new_scale = torch.maximum(new_scale, scale[at].double())
                old = cache[at, :, : lo - c * page].double() * (scale[at].double() / new_scale)[:, None, None]
                cache.view(torch.uint8)[at, :, : lo - c * page] = rounded(old, code).view(torch.uint8)
            cache.view(torch.uint8)[at, :, lo - c * page : hi - c * page] = rounded(fresh / new_scale[:, None, None], code).view(torch.uint8)
            scale[at] = new_scale.float()
