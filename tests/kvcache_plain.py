"""Plain implementations in 64 bits of the operators around the 8-bit key/value cache, one sequence, page and head at a
time, and the inputs the tests share."""
import torch

LARGEST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FORMATS = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
FLOATS = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def half_step(dtype):
    """The largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


class Batch:
    """A cache and the sequences of one call.  `new` and `lens` are host lists; pages are handed out in a shuffled order.
    Slots that hold no token have the byte `stale` (0x7F is no number in e4m3)."""

    def __init__(self, seed, lens, new, heads, dim, page, fmt, device="cuda", stale=0x7F, extra_pages=3, extra_rows=0, extra_cols=1):
        self.lens, self.new, self.heads, self.dim, self.page, self.fmt = lens, new, heads, dim, page, FORMATS[fmt]
        self.g = torch.Generator().manual_seed(seed)
        self.device = device
        self.cols = max([-(-n // page) for n in lens] + [0]) + extra_cols
        self.pages = len(lens) * self.cols + extra_pages
        order = torch.randperm(self.pages, generator=self.g)
        self.host_table = order[: len(lens) * self.cols].reshape(len(lens), self.cols)
        table = self.host_table.clone()
        for b, n in enumerate(lens):
            table[b, -(-n // page):] = 2**31 - 1  # columns no token is in are never looked at
        self.table = table.int().to(device)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.host_starts, self.rows = starts, starts[-1] + extra_rows
        self.starts = torch.tensor(starts, dtype=torch.int32, device=device)
        self.length = torch.tensor(lens, dtype=torch.int32, device=device)
        shape = (self.pages, heads, page, dim)
        self.k, self.v = (torch.full(shape, stale, dtype=torch.uint8, device=device).view(self.fmt) for _ in "kv")
        self.ks, self.vs = (torch.full(shape[:2], float("nan"), device=device) for _ in "kv")
        self.flag = torch.zeros(1, dtype=torch.int32, device=device)

    def rand(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, generator=self.g).to(dtype).to(self.device)

    def fill(self, counts, scale_exponents=(-8, -4)):
        """The first counts[b] tokens of each sequence at random: any code, any scale of the range."""
        for codes, scales in ((self.k, self.ks), (self.v, self.vs)):
            for b, n in enumerate(counts):
                for c in range(-(-n // self.page)):
                    at, m = int(self.host_table[b, c]), min(self.page, n - c * self.page)
                    if self.fmt == torch.int8:
                        x = torch.randint(-127, 128, (self.heads, m, self.dim), generator=self.g).to(torch.int8).view(torch.uint8)
                    else:
                        x = torch.randint(0, 254, (self.heads, m, self.dim), generator=self.g, dtype=torch.uint8)
                        x = torch.where(x >= 127, x + 1, x)
                    codes.view(torch.uint8)[at, :, :m] = x.to(self.device)
                    e = torch.randint(scale_exponents[0], scale_exponents[1] + 1, (self.heads,), generator=self.g)
                    scales[at] = torch.ldexp(torch.ones(self.heads), e).to(self.device)
        return self

    def cache(self):
        return self.k, self.v, self.ks, self.vs

    def seqs(self):
        return self.starts, self.length, self.table

    def history(self, codes, scales, b, n=None):
        """[token, head, dim] of sequence b in float64."""
        n = self.lens[b] if n is None else n
        out = torch.zeros(n, self.heads, self.dim, dtype=torch.float64, device=codes.device)
        for c in range(-(-n // self.page)):
            at, m = int(self.host_table[b, c]), min(self.page, n - c * self.page)
            out[c * self.page: c * self.page + m] = (codes[at, :, :m].double() * scales[at].double()[:, None, None]).transpose(0, 1)
        return out


def power_of_two(amax, largest):
    """Least 2^e >= amax / largest, e >= -126, amax a float64 tensor (the division is by a power of two times 127 or 448: compared, not divided)."""
    e = torch.full(amax.shape, -126, dtype=torch.int64)
    for i in range(amax.numel()):
        x, k = float(amax.flatten()[i]), -126
        while largest * 2.0**k < x:
            k += 1
        e.view(-1)[i] = k
    return torch.ldexp(torch.ones(amax.shape, dtype=torch.float64), e)


def encode(x, fmt):
    """float64 values in units of their scale → codes."""
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-LARGEST[fmt], LARGEST[fmt])
    return x.round().to(torch.int8) if fmt == torch.int8 else x.float().to(fmt)


def write(batch, K, V):
    """What kvcache_write makes of batch's cache, on the host: (k, v, k_scale, v_scale)."""
    out = []
    for X, codes, scales in ((K, batch.k, batch.ks), (V, batch.v, batch.vs)):
        codes, scales, X = codes.cpu().clone(), scales.cpu().clone(), X.cpu().double()
        for b, (n, m) in enumerate(zip(batch.lens, batch.new)):
            x = X[batch.host_starts[b]: batch.host_starts[b] + m][max(0, m - n):]
            first = max(0, n - m)
            for c in range(first // batch.page, -(-n // batch.page) if n > first else 0):
                at = int(batch.host_table[b, c])
                lo, hi = max(first, c * batch.page), min(n, (c + 1) * batch.page)
                part = x[lo - first: hi - first].transpose(0, 1)
                size = torch.where(torch.isfinite(part), part.abs(), torch.zeros_like(part)).amax((1, 2))
                scale = power_of_two(size, LARGEST[batch.fmt])
                slot = lo - c * batch.page
                if slot:
                    old = scales[at].double()
                    scale = torch.maximum(scale, old)
                    codes[at, :, :slot] = encode(codes[at, :, :slot].double() * (old / scale)[:, None, None], batch.fmt)
                codes[at, :, slot: slot + hi - lo] = encode(part / scale[:, None, None], batch.fmt)
                scales[at] = scale.float()
        out += [codes, scales]
    return out[0], out[2], out[1], out[3]


def attention(batch, Q, scale, window=0):
    """(out, bound): the attention of the new tokens in float64, and how far a kernel may be from it before its last rounding.

    The bound: weights are held in 16 bits (11 significant ones): each is off by 2^-11 at most, and so is their sum that
    divides, 2^-10 of A = sum p|v| together.  A score is a float32 sum of dim products, each addition off by 2^-23 (tensor cores
    may cut where others round): an error of dim * 2^-23 * scale * sum |q||k| in the exponent, twice since the maximum has it
    too, and the weights and their sum have it both: four times.  The output is a float32 sum over the keys: keys * 2^-23 of A.
    A q of bfloat16 keeps its 8 bits; 2^-24 of the row's largest for elements far below it is inside the dim term.  The exponential
    itself and its argument's rounding: 2^-21 + 2^-23 * |argument|, the argument below 200 where a weight counts: 2^-15 of A.
    16-bit floats below 2^-14 have the fixed step 2^-24: with weights held so that the largest is 2^7 or more, each is off by
    2^-25 / 2^7 of the sum at most on top, where the largest value is that of the largest code and scale (codes may be in units of the
    largest scale, the weights taking the difference, in which a scale that is no power of two rounds once more: 2^-11 of A)."""
    heads = Q.shape[1]
    group = heads // batch.heads
    out = torch.zeros(Q.shape, dtype=torch.float64, device=Q.device)
    bound = torch.zeros_like(out)
    for b, (n, m) in enumerate(zip(batch.lens, batch.new)):
        if m == 0 or n == 0:
            continue
        k, v = batch.history(batch.k, batch.ks, b), batch.history(batch.v, batch.vs, b)
        largest = batch.vs[batch.host_table[b, : -(-n // batch.page)].to(Q.device)].max()
        key = torch.arange(n, device=Q.device)[None, :]
        pos = torch.arange(n - m, n, device=Q.device)[:, None]
        seen = key <= pos
        if window:
            seen &= key > pos - window
        row = batch.host_starts[b]
        for h in range(heads):
            q, kh, vh = Q[row: row + m, h].double(), k[:, h // group], v[:, h // group]
            s = (q @ kh.T) * scale
            p = torch.exp((s - s.masked_fill(~seen, -torch.inf).amax(-1, keepdim=True).clamp(min=-1e300)).masked_fill(~seen, -torch.inf))
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, torch.zeros_like(p))
            out[row: row + m, h] = p @ vh
            size = p @ vh.abs()
            score = ((q.abs() @ kh.abs().T) * scale * seen).amax(-1, keepdim=True)
            fixed = 2.0**-32 * seen.double().sum(-1, keepdim=True) * (LARGEST[batch.fmt] * float(largest))
            bound[row: row + m, h] = fixed + size * (2.0**-10 + 2.0**-11 + 4 * batch.dim * 2.0**-23 * score + n * 2.0**-23 + 2.0**-15)
    return out, bound


def attention_rows(batch, Q, scale, window=0):
    """(out, bound) as `attention`, with a bound that depends on nothing but what a row weighs: its weights p, and the values v = s * code
    of the tokens it sees, s the scale of a token's page.

    A weight times its page's scale (a power of two) is held in 16 bits, so that the largest of a row is 2^7 or more times (a maximum may be
    rounded up to a whole power of two: 2^6): relative to its own size each is off by 2^-11, or by the fixed half step 2^-25 of what is below 2^-14,
    which is 2^-31 of the row's largest p * s.  A code is at most 127 (448): together 2^-11 of A = sum p|v|, and 2^-31 * keys * 127 (448) * max(p * s).
    Weights are 32-bit numbers: those below 2^-126 of the largest are zero, at most 2^-126 * sum |v|.
    The sum that divides is of weights in 32 bits.  Scores, sums and exponentials as in `attention`; the arguments of the exponentials
    that count are below 256, and there are three of them for a weight (its own, that of the scale's unit, that of the parts' maxima): 3 * 2^-17
    is inside 2^-15."""
    heads = Q.shape[1]
    group = heads // batch.heads
    out = torch.zeros(Q.shape, dtype=torch.float64, device=Q.device)
    bound = torch.zeros_like(out)
    for b, (n, m) in enumerate(zip(batch.lens, batch.new)):
        if m == 0 or n == 0:
            continue
        pages = batch.host_table[b, torch.arange(n) // batch.page].to(Q.device)
        slot = torch.arange(n, device=Q.device) % batch.page
        key = torch.arange(n, device=Q.device)[None, :]
        pos = torch.arange(n - m, n, device=Q.device)[:, None]
        seen = key <= pos
        if window:
            seen &= key > pos - window
        row = batch.host_starts[b]
        for h in range(heads):
            kv = h // group
            ks, vs = (x[pages, kv].double() for x in (batch.ks, batch.vs))
            kh = torch.nan_to_num(batch.k[pages, kv, slot].double()) * torch.nan_to_num(ks)[:, None]
            vh = torch.nan_to_num(batch.v[pages, kv, slot].double()) * torch.nan_to_num(vs)[:, None]
            q = Q[row: row + m, h].double()
            s = ((q @ kh.T) * scale).masked_fill(~seen, -torch.inf)
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, torch.zeros_like(p))
            out[row: row + m, h] = p @ vh
            score = ((q.abs() @ kh.abs().T) * scale * seen).amax(-1, keepdim=True)
            fixed = 2.0**-31 * seen.double().sum(-1, keepdim=True) * LARGEST[batch.fmt] * (p * torch.nan_to_num(vs)).amax(-1, keepdim=True)
            fixed = fixed + 2.0**-126 * (seen.double() @ vh.abs())
            bound[row: row + m, h] = fixed + (p @ vh.abs()) * (2.0**-11 + 4 * batch.dim * 2.0**-23 * score + n * 2.0**-23 + 2.0**-15)
    return out, bound


def rope(x, weight, inv_freq, positions, eps, interleaved):
    """(y, scale): the norm and rotation of [tokens, heads, dim] in float64, and the size of the pair each element is of."""
    y = x.double()
    if eps is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if weight is not None:
            y = y * weight.double()
    y = y.clone()
    size = y.abs()
    r = 2 * inv_freq.numel()
    for i in range(r // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
        angle = (positions.double() * inv_freq[i].double())[:, None]
        u, w = y[..., a].clone(), y[..., b].clone()
        y[..., a], y[..., b] = u * angle.cos() - w * angle.sin(), w * angle.cos() + u * angle.sin()
        size[..., a] = size[..., b] = u.abs() + w.abs()
    return y, size
