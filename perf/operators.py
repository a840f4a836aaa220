"""The work by which the operators of serving in few bits are judged: matrices held in microscaled 4-bit floating point and
keys and values held in 8 bits with a scale for each page and head.

Each case is one call (with the read-out of what it stores, where it stores bits):

* ``quantize``: rows of activations or weights to 4-bit elements (sign, two bits of exponent, one of mantissa) with one
  power of two for each 32 elements of a row.  Returned as the values that the bits stand for.
* ``linear``: activations, rounded the same way within the call, times a matrix that is kept so; plain, or with the
  gated activation silu(gate) * up over the two halves of the matrix.
* ``store``: keys and values of a step's tokens into their pages, as 8-bit numbers with one power of two for each page,
  head and kind.  A page whose largest number grows gives its older tokens the larger step.  Returned as the values of
  all pages of the pool, the older tokens' among them.
* ``attend``: causal attention of a step's queries over such pages, for decoded tokens, portions of prompts and both.

``prepare`` makes inputs, pages and matrices with torch; ``run`` is the call, in its plain form or (``own``) through the
package's kernels; ``exact`` states the same in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 32             # elements of a row that share a scale
DEV = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    def quantize(name, rows, k, dtype="bfloat16"):
        return dict(name=name, kind="quantize", rows=rows, k=k, dtype=dtype)

    def linear(name, rows, k, features, dtype="bfloat16", gated=False):
        return dict(name=name, kind="linear", rows=rows, k=k, features=features, dtype=dtype, gated=gated)

    def store(name, requests, shortest, longest, tokens, page, kv_heads=8, dim=128, dtype="bfloat16"):
        return dict(name=name, kind="store", requests=requests, shortest=shortest, longest=longest, tokens=tokens, page=page,
                    kv_heads=kv_heads, group=1, dim=dim, dtype=dtype)

    def attend(name, requests, shortest, longest, tokens, page, kv_heads=8, group=2, dim=128, window=0, dtype="bfloat16"):
        """``requests`` with ``shortest`` to ``longest`` keys each, of which the first has ``tokens`` queries and the others one."""
        return dict(name=name, kind="attend", requests=requests, shortest=shortest, longest=longest, tokens=tokens, page=page,
                    kv_heads=kv_heads, group=group, dim=dim, window=window, dtype=dtype)

    return [
        # the normed rows of a decode step of eight requests, before a layer's first product (8B sizes)
        quantize("quantize-decode-8", 8, 4096),
        # a gate and up matrix when a model is loaded
        quantize("quantize-weights", 24576, 4096),
        # one chat: the q | k | v product of the 0.6B sizes, where latency counts
        linear("linear-decode-1", 1, 1024, 4096),
        # a decode step of eight: down of the 8B sizes, a long k
        linear("linear-decode-8-down", 8, 12288, 4096),
        # an odd number of decoding requests: gate and up of the 8B sizes
        linear("linear-decode-33-gate", 33, 4096, 12288, gated=True),
        # a document: gate and up of the 8B sizes
        linear("linear-prompt-2048-gate", 2048, 4096, 12288, gated=True),
        # a short prompt in the 32-bit mode, o of the 0.6B sizes
        linear("linear-prompt-193-fp32", 193, 2048, 1024, dtype="float32"),
        # a decode step of a full batch: each token joins a page that has older ones
        store("store-decode-64", 64, 1, 48, 1, 16),
        # a document that begins in the middle of a page
        store("store-prompt-2043", 1, 2100, 2100, 2043, 16),
        # a few long contexts decoding (8B heads)
        attend("attend-decode-8-long", 8, 3967, 8095, 1, 16, group=4),
        # a full batch of short chats (0.6B heads)
        attend("attend-decode-64", 64, 129, 383, 1, 16),
        # a portion of a long document beside decoding requests (8B heads)
        attend("attend-prompt-2000-mixed", 4, 2500, 8000, 2000, 16, group=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "store", "attend", "attend", "attend"])
    dtype = "float32" if rng.random() < 0.2 else "bfloat16"
    if kind == "quantize":
        k = BLOCK * _log(rng, 1, 384)
        return dict(kind=kind, rows=_log(rng, 1, min(24576, 100_000_000 // k)), k=k, dtype=dtype)
    if kind == "linear":
        k, gated = BLOCK * _log(rng, 2, 384), rng.random() < 0.4
        features = _log(rng, 17, 12288)
        return dict(kind=kind, rows=_log(rng, 1, 2048), k=k, features=features, dtype=dtype, gated=gated)
    c = dict(kind=kind, page=rng.choice([16, 16, 32, 64]), kv_heads=rng.choice([1, 2, 4, 8]), group=rng.choice([1, 2, 4, 5, 8]),
             dim=rng.choice([64, 128, 128, 256]), dtype=dtype, tokens=1)
    if kind == "store":
        c.update(group=1, requests=_log(rng, 1, 64))
        if rng.random() < 0.5:
            c["tokens"] = _log(rng, 2, 2048 // c["requests"] + 2)
        c["longest"] = c["tokens"] + rng.randint(0, 80)
        c["shortest"] = rng.randint(c["tokens"], c["longest"])
        return c
    c["window"] = rng.choice([0, 0, 0, _log(rng, 16, 2000)])
    if rng.random() < 0.55:
        c["requests"] = _log(rng, 1, 64)
        c["longest"] = _log(rng, 1, min(8000, 32000 // c["requests"]))
    else:
        c.update(requests=rng.randint(1, 4), tokens=_log(rng, 2, 1800))
        c["longest"] = c["tokens"] + _log(rng, 1, 4000)
        if c["kv_heads"] * c["group"] > 32:
            c["group"] = 4
    c["shortest"] = rng.randint(max(1, c["tokens"], c["longest"] // 4), c["longest"])
    return c


def _lengths(case):
    """(keys, queries) of each request: the lengths run evenly from the longest to the shortest."""
    n, lo, hi = case["requests"], case["shortest"], case["longest"]
    lens = [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]
    brings = [case["tokens"]] * n if case["kind"] == "store" else [case["tokens"]] + [1] * (n - 1)
    return lens, [min(a, b) for a, b in zip(lens, brings)]


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _activations(g, rows, k):
    """Rows as they leave a norm: most features alike, a few much larger."""
    gain = torch.exp(0.5 * _normal(g, (k,)))
    gain[torch.randint(0, k, (max(1, k // 256),), generator=g, device=DEV)] *= 12.0
    return _normal(g, (rows, k)) * gain


def _matrix(g, rows, k):
    """Codes [rows, k / 2] (element 2 i in the low half of a byte) and scales [rows, k / 32] of a random matrix."""
    codes = torch.empty((rows, k // 2), dtype=torch.uint8, device=DEV)
    scales = torch.empty((rows, k // BLOCK), dtype=torch.uint8, device=DEV)
    for at in range(0, rows, 8192):
        w = _normal(g, (min(8192, rows - at), k), 0.02).to(torch.bfloat16).float()
        value, scale = _round4(w)
        code = torch.bucketize(value.abs(), torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEV)).to(torch.uint8)
        code += 8 * (w < 0).to(torch.uint8)
        codes[at:at + w.shape[0]] = code[:, 0::2] | (code[:, 1::2] << 4)
        scales[at:at + w.shape[0]] = scale
    return codes, scales


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case, dtype=dtype)
    if case["kind"] == "quantize":
        s["x"] = _activations(g, case["rows"], case["k"]).to(dtype)
    elif case["kind"] == "linear":
        s["x"] = _activations(g, case["rows"], case["k"]).to(dtype)
        s["codes"], s["scales"] = _matrix(g, case["features"] * (2 if case["gated"] else 1), case["k"])
    else:
        _prepare_pages(case, s, g)
    if own:
        _prepare_own(case, s)
    return s


def _prepare_pages(case, s, g):
    page, heads, dim = case["page"], case["kv_heads"], case["dim"]
    lens, brings = _lengths(case)
    held = [-(-n // page) for n in lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    tables = torch.full((len(lens), max(held)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for r, n in enumerate(held):
        tables[r, :n] = order[at:at + n]
        at += n
    # what the pages hold: keys of uneven size by head and feature, values of uneven size by head
    size = torch.exp(0.4 * _normal(g, (2, heads, 1, 1)))
    feature = torch.stack((torch.exp(0.5 * _normal(g, (heads, 1, dim))), torch.ones((heads, 1, dim), device=DEV)))
    s["codes"] = torch.empty((pages, 2, heads, page, dim), dtype=torch.int8, device=DEV)
    s["exponents"] = torch.empty((pages, 2, heads), dtype=torch.uint8, device=DEV)
    for a in range(0, pages, 256):
        kv = _normal(g, (min(256, pages - a), 2, heads, page, dim)) * (size * feature)
        field = _field(kv.abs().amax(dim=(3, 4)))
        s["codes"][a:a + kv.shape[0]] = _codes8(kv, field[..., None, None])
        s["exponents"][a:a + kv.shape[0]] = field.to(torch.uint8)
    total = sum(brings)
    cu = [0]
    for n in brings:
        cu.append(cu[-1] + n)
    s.update(tables=tables, cu_q=torch.tensor(cu, dtype=torch.int32, device=DEV),
             seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV), max_q=max(brings), min_q=min(brings), max_len=max(lens),
             total=total)
    if case["kind"] == "attend":
        s["q"] = (_normal(g, (total, heads * case["group"], dim))).to(s["dtype"])
        s["scale"] = dim ** -0.5
        return
    new = _normal(g, (2, total, heads, dim)) * (size * feature).movedim(2, 1) * torch.exp(0.4 * _normal(g, (1, total, 1, 1)))
    s["k"], s["v"] = new[0].to(s["dtype"]).contiguous(), new[1].to(s["dtype"]).contiguous()
    owner = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(brings, device=DEV))
    position = s["seq_lens"][owner] - s["cu_q"][1:][owner] + torch.arange(total, device=DEV)
    s["slots"] = (tables[owner, position // page] * page + position % page).to(torch.int32)


def _prepare_own(case, s):
    """What a user of the package keeps besides: the kernels, a matrix in their layout, pages, and room for results."""
    from infurnace_b200.kernels import Kv8Pages, Mx4Matrix, load_cuda_kernels
    s["kernels"] = load_cuda_kernels()
    if case["kind"] == "quantize":
        s["matrix"] = Mx4Matrix.empty(case["rows"], case["k"], DEV)
    elif case["kind"] == "linear":
        s["matrix"] = Mx4Matrix.from_parts(s.pop("codes"), s.pop("scales"), gated=case["gated"])
    else:
        s["pages"] = Kv8Pages(s["codes"], s["exponents"])


# ------------------------------------------------------------------------------------------------ the plain forms
def _power(e):
    """2^e in float32 for whole e from -149 to 127, from its bits."""
    e = e.to(torch.int32)
    normal = (e + 127) << 23
    return torch.where(e >= -126, normal, 1 << (e + 149).clamp(0, 22)).view(torch.float32)


def _field(amax):
    """floor(log2) + 127 of a float32 number (its exponent field): 0 for zeros, 255 for infinities and NaN."""
    return (amax.float().view(torch.int32) >> 23) & 255


def _round4(x):
    """Elements rounded to 4 bits, in units of their block's scale, and the scales' bytes (a power of two, 127 more than its
    exponent; 255: NaN).  The largest of a block lies in [4, 8) units; what exceeds 6 becomes 6, ties go to the even code."""
    b = x.reshape(x.shape[0], -1, BLOCK)
    field = _field(b.abs().amax(dim=2))
    scale = torch.where(field == 255, 255, (field - 2).clamp(min=0))
    t = b * _power(127 - scale.clamp(max=254))[..., None]
    mag = t.abs().clamp(max=6.0)
    unit = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    value = torch.copysign(torch.round(mag / unit) * unit, t)
    return value.reshape(x.shape), scale.to(torch.uint8)


def _scaled(value, scale):
    """Values in units, times their blocks' scales."""
    factor = torch.where(scale == 255, math.nan, _power(scale.to(torch.int32).clamp(max=254) - 127))
    return (value.reshape(value.shape[0], -1, BLOCK) * factor[..., None]).reshape(value.shape)


def _values4(codes, scales):
    nibbles = torch.stack((codes & 15, codes >> 4), dim=2).reshape(codes.shape[0], -1).long()
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
    return _scaled(torch.cat((levels, -levels))[nibbles], scales)


def _codes8(x, field):
    """floor(x / step), step = 2^(field - 133): a number of a block whose largest has the exponent field ``field``."""
    e = 133 - field
    half = e // 2
    t = torch.floor(x.float() * _power(half) * _power(e - half))
    return torch.where((x < 0) & (t == 0), -1, t).clamp(-128, 127).to(torch.int8)


def _values8(codes, exponents):
    """(code + 1/2) steps; a block of zeros is zero, one that held an infinity or NaN is NaN."""
    f = exponents.to(torch.int32)
    step = torch.where(f == 0, 0.0, torch.where(f == 255, math.nan, _power(f - 133)))
    return (codes.float() + 0.5) * step[..., None, None]


def _plain_quantize(s):
    return _scaled(*_round4(s["x"].float())).to(s["dtype"])


def _plain_linear(s):
    x = _scaled(*_round4(s["x"].float()))
    y = x @ _values4(s["codes"], s["scales"]).T
    if s["case"]["gated"]:
        gate, up = y.chunk(2, dim=1)
        y = gate * torch.sigmoid(gate) * up
    return y.to(s["dtype"])


def _plain_store(s):
    codes, old = s["codes"], s["exponents"].to(torch.int32)
    slots = s["slots"].long()
    page, offset = slots // codes.shape[3], slots % codes.shape[3]
    kv = torch.stack((s["k"], s["v"]), dim=1)                           # [tokens, 2, heads, dim]
    base = old.clone()
    base[page[offset == 0]] = 0                                         # a page that begins anew
    fresh = torch.zeros(old.shape[0], dtype=torch.bool, device=DEV)
    fresh[page[offset == 0]] = True
    largest = _field(kv.abs().amax(dim=3))
    field = base.scatter_reduce(0, page[:, None, None].expand_as(largest), largest, "amax")
    shift = torch.where(fresh[:, None, None] | (field == 255), 0, (field - old).clamp(0, 7))
    codes.copy_((codes.to(torch.int32) >> shift[..., None, None]).to(torch.int8))
    codes[page, :, :, offset] = _codes8(kv, field[page][..., None])
    s["exponents"].copy_(field.to(torch.uint8))
    return _values8(codes, s["exponents"]).to(s["dtype"])


def _plain_attend(s):
    case, page = s["case"], s["case"]["page"]
    heads, group, dim = case["kv_heads"], case["group"], case["dim"]
    requests, longest, most = case["requests"], s["max_len"], s["max_q"]
    held = -(-longest // page)
    tables = s["tables"].clamp(min=0).long()
    kv = _values8(s["codes"], s["exponents"])[tables]                   # [requests, held, 2, heads, page, dim]
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, requests, heads, held * page, dim)
    counts = s["cu_q"][1:] - s["cu_q"][:-1]
    token = torch.arange(most, device=DEV)
    real = token < counts[:, None]                                      # [requests, most]
    row = (s["cu_q"][:-1, None] + token).clamp(max=s["total"] - 1).long()
    q = s["q"].float()[row].reshape(requests, most, heads, group, dim).permute(0, 2, 3, 1, 4)
    scores = (q.reshape(requests, heads, group * most, dim) @ kv[0].transpose(2, 3)).reshape(requests, heads, group, most, -1)
    position = (s["seq_lens"] - counts)[:, None] + token
    key = torch.arange(held * page, device=DEV)
    seen = key <= position[:, :, None]
    if case["window"]:
        seen &= key > position[:, :, None] - case["window"]
    scores = torch.where(seen[:, None, None], scores * s["scale"], -math.inf)
    weight = torch.exp(scores - scores.amax(dim=4, keepdim=True))
    weight = weight / weight.sum(dim=4, keepdim=True)
    y = (weight.reshape(requests, heads, group * most, -1) @ kv[1]).reshape(requests, heads, group, most, dim)
    return y.permute(0, 3, 1, 2, 4).reshape(requests, most, heads * group, dim)[real].to(s["dtype"])


# ------------------------------------------------------------------------------------------------ the package's kernels
def _own_quantize(s):
    s["kernels"].mx4_quantize(s["x"], s["matrix"])
    out = torch.empty_like(s["x"])
    s["kernels"].mx4_values(s["matrix"], out)
    return out


def _own_linear(s):
    case = s["case"]
    out = torch.empty((case["rows"], case["features"]), dtype=s["dtype"], device=DEV)
    s["kernels"].mx4_linear(s["x"], s["matrix"], out, epilogue="silu_gate" if case["gated"] else "none")
    return out


def _own_store(s):
    s["kernels"].kv8_store(s["k"], s["v"], s["slots"], s["pages"])
    out = torch.empty(s["codes"].shape, dtype=s["dtype"], device=DEV)
    s["kernels"].kv8_values(s["pages"], out)
    return out


def _own_attend(s):
    out = torch.empty_like(s["q"])
    s["kernels"].kv8_attention(s["q"], s["pages"], s["tables"], s["cu_q"], s["seq_lens"], out, s["scale"], s["case"]["window"],
                               s["max_q"], s["max_len"], min_q_len=s["min_q"])
    return out


def run(state):
    forms = (dict(quantize=_own_quantize, linear=_own_linear, store=_own_store, attend=_own_attend) if own else
             dict(quantize=_plain_quantize, linear=_plain_linear, store=_plain_store, attend=_plain_attend))
    return forms[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    width = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "quantize":
        n = case["rows"] * case["k"]
        return dict(bytes=n * (2 * width + 0.5 + 1 / BLOCK), flops=0)
    if case["kind"] == "linear":
        rows, k, features = case["rows"], case["k"], case["features"]
        w = features * (2 if case["gated"] else 1)
        return dict(bytes=rows * k * width + w * k * (0.5 + 1 / BLOCK) + rows * features * width, flops=2 * rows * k * w)
    lens, brings = _lengths(case)
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "store":
        pool = (sum(-(-n // page) for n in lens) + 3) * 2 * heads * page * dim
        return dict(bytes=sum(brings) * 2 * heads * dim * (width + 1) + pool * (1 + width), flops=0)
    w, pairs, read = case["window"], 0, 0
    for n, m in zip(lens, brings):
        first = n - m
        read += n - max(0, first - w + 1) if w else n
        pairs += sum(min(p + 1, w) for p in range(first, n)) if w else m * first + m * (m + 1) // 2
    rows = sum(brings) * heads * case["group"]
    return dict(bytes=read * 2 * heads * dim + 2 * rows * dim * width, flops=4 * pairs * heads * case["group"] * dim)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _two(e):
    """2^e in float64 for whole e, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _blocks64(x):
    """Rows rounded to 4 bits in 64-bit arithmetic: the nearest of the 8 levels, found among all of them."""
    b = x.double().reshape(x.shape[0], -1, BLOCK)
    exponent = torch.frexp(b.abs().amax(dim=2))[1] - 1                  # amax = m 2^exponent, 1 <= m < 2
    scale = _two((exponent - 2).clamp(min=-127))[..., None]
    t = b / scale
    best, far = torch.zeros_like(t), t.abs()
    for code, level in enumerate((0, 0.5, 1, 1.5, 2, 3, 4, 6)):
        d = (t.abs() - level).abs()
        take = (d < far) | ((d == far) & (code % 2 == 0))
        best, far = torch.where(take, float(level), best), torch.minimum(far, d)
    return (torch.where(t < 0, -best, best) * scale).reshape(x.shape)


def _matrix64(codes, scales):
    low, high = (codes & 15).long(), (codes >> 4).long()
    n = torch.stack((low, high), dim=2).reshape(codes.shape[0], -1)
    e, m = (n >> 1) & 3, (n & 1).double()
    value = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * _two(e - 1)) * (1 - 2 * (n >> 3).double())
    return value * _two(scales.long().repeat_interleave(BLOCK, dim=1) - 127)


def _pages64(codes, exponents):
    return (2 * codes.double() + 1) * (_two(exponents.long() - 134) * (exponents > 0))[..., None, None]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        return torch.cat([_blocks64(x) for x in s["x"].split(2048)])
    if case["kind"] == "linear":
        y = _blocks64(s["x"]) @ _matrix64(s["codes"], s["scales"]).T
        if case["gated"]:
            n = case["features"]
            y = y[:, :n] / (1 + torch.exp(-y[:, :n])) * y[:, n:]
        return y
    return _exact_store(case, s) if case["kind"] == "store" else _exact_attend(case, s)


def _exact_store(case, s):
    """A page's numbers under the step of its largest: floor of a floor is the floor of the whole, so the older codes and the
    new numbers go by the same rule."""
    page = case["page"]
    codes, field = s["codes"].double(), s["exponents"].long()
    for t, slot in enumerate(s["slots"].tolist()):                      # the exponents first, token by token
        p = slot // page
        kv = torch.stack((s["k"][t], s["v"][t])).double()
        largest = torch.frexp(kv.abs().amax(dim=2))[1] + 126
        field[p] = largest if slot % page == 0 else torch.maximum(field[p], largest)
    begun = torch.zeros(codes.shape[0], dtype=torch.bool, device=DEV)
    begun[s["slots"].long()[s["slots"] % page == 0] // page] = True
    drop = torch.where(begun[:, None, None], 0, field - s["exponents"].long())
    codes = torch.floor(codes / _two(drop)[..., None, None])
    p, o = s["slots"].long() // page, s["slots"].long() % page
    step = _two(field - 133)
    codes[p, :, :, o] = torch.floor(torch.stack((s["k"], s["v"]), dim=1).double() / step[p][..., None])
    return (codes + 0.5) * step[..., None, None]


def _exact_attend(case, s):
    heads, group, dim, page = case["kv_heads"], case["group"], case["dim"], case["page"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    lens, brings = _lengths(case)
    at = 0
    for r, (n, m) in enumerate(zip(lens, brings)):
        used = s["tables"][r, :-(-n // page)].long()
        kv = _pages64(s["codes"][used], s["exponents"][used]).transpose(0, 2).transpose(0, 1)       # [2, heads, pages, page, dim]
        kv = kv.reshape(2, heads, -1, dim)[:, :, :n]
        p = torch.arange(n - m, n, device=DEV)[:, None]
        key = torch.arange(n, device=DEV)[None]
        hidden = key > p
        if case["window"]:
            hidden |= key + case["window"] <= p
        for h in range(heads * group):
            score = s["q"][at:at + m, h].double() @ kv[0, h // group].T * s["scale"]
            out[at:at + m, h] = torch.softmax(score.masked_fill(hidden, -math.inf), dim=1) @ kv[1, h // group]
        at += m
    return out
