"""Plain statements in 64 bits of the operators over few bits: rows rounded to 4 bits with a scale for each 32 elements, and
keys and values of 8 bits with a scale for each page and head.  Written from the definitions, level by level, for the CPU."""
import math

import torch

from kernel_refs import ReferenceKernels

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def field_of(amax):
    """The exponent field of a float32 number: floor(log2) + 127, 0 for zeros and subnormal numbers, 255 for infinities and NaN."""
    return (amax.float().contiguous().view(torch.int32) >> 23) & 255


def two(e):
    return torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())


def round4(x):
    """(codes [rows, k] 0 .. 15, scale bytes [rows, k / 32], values [rows, k] float64) of rows."""
    rows, k = x.shape
    b = x.double().view(rows, k // 32, 32)
    f = field_of(x.float().view(rows, k // 32, 32).abs().nan_to_num(math.inf, math.inf, -math.inf).amax(2)).long()
    scale = torch.where(f == 255, 255, (f - 2).clamp(min=0))
    t = b / two(scale.clamp(max=254) - 127)[..., None]
    mag = t.abs().nan_to_num(0.0, 1e300)
    code = torch.zeros_like(mag, dtype=torch.long)
    for i in range(1, 8):
        mid = (LEVELS[i] + LEVELS[i - 1]) / 2
        code += ((mag > mid) | ((mag == mid) & (i % 2 == 0))).long()          # a tie goes to the even code
    value = torch.tensor(LEVELS, dtype=torch.float64)[code] * torch.where(t < 0, -1.0, 1.0)
    value = torch.where(scale[..., None] == 255, math.nan, value * two(scale - 127)[..., None])
    return (code + 8 * torch.signbit(b)).view(rows, k), scale, value.reshape(rows, k)


def step_of(field):
    """The step of a block of 8-bit numbers from its exponent field."""
    f = field.long()
    return torch.where(f == 0, 0.0, torch.where(f == 255, math.nan, two(f - 133)))


def values8(codes, fields):
    return (codes.double() + 0.5) * step_of(fields)[..., None, None]


def code8(x, field):
    """floor(x / step) of numbers of a block whose largest has the exponent field ``field`` (1 .. 254); -1 or 0 where it is 0."""
    return torch.floor(x.double() / two(field.long() - 133)).clamp(-128, 127)


def store8(codes, fields, k, v, slots):
    """Codes and exponent fields after a step's tokens (k, v [tokens, heads, dim]) are stored at ``slots``, from the definition:
    a block holds floor(number / step) of all its numbers, for the step of its largest."""
    codes, fields = codes.double().clone(), fields.long().clone()
    page_size = codes.shape[3]
    slots = slots.tolist()
    new = fields.clone()
    for t, s in enumerate(slots):
        if s < 0:
            continue
        f = field_of(torch.stack((k[t], v[t])).float().abs().nan_to_num(math.inf, math.inf, -math.inf).amax(2)).long()
        p = s // page_size
        new[p] = f if s % page_size == 0 else torch.maximum(new[p], f)
    begun = {s // page_size for s in slots if s >= 0 and s % page_size == 0}
    for p in {s // page_size for s in slots if s >= 0}:
        if p not in begun:
            grow = (new[p] - fields[p]).clamp(0, 60)
            grow[(new[p] == 255)] = 0
            codes[p] = torch.floor(codes[p] / two(grow)[..., None, None])
    for t, s in enumerate(slots):
        if s >= 0:
            p, o = s // page_size, s % page_size
            codes[p, :, :, o] = code8(torch.stack((k[t], v[t])).nan_to_num(0.0, 0.0, 0.0), new[p][..., None])
    return codes, new


def attention8(q, codes, fields, tables, cu_q, seq_lens, scale, window=0):
    """Causal attention over the pages' values, request by request; a row that sees no key is zero.  Returns the output, for
    each of its numbers the weighted sum of magnitudes, and for each row the most that rounding could act on in a score:
    scale * sum |q| * 256 * the largest step."""
    heads, page_size, dim = codes.shape[2:]
    out = torch.zeros(q.shape, dtype=torch.float64)
    mag, reach = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64)
    group = q.shape[1] // heads
    for r in range(len(seq_lens)):
        a, b, n = int(cu_q[r]), int(cu_q[r + 1]), int(seq_lens[r])
        if n == 0 or a == b:
            continue
        pos = torch.arange(n)
        kv = torch.zeros((n, 2, heads, dim), dtype=torch.float64)
        lowest = max(0, n - (b - a) - window + 1) if window else 0         # entries of pages before it may have been given back
        pages = tables[r][pos[lowest:] // page_size].long()
        kv[lowest:] = (codes[pages, :, :, pos[lowest:] % page_size].double() + 0.5) * step_of(fields)[pages][..., None]
        step = step_of(fields)[pages, 0].nan_to_num(0.0)
        p = torch.arange(n - (b - a), n)[:, None]
        seen = (pos <= p) & ((pos > p - window) if window else torch.ones((), dtype=torch.bool))
        for h in range(heads * group):
            x = q[a:b, h].double()
            kvh, vis = kv[:, :, h // group], seen
            s = torch.where(vis, (x @ kvh[:, 0].T) * scale, -math.inf)
            w = torch.where(vis.any(1, keepdim=True), torch.softmax(s, 1), 0.0)
            # a number that is not seen has no part, be it NaN
            v = torch.where(vis[:, :, None], kvh[None, :, 1], 0.0)
            out[a:b, h] = torch.einsum("tn,tnd->td", w.nan_to_num(0.0) if not torch.isnan(s[vis]).any() else w, v)
            mag[a:b, h] = torch.einsum("tn,tnd->td", w, v.abs())
            reach[a:b, h] = scale * x.abs().sum(1) * 256 * step[:, h // group].max()
    return out, mag, reach


class LowBitReference(ReferenceKernels):
    """The stand-in kernel set with the operators over few bits: a 4-bit matrix is its values, pages are the package's."""

    def mx4_matrix(self, w, gated=False):
        return FourBits(round4(w.float())[2])

    def linear(self, x, w, out, epilogue="none", row_scale=None, bias=None):
        if isinstance(w, FourBits):
            assert row_scale is None and bias is None
            x, w = round4(x.float())[2], w.values
        super().linear(x, w, out, epilogue, row_scale, bias)

    def can_fold_norm(self, n, dtype, w, epilogue="none"):
        return not isinstance(w, FourBits) and super().can_fold_norm(n, dtype, w, epilogue)

    def kv8_store(self, k, v, slot_mapping, pages):
        codes, fields = store8(pages.codes, pages.exponents, k, v, slot_mapping)
        pages.codes.copy_(codes.to(torch.int8))
        pages.exponents.copy_(fields.to(torch.uint8))

    def kv8_attention(self, q, pages, block_tables, cu_q, seq_lens, out, scale, window, max_q_len, max_seq_len, min_q_len=1, exact_lens=False):
        assert max_seq_len <= block_tables.shape[1] * pages.page_size
        out.copy_(attention8(q, pages.codes, pages.exponents, block_tables, cu_q, seq_lens, scale, window)[0].to(out.dtype))


class FourBits:
    """A matrix rounded to 4 bits, as its values."""
    dtype = torch.uint8

    def __init__(self, values):
        self.values, self.shape = values, values.shape
