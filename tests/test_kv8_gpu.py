"""Pages of keys and values in 8 bits on the device against their plain statement in 64 bits (tests/low_bit_refs.py): the store
bit for bit and however the tokens are cut, attention within the bounds of its roundings."""
import math

import pytest
import torch

from low_bit_refs import attention8, store8, values8

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


def pages_of(n, heads, ps, dim, seed):
    """Codes and exponent fields of blocks of uneven size, one of them of zeros."""
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(-128, 128, (n, 2, heads, ps, dim), generator=g, dtype=torch.int64).to(torch.int8)
    fields = torch.randint(121, 131, (n, 2, heads), generator=g).to(torch.uint8)
    fields[0, :, 0] = 0
    return codes, fields


def on_device(codes, fields):
    from infurnace_b200.kernels import Kv8Pages
    return Kv8Pages(codes.cuda(), fields.cuda())


def tokens_of(n, heads, dim, seed, dtype):
    """Keys and values whose size grows and shrinks from token to token, so that steps grow inside a page."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((2, n, heads, dim), generator=g) * torch.exp(1.5 * torch.randn((2, n, heads, 1), generator=g))
    return x.to(dtype)


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


# ------------------------------------------------------------------------------------------------ store
STORES = [(16, 1, 16, 1), (16, 2, 128, 5), (32, 3, 80, 70), (64, 8, 128, 200), (48, 2, 256, 100), (128, 1, 64, 300)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps,heads,dim,n", STORES)
def test_store_is_the_definitions_bit_for_bit(K, dtype, ps, heads, dim, n):
    """Two requests, one from the middle of a page on, in pages out of order, between rows that are not stored."""
    codes, fields = pages_of(2 * (n // ps + 3), heads, ps, dim, n)
    k, v = tokens_of(2 * n + 3, heads, dim, n + 1, dtype)
    order = torch.randperm(codes.shape[0], generator=torch.Generator().manual_seed(3))
    need = n // ps + 2
    pos = torch.arange(ps // 2 + 1, ps // 2 + 1 + n)
    slots = torch.full((2 * n + 3,), -1, dtype=torch.int64)
    slots[1:n + 1] = order[pos // ps] * ps + pos % ps
    slots[n + 2:2 * n + 2] = order[need + torch.arange(n) // ps] * ps + torch.arange(n) % ps
    ref_codes, ref_fields = store8(codes, fields, k, v, slots)
    pages = on_device(codes, fields)
    K.kv8_store(k.cuda(), v.cuda(), slots.to(torch.int32).cuda(), pages)
    assert torch.equal(pages.exponents.cpu().long(), ref_fields)
    assert torch.equal(pages.codes.cpu().double(), ref_codes)
    for out_dtype in DTYPES:
        out = torch.empty(codes.shape, dtype=out_dtype, device="cuda")
        assert torch.equal(K.kv8_values(pages, out).cpu().double(), values8(ref_codes, ref_fields))


@pytest.mark.parametrize("ps", [16, 64])
def test_however_a_prompt_is_cut_the_pages_hold_the_same_bits(K, ps):
    from infurnace_b200.kernels import Kv8Pages
    n, heads, dim = 150, 2, 64
    k, v = tokens_of(n, heads, dim, 5, torch.bfloat16)
    slots = torch.arange(n, dtype=torch.int32).cuda()
    k, v, held = k.cuda(), v.cuda(), []
    for cuts in ([n], [1] * n, [7, 30, 1, 90, 22], [75, 75]):
        pages = Kv8Pages.empty(-(-n // ps), heads, ps, dim)
        pages.exponents.fill_(200)                     # what another request left
        at = 0
        for m in cuts:
            K.kv8_store(k[at:at + m], v[at:at + m], slots[at:at + m], pages)
            at += m
        held.append((pages.exponents.clone(), pages.codes.view(-1, heads, ps, dim).clone()))
    for exponents, codes in held[1:]:
        assert torch.equal(exponents, held[0][0])
        assert torch.equal(codes, held[0][1])


@pytest.mark.parametrize("dtype", DTYPES)
def test_zeros_infinities_nan_and_the_ends_of_the_range(K, dtype):
    """A block of zeros is zero until a number joins it; an infinity or NaN makes its block NaN and no other; huge and tiny numbers."""
    heads, ps, dim = 3, 16, 16
    k, v = torch.zeros((6, heads, dim)), torch.zeros((6, heads, dim))
    k[3, 1], v[2, 0, 3], v[4, 2, 0] = 0.7, math.inf, math.nan
    k[:, 2] = torch.tensor([3.0e38, 1e-30, -1e-30, 2.0 ** 100, -3.0e38, -2.0 ** -126])[:, None]
    v[:, 1] = torch.tensor([2.0 ** -126, -2.0 ** -126, 2.0 ** -124, -2.0 ** -125, 0.0, 2.0 ** -121])[:, None]
    k, v = k.to(dtype), v.to(dtype)
    for cut in ([6], [1] * 6):
        pages = on_device(*pages_of(1, heads, ps, dim, 1))
        codes, fields = pages.codes.cpu(), pages.exponents.cpu()
        at = 0
        for m in cut:
            K.kv8_store(k[at:at + m].cuda(), v[at:at + m].cuda(), torch.arange(at, at + m, dtype=torch.int32).cuda(), pages)
            at += m
        ref_codes, ref_fields = store8(codes, fields, k, v, torch.arange(6))
        assert torch.equal(pages.exponents.cpu().long(), ref_fields)
        out = torch.empty(codes.shape, dtype=torch.float32, device="cuda")
        K.kv8_values(pages, out)
        assert same(out.cpu().double()[:, :, :, :6], values8(ref_codes, ref_fields)[:, :, :, :6])
        assert (out[0, 0, 0] == 0).all() and out[0, 1, 0].isnan().all() and out[0, 1, 2].isnan().all()


def test_keys_and_values_of_a_fused_row(K):
    """Views into rows of q | k | v."""
    n, heads, dim, width = 20, 2, 64, 5 * 64 + 2 * 64 * 2
    rows = torch.randn((n, width), device="cuda").to(torch.bfloat16)
    k, v = rows[:, 320:448].view(n, 2, 64), rows[:, 448:576].view(n, 2, 64)
    from infurnace_b200.kernels import Kv8Pages
    a, b = Kv8Pages.empty(2, heads, 16, dim), Kv8Pages.empty(2, heads, 16, dim)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    K.kv8_store(k, v, slots, a)
    K.kv8_store(k.contiguous(), v.contiguous(), slots, b)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.exponents, b.exponents)


# ------------------------------------------------------------------------------------------------ attention
def scene(q_lens, seq_lens, heads, group, dim, ps, dtype, seed=0, spare=0):
    """Queries and pages for requests with so many queries and keys; tables end in entries that must not be followed."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-n // ps) for n in seq_lens]
    codes, fields = pages_of(sum(held) + 1, heads, ps, dim, seed)
    order = torch.randperm(sum(held) + 1, generator=g)
    tables = torch.full((len(held), max(held + [1]) + spare), -1, dtype=torch.int32)
    at = 0
    for r, m in enumerate(held):
        tables[r, :m] = order[at:at + m]
        at += m
    cu = torch.tensor([0] + list(q_lens)).cumsum(0).to(torch.int32)
    q = (torch.randn((int(cu[-1]), heads * group, dim), generator=g) * 0.6).to(dtype)
    return q, codes, fields, tables, cu, torch.tensor(seq_lens, dtype=torch.int32)


def bound(ref, mag, reach, dim, keys, dtype):
    """What the kernel's roundings may add up to.  A score is a float32 sum of dim / 16 products of matrices whose numbers reach
    256 steps, each sum off by 2^-23 of that; its query is exact (bfloat16) or within 2^-21 (two halves).  A weight follows
    with twice the score's error, and has its own rounding: 2^-11 (half precision; 2^-21 with two) and 2^-20 for the
    exponential; the sums over the keys are float32; the output is rounded once (2^-9)."""
    score = reach * (dim / 16 * 2.0 ** -23 + (2.0 ** -21 if dtype == torch.float32 else 0))
    weight = (2.0 ** -20 if dtype == torch.float32 else 2.0 ** -10) + keys * 2.0 ** -23
    return (weight + 2 * score[..., None]) * mag + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22) * ref.abs() + 1e-30


def attend(K, q, codes, fields, tables, cu, lens, window, min_q=None, max_len=None):
    out = torch.full(q.shape, math.nan, dtype=q.dtype, device="cuda")
    q_lens = (cu[1:] - cu[:-1]).tolist()
    K.kv8_attention(q.cuda(), on_device(codes, fields), tables.cuda(), cu.cuda(), lens.cuda(), out, q.shape[2] ** -0.5, window,
                    max(q_lens), max_len or max(1, int(lens.max())), min_q_len=min_q or max(1, min(q_lens)))
    return out.cpu()


SCENES = [   # q_lens, seq_lens, kv heads, group, head size, page size, window
    ([1], [1], 1, 1, 16, 16, 0), ([1], [16], 2, 4, 128, 16, 0), ([1], [17], 2, 8, 128, 16, 0), ([1, 1, 1], [1, 500, 64], 2, 4, 128, 16, 0),
    ([1] * 9, [3, 700, 65, 64, 63, 1, 1000, 16, 15], 2, 2, 64, 32, 0), ([1, 1], [300, 900], 1, 5, 256, 64, 0), ([1, 1], [300, 900], 2, 16, 128, 16, 0),
    ([1, 1], [300, 900], 2, 4, 128, 16, 100), ([1, 1], [300, 900], 2, 3, 80, 48, 1), ([2, 1, 3], [40, 900, 3], 2, 8, 128, 16, 0),
    ([7, 5], [7, 300], 2, 4, 48, 16, 0), ([17], [117], 2, 4, 128, 16, 0), ([33, 1], [33, 77], 1, 2, 128, 16, 20), ([130], [130], 2, 4, 128, 16, 0),
    ([200, 1, 4], [500, 320, 4], 2, 2, 128, 32, 0), ([150, 90], [400, 90], 1, 8, 64, 16, 33), ([100], [333], 1, 5, 256, 16, 0), ([70], [70], 1, 32, 32, 16, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_lens,seq_lens,heads,group,dim,ps,window", SCENES)
def test_attention(K, dtype, q_lens, seq_lens, heads, group, dim, ps, window):
    s = scene(q_lens, seq_lens, heads, group, dim, ps, dtype, seed=len(q_lens) + dim + window)
    ref, mag, reach = attention8(*s, dim ** -0.5, window)
    out = attend(K, *s, window)
    assert (out.double() - ref).abs().le(bound(ref, mag, reach, dim, max(seq_lens), dtype)).all()
    assert torch.equal(out, attend(K, *s, window))                      # the same bits every time


@pytest.mark.parametrize("form,dtype", [("tiles", torch.bfloat16), ("whole", torch.bfloat16), ("whole", torch.float32), ("split", torch.bfloat16), ("split", torch.float32)])
@pytest.mark.parametrize("q_lens,seq_lens,heads,group,dim,ps,window", [s for s in SCENES if max(s[0]) * s[3] > 16] + [([700, 3], [700, 1100], 2, 4, 64, 64, 0)])
def test_every_form_of_attention(K, monkeypatch, form, dtype, q_lens, seq_lens, heads, group, dim, ps, window):
    """The three forms give way to one another by how much work there is; each is right for all of it, blocks of NaN included."""
    monkeypatch.setattr(K, "kv8_split_rows", (0, 0) if form == "tiles" else (1 << 20, 0))
    monkeypatch.setattr(K, "kv8_whole_rows", 0 if form == "whole" else 1 << 20)
    s = scene(q_lens, seq_lens, heads, group, dim, ps, dtype, seed=len(q_lens) + dim + window)
    ref, mag, reach = attention8(*s, dim ** -0.5, window)
    out = attend(K, *s, window)
    assert (out.double() - ref).abs().le(bound(ref, mag, reach, dim, max(seq_lens), dtype)).all()
    q, codes, fields, tables, cu, lens = s
    fields[tables[0, (seq_lens[0] - 1) // ps], 1, 0] = 255               # the last page of the first request, its first key head
    bad = attend(K, *s, window)
    for t in range(q.shape[0]):
        sees = t < q_lens[0] and seq_lens[0] - q_lens[0] + t >= (seq_lens[0] - 1) // ps * ps
        assert bad[t, :group].isnan().all() if sees else torch.equal(bad[t, :group], out[t, :group])
        assert torch.equal(bad[t, group:], out[t, group:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_requests_without_keys_or_queries_and_long_bounds(K, dtype):
    """A padded row (length 0) is zero, a request that brings nothing is passed over, the caller's bounds may exceed the lengths."""
    s = scene([1, 0, 1, 1], [0, 40, 70, 0], 2, 4, 128, 16, dtype, seed=4, spare=20)
    ref, mag, reach = attention8(*s, 128 ** -0.5)
    out = attend(K, *s, 0, min_q=1, max_len=300)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    assert (out.double() - ref).abs().le(bound(ref, mag, reach, 128, 70, dtype)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("requests", [40, 70, 150, 400])
def test_many_requests(K, dtype, requests):
    """More requests than a warp looks at once, than it keeps, and more items than CTAs run at a time; none, one and several pieces."""
    g = torch.Generator().manual_seed(requests)
    lens = torch.randint(0, 60, (requests,), generator=g).tolist()
    lens[requests // 2] = 700
    s = scene([1] * requests, lens, 2, 2, 64, 16, dtype, seed=requests)
    ref, mag, reach = attention8(*s, 64 ** -0.5)
    out = attend(K, *s, 0, min_q=1)
    assert (out.double() - ref).abs().le(bound(ref, mag, reach, 64, 700, dtype)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len", [1, 100])
def test_pages_far_into_a_large_pool(K, dtype, q_len):
    """Codes that begin beyond 2^31 and 2^32 bytes: the store, the values that are read back by attention, prompts and single tokens."""
    from infurnace_b200.kernels import Kv8Pages
    ps, heads, dim = 64, 8, 128                                        # 128 KB a page
    n = (1 << 32) // (2 * heads * ps * dim) + 8
    pages = Kv8Pages(torch.zeros((n, 2, heads, ps, dim), dtype=torch.int8, device="cuda"), torch.zeros((n, 2, heads), dtype=torch.uint8, device="cuda"))
    ids = torch.tensor([n - 1, n // 2 + 3, n - 5])                      # of the keys 0 .. 149
    k, v = tokens_of(150, heads, dim, 21, dtype)
    pos = torch.arange(150)
    slots = ids[pos // ps] * ps + pos % ps
    K.kv8_store(k.cuda(), v.cuda(), slots.to(torch.int32).cuda(), pages)
    small, fields = pages.codes[ids.cuda()].cpu(), pages.exponents[ids.cuda()].cpu()
    ref_codes, ref_fields = store8(torch.zeros_like(small), torch.zeros_like(fields), k, v, pos)
    assert torch.equal(fields.long(), ref_fields) and torch.equal(small.double(), ref_codes)
    q = (torch.randn((q_len, heads * 2, dim), generator=torch.Generator().manual_seed(1)) * 0.6).to(dtype)
    cu, lens = torch.tensor([0, q_len], dtype=torch.int32), torch.tensor([150], dtype=torch.int32)
    out = torch.empty(q.shape, dtype=dtype, device="cuda")
    K.kv8_attention(q.cuda(), pages, ids[None].to(torch.int32).cuda(), cu.cuda(), lens.cuda(), out, dim ** -0.5, 0, q_len, 150, min_q_len=q_len)
    ref, mag, reach = attention8(q, small, fields, torch.tensor([[0, 1, 2]]), cu, lens, dim ** -0.5)
    assert (out.cpu().double() - ref).abs().le(bound(ref, mag, reach, dim, 150, dtype)).all()


def test_pages_that_a_window_has_passed_are_not_followed(K):
    q, codes, fields, tables, cu, lens = scene([1, 5], [800, 600], 2, 4, 128, 16, torch.bfloat16, seed=6)
    ref, mag, reach = attention8(q, codes, fields, tables, cu, lens, 128 ** -0.5, 50)
    tables[0, :(800 - 50) // 16] = -1
    tables[1, :(595 - 49) // 16] = -1
    out = attend(K, q, codes, fields, tables, cu, lens, 50)
    assert (out.double() - ref).abs().le(bound(ref, mag, reach, 128, 800, torch.bfloat16)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_len,seq", [(1, 200), (40, 200), (150, 200)])
def test_a_block_of_nan_is_seen_by_the_rows_that_see_it_only(K, dtype, q_len, seq):
    """Keys or values of a page become NaN: rows that see none of its keys keep their bits, the others of that key head are NaN."""
    s = scene([q_len], [seq], 2, 2, 128, 16, dtype, seed=8)
    q, codes, fields, tables, cu, lens = s
    window = 30
    clean = attend(K, *s, window)
    for kind in (0, 1):
        bad = fields.clone()
        bad[tables[0, 165 // 16], kind, 1] = 255
        out = attend(K, q, codes, bad, tables, cu, lens, window)
        for t in range(q_len):
            p = seq - q_len + t
            sees = p >= 160 and p - window + 1 <= 175
            assert torch.equal(out[t, :2], clean[t, :2])
            assert out[t, 2:].isnan().all() if sees else torch.equal(out[t, 2:], clean[t, 2:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_every_size(K, dtype):
    """One key far above all others, scores of thousands, queries of 1e-20 and 1e20, values of very uneven size."""
    q, codes, fields, tables, cu, lens = scene([1, 1, 1], [300, 300, 300], 1, 4, 128, 16, dtype, seed=9)
    q[0] *= 300.0
    q[1] *= 1e-20
    q[2, 0] *= 1e20
    q[2, 0, 1:] = 0
    fields[tables[2].long(), 1] = torch.arange(fields.shape[0])[tables[2].long(), None].to(torch.uint8) * 3 + 90
    ref, mag, reach = attention8(q, codes, fields, tables, cu, lens, 128 ** -0.5)
    out = attend(K, q, codes, fields, tables, cu, lens, 0)
    b = bound(ref, mag, reach, 128, 300, dtype)
    assert out.isfinite().all()
    for t in (1, 2):       # scores of 1e18: one key has all the weight whatever their rounding
        assert (out[t].double() - ref[t]).abs().le(b[t].nan_to_num(math.inf)).all()
    # scores in the thousands: the winner of each row is the same wherever it leads by more than the rounding of two scores
    lead = out[0].double() - ref[0]
    assert (lead.abs() <= b[0]).all()


def test_strided_queries_another_stream_and_a_graph(K):
    q, codes, fields, tables, cu, lens = scene([1, 1, 1], [700, 90, 300], 2, 4, 128, 16, torch.bfloat16, seed=10)
    pages = on_device(codes, fields)
    wide = torch.randn((3, 2000), device="cuda").to(torch.bfloat16)
    wide[:, 64:64 + 1024] = q.cuda().view(3, 1024)
    view = wide[:, 64:64 + 1024].view(3, 8, 128)
    args = (pages, tables.cuda(), cu.cuda(), lens.cuda())
    plain = attend(K, q, codes, fields, tables, cu, lens, 0)
    outs = [torch.zeros((3, 8, 128), dtype=torch.bfloat16, device="cuda") for _ in range(3)]

    def call(out):
        K.kv8_attention(view, *args, out, 128 ** -0.5, 0, 1, 700)
    call(outs[0])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        call(outs[1])
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(outs[2])
    g.replay()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o.cpu(), plain) for o in outs)


def test_a_recording_outlives_larger_calls(K):
    """A graph recorded before a call that needs more room gives its bits afterwards."""
    s = scene([1, 1], [700, 300], 2, 4, 128, 16, torch.bfloat16, seed=12)
    q, codes, fields, tables, cu, lens = s
    plain = attend(K, *s, 0)
    pages, out, held = on_device(codes, fields), torch.zeros(q.shape, dtype=q.dtype, device="cuda"), [t.cuda() for t in (q, tables, cu, lens)]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.kv8_attention(held[0], pages, *held[1:], out, 128 ** -0.5, 0, 1, 700)
    many = 3000
    big = scene([1] * many, [33] * many, 2, 4, 128, 16, torch.bfloat16, seed=13)
    attend(K, *big, 0)
    junk = [torch.full((1 << 18,), 7, dtype=torch.int32, device="cuda") for _ in range(64)]      # over whatever was freed
    g.replay()
    torch.cuda.synchronize()
    assert len(junk) == 64 and torch.equal(out.cpu(), plain)


def test_refusals(K):
    from infurnace_b200.errors import KernelError
    from infurnace_b200.kernels import Kv8Pages
    q, codes, fields, tables, cu, lens = (t.cuda() for t in scene([2], [40], 2, 2, 64, 16, torch.bfloat16))
    pages, out = Kv8Pages(codes, fields), torch.empty_like(q)
    k = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.zeros(2, dtype=torch.int32, device="cuda")
    go = lambda q=q, t=tables, cu=cu, sl=lens, out=out, w=0, mq=2, ml=40, nq=1: K.kv8_attention(q, pages, t, cu, sl, out, 0.1, w, mq, ml, min_q_len=nq)  # noqa: E731
    go()
    for call in (lambda: Kv8Pages.empty(2, 2, 8, 64), lambda: Kv8Pages.empty(2, 2, 24, 64), lambda: Kv8Pages.empty(2, 2, 16, 272),
                 lambda: Kv8Pages.empty(2, 2, 16, 24), lambda: K.kv8_store(k.half(), k.half(), slots, pages),
                 lambda: K.kv8_store(k, k.float(), slots, pages), lambda: K.kv8_store(k[:, :1], k[:, :1], slots, pages),
                 lambda: K.kv8_store(k, k, slots.long(), pages), lambda: K.kv8_store(k, k, slots[:1], pages),
                 lambda: K.kv8_store(k.transpose(0, 1), k, slots, pages), lambda: K.kv8_store(k.cpu(), k, slots, pages),
                 lambda: K.kv8_values(pages, torch.empty((1, 2), device="cuda")), lambda: K.kv8_values(pages, codes),
                 lambda: go(q=q.half()), lambda: go(q=q.float()), lambda: go(q=q[:, :3], out=out[:, :3].contiguous()), lambda: go(out=out[:1]),
                 lambda: go(t=tables.long()), lambda: go(cu=cu[:1]), lambda: go(ml=200), lambda: go(w=-1), lambda: go(nq=3), lambda: go(mq=0),
                 lambda: go(sl=lens.cpu()), lambda: go(t=tables[:0]), lambda: go(q=q[0], out=out[0]), lambda: go(q=q[:, 0], out=out[:, 0].contiguous()),
                 lambda: K.kv8_store(k[0], k[0], slots[:1], pages), lambda: K.kv8_store(k[:, :, :, None], k[:, :, :, None], slots, pages)):
        with pytest.raises(KernelError):
            call()
