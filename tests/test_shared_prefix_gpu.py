"""Attention over pages that requests share, on the device, against each request by itself in 64 bits (tests/answer_refs.py)."""
import math

import pytest
import torch

from answer_refs import attention

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


class Scene:
    """Requests in groups with pages of their own and shared ones, everything that no query sees being NaN.

    ``groups``: a list of (shared keys, [(keys in all, queries), ...]); ``alone``: requests of no group, behind them."""

    def __init__(self, groups, alone=(), page=16, kv_heads=2, group=2, dim=64, window=0, dtype=torch.bfloat16, seed=0, spread=1.0, rows_behind=0):
        g = torch.Generator().manual_seed(seed)
        self.window, self.dtype, self.scale, self.page = window, dtype, dim ** -0.5, page
        requests = [x for _, members in groups for x in members] + list(alone)
        self.lens = [x[0] for x in requests]
        self.cu_q = [0]
        for _, q in requests:
            self.cu_q.append(self.cu_q[-1] + q)
        self.cu_groups = [0]
        for _, members in groups:
            self.cu_groups.append(self.cu_groups[-1] + len(members))
        self.shared = [x[0] for x in groups]
        width = max([-(-n // page) for n in self.lens] + [-(-n // page) for n in self.shared] + [1]) + 1
        need = sum(-(-n // page) + 1 for n in self.lens) + sum(-(-n // page) for n in self.shared) + 2
        order = torch.randperm(need, generator=g).tolist()
        self.tables = torch.full((len(requests), width), -1, dtype=torch.int32)
        self.pages = torch.full((need, 2, kv_heads, page, dim), math.nan)

        def fill(r, lo, hi):
            for i in range(lo, hi):
                if self.tables[r, i // page] < 0:
                    self.tables[r, i // page] = order.pop()
                self.pages[int(self.tables[r, i // page]), :, :, i % page] = spread * torch.randn((2, kv_heads, dim), generator=g)

        for r, n in enumerate(self.lens):
            j = next((j for j in range(len(groups)) if self.cu_groups[j] <= r < self.cu_groups[j + 1]), None)
            first = j is not None and self.cu_groups[j] == r
            if first:
                fill(r, 0, self.shared[j])
            fill(r, 0 if j is None else self.shared[j], n)      # (the others' entries for what they share stay -1)
        self.rows = self.cu_q[-1] + rows_behind
        self.q = torch.randn((self.rows, kv_heads * group, dim), generator=g).to(dtype)
        self.pages = self.pages.to(dtype)

    def device(self):
        one = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
        return dict(q=self.q.cuda(), kv_pages=self.pages.cuda(), block_tables=self.tables.cuda(), cu_q=one(self.cu_q), seq_lens=one(self.lens),
                    cu_groups=one(self.cu_groups), shared_lens=one(self.shared))

    def run(self, K, room=None, **other):
        d = {**self.device(), **other}
        out = torch.full_like(d["q"], 7.0) if "out" not in d else d.pop("out")
        most = max(b - a for a, b in zip(self.cu_q, self.cu_q[1:]))
        K.shared_prefix_attention(d["q"], d["kv_pages"], d["block_tables"], d["cu_q"], d["seq_lens"], d["cu_groups"], d["shared_lens"], out, self.scale,
                                  self.window, max(1, most), max(self.lens + self.shared), room=room)
        return out

    def check(self, out):
        want, size = attention(self.q[:self.cu_q[-1]].float(), self.pages.float(), self.tables, self.cu_q, self.lens, self.cu_groups, self.shared, self.scale,
                               self.window)
        got = out[:self.cu_q[-1]].double().cpu()
        dim = self.q.shape[2]
        # Scores: dim products of float32, each sum off by at most dim 2^-24 |q| |k| scale (inputs are exact); as the exponent of a weight in a
        # numerator and a denominator that counts twice.  Weights: exp2 and the rounding of its argument, 2^-21.  Sums over the keys, one after
        # the other at worst: keys 2^-24 each.  A weight in two bfloat16 terms keeps 16 bits: 2^-16.  The output: half a step of its type.
        finite = torch.nan_to_num(self.pages.float())
        norm = self.q.float().norm(dim=2).max() * finite[:, 0].norm(dim=3).max() * self.scale
        wide = 2 * dim * 2.0 ** -24 * norm + 2.0 ** -20 + 2 * max(self.lens) * 2.0 ** -24 + (2.0 ** -16 if self.dtype == torch.bfloat16 else 0.0)
        bound = float(wide) * size + torch.finfo(self.dtype).eps / 2 * want.abs()
        worst = ((got - want).abs() - bound).max().item()
        assert worst <= 0, worst
        assert (out[self.cu_q[-1]:] == 7.0).all()


SCENES = {
    "samples": dict(groups=[(160, [(163, 1), (170, 1), (161, 1), (200, 1)])]),
    "uneven": dict(groups=[(333, [(340, 1), (400, 1)]), (16, [(17, 1)] * 5), (1, [(2, 1), (90, 1)])], alone=[(70, 1), (1, 1)]),
    "inside-a-page": dict(groups=[(37, [(45, 1), (38, 1), (60, 2)]), (129, [(130, 1), (140, 1)])]),
    "nothing-shared": dict(groups=[(0, [(5, 1), (200, 1)]), (0, [(1, 1)])], alone=[(33, 4)]),
    "no-groups": dict(groups=[], alone=[(5, 1), (130, 1), (257, 1), (64, 30)]),
    "nothing-of-its-own": dict(groups=[(64, [(64, 1), (64, 1), (64, 3)])]),
    "questions": dict(groups=[(300, [(330, 30), (341, 41), (301, 1)]), (128, [(200, 72), (128, 2)])]),
    "full-tiles": dict(groups=[(208, [(330, 90), (208, 70), (200, 60), (209, 1)]), (37, [(150, 100), (120, 80)]), (64, [(64, 64)])], alone=[(130, 130)]),
    "full-tiles-window": dict(groups=[(208, [(330, 90), (208, 70), (200, 60), (209, 1)])], window=77, page=32),
    "empty-requests": dict(groups=[(48, [(50, 1), (0, 1), (49, 0), (51, 2)]), (20, [(0, 0)])], alone=[(0, 1), (3, 3)], rows_behind=5),
    "in-the-shared-part": dict(groups=[(200, [(200, 60), (150, 10), (260, 20)])]),
    "window": dict(groups=[(300, [(310, 1), (420, 1), (305, 5)]), (64, [(500, 1)])], alone=[(90, 40)], window=100),
    "window-of-one": dict(groups=[(40, [(41, 1), (42, 2), (80, 1)])], window=1),
    "window-in-the-middle": dict(groups=[(511, [(520, 1), (512, 1), (600, 8)])], window=250),
    "long": dict(groups=[(2500, [(2510, 1), (2600, 1), (2501, 1)])], kv_heads=1, group=3),
    "many": dict(groups=[(64, [(65 + i, 1) for i in range(70)])], kv_heads=1, group=2),
    "page-of-groups": dict(groups=[(32 + 16 * (i % 3), [(90, 1), (95 + i, 1)]) for i in range(20)], kv_heads=1, group=1),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", SCENES)
def test_requests_that_share_see_what_they_would_alone(K, name, dtype):
    s = Scene(dtype=dtype, **SCENES[name])
    s.check(s.run(K))
    K.check_device_errors()


# Keys that some rows of a tile see and others do not: what they hold may be anything for the others.
PARTLY_SEEN = {
    "questions": dict(groups=[(300, [(330, 30), (341, 41), (301, 1)])], group=4),
    "full-tiles": dict(groups=[(208, [(330, 90), (290, 70)])], group=2),
    "few-queries": dict(groups=[(48, [(55, 4), (60, 2), (49, 1)])], alone=[(20, 7), (3, 3)]),
    "window": dict(groups=[(300, [(310, 1), (420, 1), (305, 5), (330, 1)] * 5)], window=100, group=4),
    "few-in-a-window": dict(groups=[(300, [(310, 1), (340, 1), (305, 2)])], window=100),
    "a-short-one-in-a-group": dict(groups=[(200, [(230, 1), (120, 1), (160, 3), (220, 60)])]),
}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [64, 128, 80, 144])
@pytest.mark.parametrize("name", PARTLY_SEEN)
def test_what_other_rows_see_may_be_anything(K, name, dim, what, dtype):
    scene = Scene(**PARTLY_SEEN[name], dim=dim, dtype=dtype, seed=31)
    # the last keys of every request and the shared ones that the windows or lengths of some leave out, in some columns of the values
    for r, n in enumerate(scene.lens):
        j = next((j for j in range(len(scene.shared)) if scene.cu_groups[j] <= r < scene.cu_groups[j + 1]), None)
        for key, columns in ((n - 1, slice(3, 4)), (n - 2, slice(5, 20)), (n - scene.window - 2 if scene.window else n - 3, slice(dim - 1, dim))):
            if key >= 0:
                owner = scene.cu_groups[j] if j is not None and key < scene.shared[j] else r
                scene.pages[int(scene.tables[owner, key // scene.page]), 1, :, key % scene.page, columns] = what
    out = scene.run(K)
    want, _ = attention(scene.q[:scene.cu_q[-1]].float(), scene.pages.float(), scene.tables, scene.cu_q, scene.lens, scene.cu_groups, scene.shared, scene.scale,
                        scene.window)
    got = out[:scene.cu_q[-1]].double().cpu()
    assert (want.isfinite()).any() and not want.isfinite().all()
    assert (got.isfinite() == want.isfinite()).all()
    assert (got.isnan() == want.isnan()).all() and (got[want == math.inf] == math.inf).all() and (got[want == -math.inf] == -math.inf).all()
    # the finite ones: those of the same scene with zeros in those places, which none of their rows sees
    seen = want.isfinite()
    scene.pages = torch.nan_to_num(scene.pages, nan=0.0, posinf=0.0, neginf=0.0)
    plain, size = attention(scene.q[:scene.cu_q[-1]].float(), scene.pages.float(), scene.tables, scene.cu_q, scene.lens, scene.cu_groups, scene.shared,
                            scene.scale, scene.window)
    norm = scene.q.float().norm(dim=2).max() * scene.pages[:, 0].float().norm(dim=3).max() * scene.scale
    wide = 2 * dim * 2.0 ** -24 * norm + 2.0 ** -20 + 2 * max(scene.lens) * 2.0 ** -24 + (2.0 ** -16 if dtype == torch.bfloat16 else 0.0)      # as in check
    bound = float(wide) * size + torch.finfo(dtype).eps / 2 * plain.abs()
    assert (((got - plain).abs() - bound)[seen] <= 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 8, 16, 24, 32, 64, 128])
def test_pages_of_any_size(K, page, dtype):
    s = Scene([(100, [(103, 1), (190, 1)]), (page, [(page + 2, 2)])], alone=[(3 * page, 1)], page=page, dtype=dtype, seed=page)
    s.check(s.run(K))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 112, 128, 144, 192, 256])
def test_heads_of_any_size(K, dim, dtype):
    s = Scene([(150, [(153, 1), (300, 3)])], alone=[(140, 2)], dim=dim, dtype=dtype, seed=dim)
    s.check(s.run(K))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (3, 1), (8, 1), (1, 5), (2, 7), (1, 16), (1, 33), (1, 64), (4, 8)])
def test_groups_of_heads(K, kv_heads, group, dtype):
    s = Scene([(100, [(103, 1), (190, 5), (101, 1)])], kv_heads=kv_heads, group=group, dim=32 if group > 8 else 64, dtype=dtype, seed=group)
    s.check(s.run(K))


@pytest.mark.parametrize("dim,page", [(144, 16), (256, 24), (128, 24), (80, 128)])
@pytest.mark.parametrize("kv_heads,group", [(3, 1), (1, 5), (2, 7), (1, 16), (1, 17), (1, 64)])
@pytest.mark.parametrize("name", ["questions", "full-tiles-window", "uneven"])
def test_groups_of_heads_where_large_tiles_do_not_fit(K, name, kv_heads, group, dim, page):
    s = Scene(**{**SCENES[name], "kv_heads": kv_heads, "group": group, "dim": dim, "page": page}, seed=21)
    s.check(s.run(K))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,requests", [(64, 1100), (256, 480)])
def test_many_requests(K, dim, requests, dtype):
    """More than the plan of the large tiles' kernel has room for."""
    groups = [(40 + 16 * j, [(41 + 16 * j + i % 9, 1 + (i % 50 == 0)) for i in range(requests // 4)]) for j in range(3)]
    s = Scene(groups, alone=[(1 + i % 20, 1) for i in range(requests - 3 * (requests // 4))], kv_heads=1, group=2, dim=dim, dtype=dtype, seed=22)
    s.check(s.run(K))


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_any_size(K, dtype):
    """Rows with one weight that is all, and scores far beyond the exponents' range."""
    for spread, factor in ((1.0, 40.0), (30.0, 30.0), (1e-3, 1e-3)):
        s = Scene([(200, [(203, 1), (290, 1)])], dtype=dtype, spread=spread, seed=int(spread))
        s.q = (s.q.float() * factor).to(dtype)
        out = s.run(K)
        want, size = attention(s.q.float(), s.pages.float(), s.tables, s.cu_q, s.lens, s.cu_groups, s.shared, s.scale, 0)
        assert out.isfinite().all()
        if factor * spread < 1:
            s.check(out)
        else:
            # a score of size x is off by up to dim 2^-24 x, and weights by as much: what remains is a mean of the values that count
            norm = float(s.q.float().norm(dim=2).max() * torch.nan_to_num(s.pages.float())[:, 0].norm(dim=3).max() * s.scale)
            near = 2 * 64 * 2.0 ** -24 * norm
            if near < 0.5:
                assert ((out.double().cpu() - want).abs() <= (math.expm1(near) + torch.finfo(dtype).eps) * size).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_lie_apart_and_pages_that_lie_apart(K, dtype):
    s = Scene(**SCENES["questions"], dtype=dtype)
    d = s.device()
    n, heads, dim = s.q.shape
    wide = torch.full((n, heads * dim + 64), 9.0, dtype=dtype, device="cuda")
    wide[:, 32:32 + heads * dim] = d["q"].view(n, -1)
    q = wide[:, 32:32 + heads * dim].view(n, heads, dim)
    pool = torch.full((s.pages.shape[0], 2, *s.pages.shape[1:]), math.nan, dtype=dtype, device="cuda")
    pool[:, 1] = d["kv_pages"]
    tables = torch.full((s.tables.shape[0] + 2, s.tables.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    tables[:-2, :-3] = d["block_tables"]
    out = s.run(K, q=q, kv_pages=pool[:, 1], block_tables=tables[:, :-3])
    assert torch.equal(out, s.run(K))
    s.check(out)


def test_a_page_that_is_none_counts_as_zeros_and_is_recorded(K):
    from infurnace_b200.errors import KernelError
    for dtype in DTYPES:
        for bad in (-1, 1 << 30, -(1 << 31)):
            s = Scene([(64, [(70, 1), (90, 1)])], dtype=dtype)
            zeros = s.pages[int(s.tables[1, 5])]
            zeros.zero_()
            d = s.device()
            d["block_tables"][1, 5] = bad                            # keys 80 .. 89 of the second request
            out = s.run(K, block_tables=d["block_tables"])
            with pytest.raises(KernelError, match="no page of the pool"):
                K.check_device_errors()
            s.check(out)
    K.check_device_errors()


@pytest.mark.parametrize("dtype", DTYPES)
def test_bits_repeat_and_a_room_may_be_the_callers(K, dtype):
    s = Scene(**SCENES["uneven"], dtype=dtype)
    first = s.run(K)
    heads, dim = s.q.shape[1:]
    size = K.shared_prefix_room(s.rows, len(s.lens), len(s.shared), heads, 2, dim, dtype)
    room = torch.full((size,), 255, dtype=torch.uint8, device="cuda")              # NaN wherever it is read as numbers
    for _ in range(3):
        assert torch.equal(s.run(K, room=room), first)


@pytest.mark.parametrize("dtype", DTYPES)
def test_recorded_and_replayed_with_new_lengths_and_on_another_stream(K, dtype):
    a = Scene([(160, [(163, 1), (170, 1), (161, 1)]), (32, [(40, 1)])], dtype=dtype, seed=1)
    b = Scene([(96, [(130, 1), (97, 1), (150, 1)]), (48, [(170, 1)])], dtype=dtype, seed=2)
    width, pages = max(a.tables.shape[1], b.tables.shape[1]), max(a.pages.shape[0], b.pages.shape[0])

    def padded(s):
        d = s.device()
        tables = torch.full((4, width), -1, dtype=torch.int32, device="cuda")
        tables[:, :s.tables.shape[1]] = d["block_tables"]
        pool = torch.zeros((pages, *s.pages.shape[1:]), dtype=dtype, device="cuda")
        pool[:s.pages.shape[0]] = d["kv_pages"]
        return {**d, "block_tables": tables, "kv_pages": pool}

    held = padded(a)
    out = torch.full_like(held["q"], 7.0)

    def call():
        K.shared_prefix_attention(held["q"], held["kv_pages"], held["block_tables"], held["cu_q"], held["seq_lens"], held["cu_groups"], held["shared_lens"],
                                  out, a.scale, 0, 1, width * 16)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
        call()
    for s in (b, a, b):
        for name, t in padded(s).items():
            held[name].copy_(t)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        s.check(out)
        replayed = out.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        assert torch.equal(out, replayed)


def test_nothing_to_do(K):
    empty = lambda *shape, dtype=torch.int32: torch.zeros(shape, dtype=dtype, device="cuda")
    pages = empty(2, 2, 1, 16, 64, dtype=torch.bfloat16)
    out = empty(0, 2, 64, dtype=torch.bfloat16)
    K.shared_prefix_attention(out, pages, empty(0, 4), empty(1), empty(0), empty(1), empty(0), out, 1.0, 0, 1, 10)
    rows = torch.full((3, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")          # rows, but no request
    K.shared_prefix_attention(rows, pages, empty(0, 4), empty(1), empty(0), empty(1), empty(0), rows, 1.0, 0, 1, 10)
    assert (rows == 7.0).all()


def test_it_is_the_ordinary_attention_of_the_same_tables(K):
    """Beside ``paged_attention``, whose tables name the shared pages for every request."""
    s = Scene([(320, [(340, 1), (321, 1), (400, 1)]), (160, [(163, 1), (290, 1)])], dtype=torch.bfloat16, kv_heads=2, group=4, dim=128)
    d = s.device()
    pages = torch.nan_to_num(d["kv_pages"])
    tables = d["block_tables"].clone()
    for g, n in enumerate(s.shared):
        for r in range(s.cu_groups[g], s.cu_groups[g + 1]):
            tables[r, :n // 16] = tables[s.cu_groups[g], :n // 16]
    out = s.run(K, kv_pages=pages, block_tables=tables)
    s.check(out)
    ordinary = torch.empty_like(out)
    K.paged_attention(d["q"].view(5, -1), 8, 2, 128, pages, tables, d["cu_q"], d["seq_lens"], ordinary.view(5, -1), s.scale, 0, 1, 400)
    # both within their bounds of the same numbers: the ordinary kernel's weights have one bfloat16 term
    want, size = attention(s.q.float(), s.pages.float(), s.tables, s.cu_q, s.lens, s.cu_groups, s.shared, s.scale, 0)
    assert ((out.double() - ordinary.double()).abs().cpu() <= 2.0 ** -7 * size + 2.0 ** -6 * want.abs()).all()
