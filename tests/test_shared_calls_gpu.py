"""Attention over shared pages where the calls' own numbers end: pools beyond 32 bits, groups of nobody, requests ahead of the first group."""
import pytest
import torch

from test_shared_prefix_gpu import K, Scene      # noqa: F401 (K: a fixture)

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim,page,tokens", [(128, 16, 1), (128, 16, 40), (64, 64, 3), (80, 16, 5), (256, 16, 20)])
def test_a_pool_whose_places_pass_32_bits(K, dim, page, tokens, dtype):      # noqa: F811
    s = Scene([(150, [(150 + tokens, tokens), (300, tokens)])], alone=[(140, tokens)], dim=dim, page=page, dtype=dtype, seed=81)
    each = s.pages[0].numel()
    pages = (1 << 32) // each + 3                        # 2^32 elements and some
    if pages * each * s.pages.element_size() > torch.cuda.mem_get_info()[0] // 2:
        pytest.skip("not enough memory")
    pool = torch.empty((pages, *s.pages.shape[1:]), dtype=dtype, device="cuda")
    order = torch.randperm(len(s.pages), generator=torch.Generator().manual_seed(82))
    # places around 2^31 and 2^32 elements, at both ends and in between
    ids = torch.cat((torch.arange(2), (1 << 31) // each + torch.arange(-2, 3), torch.linspace(5, pages - 12, len(order)).long(), pages - 1 - torch.arange(4)))
    ids = ids.unique()[-len(order):][order]
    pool[ids.cuda()] = s.pages.cuda()
    tables = torch.where(s.tables < 0, -1, ids[s.tables.clamp(min=0).long()].int())
    s.check(s.run(K, kv_pages=pool, block_tables=tables.cuda()))
    K.check_device_errors()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("groups", [
    [(32, []), (48, [(50, 1), (60, 2)]), (16, [])], [(0, []), (0, []), (33, [(40, 30), (35, 1)])], [(48, [(50, 1)]), (16, []), (16, [(17, 1), (40, 1)])]])
def test_groups_of_nobody(K, groups, dtype):      # noqa: F811
    s = Scene(groups, alone=[(20, 2)], dtype=dtype, seed=83)
    s.check(s.run(K))
    K.check_device_errors()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 144])
def test_requests_ahead_of_the_first_group_share_nothing(K, dim, dtype):      # noqa: F811
    s = Scene([(0, [(30, 1), (100, 20)]), (64, [(70, 1), (90, 25), (65, 1)]), (20, [(21, 1), (40, 1)])], alone=[(33, 3)], dim=dim, dtype=dtype, seed=84)
    skip = s.cu_groups[1]
    one = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    s.check(s.run(K, cu_groups=one(s.cu_groups[1:]), shared_lens=one(s.shared[1:])))
    assert skip == 2
    K.check_device_errors()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_ahead_of_the_first_request_stay(K, dtype):      # noqa: F811
    """As those behind the last one do."""
    s = Scene([(64, [(70, 1), (90, 25)])], alone=[(33, 3)], dtype=dtype, seed=85, rows_behind=2)
    d = s.device()
    q = torch.cat((torch.full_like(d["q"][:4], float("nan")), d["q"]))
    out = s.run(K, q=q, cu_q=d["cu_q"] + 4)
    assert (out[:4] == 7.0).all()
    s.check(out[4:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_two_recordings_that_run_at_once(K, dtype):      # noqa: F811
    """Each has a room of its own in its graph's memory."""
    scenes = [Scene([(160, [(163, 1), (230, 3), (161, 1)]), (32, [(40, 1)])], dtype=dtype, seed=86 + i) for i in range(2)]
    held, outs, graphs, streams = [], [], [], [torch.cuda.Stream() for _ in scenes]
    for s in scenes:
        d = s.device()
        out = torch.full_like(d["q"], 7.0)
        call = lambda d=d, out=out, s=s: K.shared_prefix_attention(d["q"], d["kv_pages"], d["block_tables"], d["cu_q"], d["seq_lens"], d["cu_groups"],
                                                                    d["shared_lens"], out, s.scale, 0, 3, max(s.lens))
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
            call()
        held.append(d); outs.append(out); graphs.append(graph)
    alone = [s.run(K) for s in scenes]
    torch.cuda.synchronize()
    for _ in range(30):
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for out, want in zip(outs, alone):
        assert torch.equal(out, want)
