"""The room in which attention over 8-bit pages lays out the pages that it expands for prompts: one for an engine's layers and for all of
its recordings, no larger than the pool asks for, and another form where it does not suffice."""
import json
import os

import pytest
import torch

from low_bit_refs import attention8
from test_kv8_gpu import bound, on_device, scene

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


def recorded_growth(record, shapes):
    """Bytes that the device's memory grew by from the second of some recordings to the last."""
    graphs = []
    for i, shape in enumerate(shapes):
        graphs.append(record(shape))
        if i == 1:
            torch.cuda.synchronize()
            before = torch.cuda.memory_reserved()
    return torch.cuda.memory_reserved() - before, graphs


def test_recordings_of_an_engine_share_the_room():
    """Portions of many lengths of a long prompt, each recorded: a layer's expanded pages are 30,000 tokens' 123 MB."""
    from infurnace_b200.engine import Engine, EngineOptions, StepEntry
    with open(os.path.join(ROOT, "configs", "qwen3-0.6b.json"), encoding="utf-8") as f:
        cfg = dict(json.load(f), num_hidden_layers=2)
    eng = Engine.from_random(cfg, 5, EngineOptions(dtype="bfloat16", device="cuda", num_pages=1900, max_num_seqs=4, max_num_batched_tokens=2048,
                                                   max_model_len=30000, cache_format="int8"))
    runner = eng.runner
    runner.cache.add_request("r")
    for _ in range(8):
        runner.step([StepEntry("r", [7] * 2048)])
    k = runner.rt.kernels
    calls = k.tc_attention_calls

    def record(n):
        held = len(runner._graphs)
        for _ in range(2):
            runner.step([StepEntry("r", [5] * n)])
        assert len(runner._graphs) == held + 1
    grown, _ = recorded_growth(record, range(500, 512))
    k.check_device_errors()
    assert k.tc_attention_calls > calls
    assert grown <= 64 << 20


def prompts(K, room=None, shared=True, dim=128, many=62):
    """Two prompts of 300 and 200 queries between ``many`` - 2 decoding requests of up to 600 keys."""
    q_lens = [1] * many
    q_lens[3], q_lens[many // 2] = 300, 200
    lens = [300 + 41 * r % 301 for r in range(many)]
    s = scene(q_lens, lens, 2, 4, dim, 16, torch.bfloat16, seed=many)
    q, codes, fields, tables, cu, seq = s
    pages = on_device(codes, fields)
    pages.room, pages.shared = room, shared
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    before = K.tc_attention_calls
    K.kv8_attention(q.cuda(), pages, tables.cuda(), cu.cuda(), seq.cuda(), out, dim ** -0.5, 0, 300, 601, exact_lens=True)
    K.check_device_errors()
    return s, out.cpu(), K.tc_attention_calls - before


@pytest.mark.parametrize("dim", [64, 128])
def test_prompts_among_a_full_batch(K, monkeypatch, dim):
    """On the tcgen05 form with and without a room, and on the others where a room or the bound is too small."""
    from infurnace_b200.kernels.low_bits import kv8_room_bytes
    monkeypatch.setattr(K, "kv8_split_rows", (0, 0))
    s, out, tc = prompts(K, dim=dim)
    ref, mag, reach = attention8(*s, dim ** -0.5)
    limit = bound(ref, mag, reach, dim, 600, torch.bfloat16)
    assert tc == 1 and (out.double() - ref).abs().le(limit).all()
    size = kv8_room_bytes(s[1].shape[0], 62, 38, 2, 16, dim, torch.bfloat16)
    room = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    _, again, tc = prompts(K, room, shared=False, dim=dim)
    assert tc == 1 and torch.equal(out, again)
    _, small, tc = prompts(K, room[:size - 256 * 62], shared=False, dim=dim)
    assert tc == 0 and (small.double() - ref).abs().le(limit).all()
    monkeypatch.setattr(K, "kv8_expand_bytes", 1 << 20)
    _, small, tc = prompts(K, dim=dim)
    assert tc == 0 and (small.double() - ref).abs().le(limit).all()


@pytest.mark.parametrize("window", [0, 40, 500])
def test_a_room_of_just_the_pages_that_are_seen(K, monkeypatch, window):
    """Three prompts behind windows: the places of expanded pages count what a request's queries see."""
    from infurnace_b200.kernels.low_bits import kv8_room_bytes
    monkeypatch.setattr(K, "kv8_split_rows", (0, 0))
    q_lens, lens = [90, 1, 60, 130], [700, 300, 801, 130]
    q, codes, fields, tables, cu, seq = scene(q_lens, lens, 2, 4, 128, 16, torch.bfloat16, seed=window)
    ref, mag, reach = attention8(q, codes, fields, tables, cu, seq, 128 ** -0.5, window)
    # a pool of the pages that are seen, as an engine has it behind a window
    kept, moved = [], torch.full_like(tables, -1)
    for r in range(4):
        for p in range(max(0, lens[r] - q_lens[r] - window + 1) // 16 if window else 0, -(-lens[r] // 16)):
            moved[r, p] = len(kept)
            kept.append(int(tables[r, p]))
    pages = on_device(codes[kept], fields[kept])
    pages.shared = False
    pages.room = torch.full((kv8_room_bytes(len(kept), 4, 51, 2, 16, 128, torch.bfloat16),), 255, dtype=torch.uint8, device="cuda")
    out = torch.full(q.shape, float("nan"), dtype=q.dtype, device="cuda")
    before = K.tc_attention_calls
    K.kv8_attention(q.cuda(), pages, moved.cuda(), cu.cuda(), seq.cuda(), out, 128 ** -0.5, window, 130, 801)
    K.check_device_errors()
    assert K.tc_attention_calls == before + 1
    assert (out.cpu().double() - ref).abs().le(bound(ref, mag, reach, 128, 801, torch.bfloat16)).all()


def test_recorded_calls_in_a_room(K, monkeypatch):
    """Graphs of several shapes over one room take no memory for expanded pages, and replay to the bits of calls."""
    monkeypatch.setattr(K, "kv8_split_rows", (0, 0))
    n = 6000
    q, codes, fields, tables, cu, seq = scene([n // 40], [n], 8, 2, 128, 16, torch.bfloat16, seed=2)
    pages = on_device(codes, fields)
    pages.shared = False
    pages.room = torch.empty(n // 16 * 65536 + 4096 * 4, dtype=torch.uint8, device="cuda")
    tables, q = tables.cuda(), q.cuda()

    def call(m, out):
        K.kv8_attention(q[:m], pages, tables, torch.tensor([0, m], dtype=torch.int32, device="cuda") if m not in held else held[m],
                        seqs, out, 128 ** -0.5, 0, m, n, min_q_len=m)
    held, seqs, outs = {}, seq.cuda(), {}

    def record(m):
        held[m] = torch.tensor([0, m], dtype=torch.int32, device="cuda")
        plain, outs[m] = (torch.zeros((m, 16, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        call(m, plain)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(m, outs[m])
        return m, plain, g
    grown, graphs = recorded_growth(record, range(100, 112))
    for m, plain, g in graphs + graphs[:3]:
        outs[m].zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[m], plain)
    K.check_device_errors()
    assert grown <= 30 << 20                                           # (one call's expanded pages: 24 MB)


def test_rooms_that_are_refused(K, monkeypatch):
    from infurnace_b200.errors import KernelError
    monkeypatch.setattr(K, "kv8_split_rows", (0, 0))
    room = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    for bad in (room.view(torch.int32), room[1:], room.view(2, -1), room[::2], room.cpu()):
        with pytest.raises(KernelError):
            prompts(K, bad)
