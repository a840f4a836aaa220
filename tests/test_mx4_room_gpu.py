"""The room in which products with 4-bit matrices round their rows: one for an engine's matrices and for all of its recordings."""
import json
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


def test_recordings_of_an_engine_share_the_room(K):
    """Portions of twelve lengths, each recorded: the rows of a product of 12,288 numbers are 500 x 6.5 KB."""
    from infurnace_b200.engine import Engine, EngineOptions, StepEntry
    with open(os.path.join(ROOT, "configs", "qwen3-8b.json"), encoding="utf-8") as f:
        cfg = dict(json.load(f), num_hidden_layers=1, vocab_size=2048)
    runner = Engine.from_random(cfg, 5, EngineOptions(dtype="bfloat16", device="cuda", num_pages=1536, max_num_seqs=4, max_num_batched_tokens=1024,
                                                      max_model_len=24576, weight_format="mx4")).runner
    rooms = {w.room.data_ptr() for layer in runner.model.layers for w in (layer.mixer.w_qkv, layer.mixer.w_o, layer.ffn.w_gate_up, layer.ffn.w_down)}
    assert len(rooms) == 1
    runner.cache.add_request("r")
    for _ in range(3):
        runner.step([StepEntry("r", [5] * 1000)])
    for i, n in enumerate(range(500, 512)):
        for _ in range(3):                         # (a shape is another one where the context passes a power of two)
            if not any(key[1] == n for key in runner._graphs):
                runner.step([StepEntry("r", [5] * n)])
        if i == 1:
            torch.cuda.synchronize()
            before = torch.cuda.memory_reserved()
    K.check_device_errors()
    assert len(runner._graphs) == 12
    assert torch.cuda.memory_reserved() - before <= 64 << 20


@pytest.mark.parametrize("rows,k,features", [(40, 512, 300), (300, 1120, 258), (1100, 288, 6500)])
def test_products_in_a_room(K, rows, k, features):
    """The same bits as without one, in a room that holds something else and just suffices, and where it does not; recorded too."""
    from infurnace_b200.kernels import Mx4Matrix
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, w = (torch.randn((n, k), generator=g, device="cuda").to(torch.bfloat16) for n in (rows, features))
    m = K.mx4_matrix(w)
    plain, roomy, short, recorded = (torch.empty((rows, features), device="cuda") for _ in range(4))
    K.mx4_linear(x, m, plain)
    size = Mx4Matrix.row_bytes(rows, k)
    around = torch.full((size + 256,), 255, dtype=torch.uint8, device="cuda")
    m.room = around[:size]
    K.mx4_linear(x, m, roomy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.mx4_linear(x, m, recorded)
    around[:size] = 255
    graph.replay()
    assert (around[size:] == 255).all() and not (around[:size] == 255).all()
    m.room = around[:size - 256]
    K.mx4_linear(x, m, short)
    K.check_device_errors()
    assert torch.equal(roomy, plain) and torch.equal(short, plain) and torch.equal(recorded, plain)


def test_rooms_that_are_refused(K):
    from infurnace_b200.errors import KernelError
    m = K.mx4_matrix(torch.zeros((4, 64), device="cuda"))
    room = torch.empty(4096, dtype=torch.uint8, device="cuda")
    for bad in (room.view(torch.int32), room[1:], room.view(2, -1), room[::2], room.cpu()):
        with pytest.raises(KernelError):
            m.room = bad
    m.room = room
    m.room = None
