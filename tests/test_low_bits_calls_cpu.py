"""What the calls over few bits do on the host, without a GPU: rooms and launches under several threads."""
import threading
import time

import pytest
import torch

from infurnace_b200.kernels import low_bits
from infurnace_b200.kernels.low_bits import LowBitKernels, Mx4Matrix


class Rows:
    """What a call looks at of a tensor on a device."""
    dtype = torch.bfloat16

    def __init__(self, rows, width):
        self.shape, self.at = torch.Size((rows, width)), 4096

    def stride(self):
        return (self.shape[1], 1)

    def get_device(self):
        return 0

    def data_ptr(self):
        return self.at

    def is_contiguous(self):
        return True


class Library:
    """Stands for the products' library: notes when a call begins on a room that another call is at work in."""
    def __init__(self):
        self.at_work, self.broken, self.calls = [], 0, 0

    def ifb_mx4_linear(self, x, code, pitch, room, scales, *rest):
        self.broken += room in self.at_work
        self.at_work.append(room)
        time.sleep(0.003)
        self.at_work.remove(room)
        self.calls += 1
        return 0


class Kernels(LowBitKernels):
    _progress, launches, _dev_err_at, _epilogues = None, 0, 0, {"none": 0}
    _mx4_round_rows = {0: 16, 1: 32}

    def __init__(self, library):
        self.library = library

    def _mx4_lib(self):
        return self.library


@pytest.mark.parametrize("own", [False, True])
def test_threads_on_one_stream_do_not_share_a_room_at_a_time(monkeypatch, own):
    monkeypatch.setattr(low_bits, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(low_bits, "_capturing", lambda: False)
    library = Library()
    kernels = Kernels(library)
    w = Mx4Matrix.empty(64, 512, "cpu")
    if own:
        room = torch.empty((1 << 17) + 256, dtype=torch.uint8)
        w.room = room[-room.data_ptr() % 256:][:1 << 17]
    w._index = 0

    def work():
        for _ in range(8):
            kernels.mx4_linear(Rows(40, 512), w, Rows(40, 64))
    threads = [threading.Thread(target=work) for _ in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert library.calls == 24 and library.broken == 0


class Scratch(LowBitKernels):
    scratch_generation = 0


def test_scratch_grows_by_doubling(monkeypatch):
    """Calls that need more counters each time (prompts that grow, say) move the scratch, which makes recordings stale, few times."""
    monkeypatch.setattr(low_bits, "_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda: type("S", (), {"synchronize": lambda self: None})())
    real = {"empty": torch.empty, "zeros": torch.zeros}
    for name, make in real.items():
        monkeypatch.setattr(torch, name, lambda n, dtype=None, device=None, make=make: make(n, dtype=dtype))
    kernels = Scratch()
    for counters in range(100, 60000, 700):
        sums, zeros = kernels._kv8_scratch(7, 1000, counters)
        held = kernels._kv8_held[7]
        assert held[0] >= 1000 and held[1] >= counters and (sums, zeros) == held[2:4] and held[5].numel() == held[1]
    assert kernels.scratch_generation <= 5                              # 4,096 and up to 65,536
