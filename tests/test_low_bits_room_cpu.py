"""The room for expanded 8-bit pages in an engine's account of the device's memory."""
import json
import os

import pytest
import torch

from infurnace_b200.engine import EngineOptions
from infurnace_b200.engine.loading import default_num_pages
from infurnace_b200.models import config_from_dict, plan_for

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("free", [2 << 30, 20 << 30, 120 << 30, 1000 << 30])
@pytest.mark.parametrize("cache,dtype", [("dtype", torch.bfloat16), ("int8", torch.bfloat16), ("int8", torch.float32)])
def test_pages_and_their_room_fit(monkeypatch, free, cache, dtype):
    from infurnace_b200.engine.loading import room_bytes
    with open(os.path.join(ROOT, "configs", "qwen3-8b.json"), encoding="utf-8") as f:
        plan = plan_for(config_from_dict(json.load(f)))
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, free))
    options = EngineOptions(cache_format=cache, max_num_seqs=64, page_size=16)
    pages = default_num_pages(plan, options, dtype, torch.device("cuda"), 40960)
    page = 36 * 2 * 8 * 16 * 128 * (1 if cache == "int8" else dtype.itemsize)
    room = room_bytes(plan, options, dtype, 40960, pages)
    assert (room > 0) == (cache == "int8" and dtype == torch.bfloat16) and room <= 4 << 30
    most, want = int(free * options.memory_fraction), 64 * 2560 + 1
    assert pages * page + room <= most
    assert pages == want or (pages + 2) * page + room_bytes(plan, options, dtype, 40960, pages + 2) > most
