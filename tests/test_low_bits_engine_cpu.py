"""The engine's formats for weights and cache with stand-in kernels: what runs, what is refused, what the cache holds."""
import pytest
import torch

import tiny
from infurnace_b200.cache import CacheManager
from infurnace_b200.engine import Engine, EngineOptions, SamplingParams
from infurnace_b200.engine.loading import build_runner, check_plan, default_num_pages
from infurnace_b200.errors import ModelConfigError
from infurnace_b200.kernels.low_bits import Kv8Pages
from infurnace_b200.models import config_from_dict, plan_for
from low_bit_refs import FourBits, LowBitReference


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return tiny.make_model_dir("A", str(tmp_path_factory.mktemp("m")))


def options(**kw):
    return EngineOptions(**{**dict(dtype="float32", device="cpu", page_size=16, num_pages=24, max_num_seqs=3, max_num_batched_tokens=64), **kw})


@pytest.mark.parametrize("weight,cache", [("mx4", "dtype"), ("stored", "int8"), ("mx4", "int8")])
def test_formats_run_through_the_engine(folder, weight, cache):
    eng = Engine.from_model_dir(folder, options(weight_format=weight, cache_format=cache), kernels=LowBitReference(torch.float64))
    prompts = [tiny.random_tokens(256, n, n) for n in (1, 20, 45)]
    outs = eng.generate(prompts, SamplingParams(max_tokens=6))
    assert [len(o) for o in outs] == [6, 6, 6]
    layer = eng.runner.model.layers[0]
    assert isinstance(layer.mixer.w_qkv, FourBits) == isinstance(layer.ffn.w_down, FourBits) == (weight == "mx4")
    group = eng.runner.cache.kv_groups[0]
    assert all(isinstance(t, Kv8Pages) == (cache == "int8") for t in group.tensors.values())
    eng.runner.cache.check()
    # however the prompts are cut, a request's pages have the same bits, and so the same tokens follow
    again = Engine.from_model_dir(folder, options(weight_format=weight, cache_format=cache, max_num_batched_tokens=7),
                                  kernels=LowBitReference(torch.float64))
    assert [len(o) for o in again.generate(prompts, SamplingParams(max_tokens=6))] == [6, 6, 6]


def test_bits_of_a_token(folder):
    plan = plan_for(config_from_dict(tiny.TINY["A"]["config"]))
    args = (plan, 16, 8, 2)
    wide = CacheManager(*args, dtype=torch.bfloat16, device="cpu").bytes_per_token()
    low = CacheManager(*args, dtype=torch.bfloat16, device="cpu", cache_format="int8").bytes_per_token()
    assert wide == 2 * low
    opts = options(num_pages=None)
    assert default_num_pages(plan, opts, torch.bfloat16, torch.device("cpu"), 128) == 3 * 8 + 1


def test_refusals(folder):
    for bad in (dict(weight_format="int3"), dict(cache_format="fp8"), dict(cache_format="int8", page_size=8), dict(cache_format="int8", page_size=24)):
        with pytest.raises(ModelConfigError):
            build_runner(folder, options(**bad), kernels=LowBitReference())
    plan = plan_for(config_from_dict(tiny.TINY["C"]["config"]))          # widths of 72 and 136
    with pytest.raises(ModelConfigError, match="multiples of 32"):
        check_plan(plan, options(weight_format="mx4"))
    check_plan(plan, options(cache_format="int8"))


def test_models_whose_mixers_have_no_8_bit_pages_are_refused():
    import json
    import os
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "configs")
    for name in ("kafunex-s", "lunelorn-s", "filorax-s", "golonex-s", "mubutar-s", "tigelorn-s"):
        with open(os.path.join(root, name + ".json"), encoding="utf-8") as f:
            plan = plan_for(config_from_dict(json.load(f)))
        with pytest.raises(ModelConfigError, match="cache_format int8"):
            check_plan(plan, options(cache_format="int8"))
    with open(os.path.join(root, "qwen3-8b.json"), encoding="utf-8") as f:
        check_plan(plan_for(config_from_dict(json.load(f))), options(cache_format="int8", weight_format="mx4"))


def test_a_padded_row_stores_and_sees_nothing(folder):
    """Decode steps are padded to a power of two: the extra rows leave pages and other rows alone."""
    eng = Engine.from_model_dir(folder, options(cache_format="int8", max_num_seqs=4), kernels=LowBitReference(torch.float64))
    prompts = [tiny.random_tokens(256, n, n) for n in (5, 9, 16)]
    outs = eng.generate(prompts, SamplingParams(max_tokens=5))
    alone = []
    for p in prompts:
        one = Engine.from_model_dir(folder, options(cache_format="int8", max_num_seqs=1), kernels=LowBitReference(torch.float64))
        alone.append(one.generate([p], SamplingParams(max_tokens=5))[0])
    assert outs == alone
