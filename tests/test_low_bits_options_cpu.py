"""Formats that an engine refuses before anything is loaded, and what prompts' cuts leave in 8-bit pages and tokens."""
import pytest
import torch

import tiny
from infurnace_b200.engine import Engine, EngineOptions, SamplingParams, StepEntry
from infurnace_b200.engine.loading import build_runner
from infurnace_b200.errors import ModelConfigError
from low_bit_refs import LowBitReference


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return tiny.make_model_dir("A", str(tmp_path_factory.mktemp("m")))


def options(**kw):
    return EngineOptions(**{**dict(dtype="float32", device="cpu", page_size=16, num_pages=24, max_num_seqs=3, max_num_batched_tokens=64), **kw})


@pytest.mark.parametrize("page_size", [0, 8, 24, 4112, 8192])
def test_page_sizes_that_8_bit_pages_do_not_have(folder, page_size):
    with pytest.raises(ModelConfigError, match="cache_format int8"):
        options(cache_format="int8", page_size=page_size).check_formats()
    with pytest.raises(ModelConfigError, match="cache_format int8"):
        build_runner(folder, options(cache_format="int8", page_size=page_size, num_pages=2), kernels=None)


@pytest.mark.parametrize("weight", ["stored", "mx4"])
def test_however_prompts_are_cut_the_same_bits_and_tokens_follow(folder, weight):
    """Token budgets of 64 and of 7: the tokens of every request are the same.  And a request in portions leaves the same bits in the pages
    of the first layer, whose keys and values do not depend on the cuts (further layers' do: a token attends to its page as it is then, and
    the page's step may grow with tokens that come later)."""
    prompts = [tiny.random_tokens(256, n, n) for n in (1, 20, 45)]
    fmt = dict(weight_format=weight, cache_format="int8")
    outs = [Engine.from_model_dir(folder, options(max_num_batched_tokens=budget, **fmt),
                                  kernels=LowBitReference(torch.float64)).generate(prompts, SamplingParams(max_tokens=6)) for budget in (64, 7)]
    assert outs[0] == outs[1] and all(len(o) == 6 for o in outs[0])
    bits = []
    for cuts in ([45], [7] * 6 + [3], [1] * 45, [16, 16, 13]):
        runner = build_runner(folder, options(**fmt), kernels=LowBitReference(torch.float64))[2]
        runner.cache.add_request("r")
        at = 0
        for n in cuts:
            runner.step([StepEntry("r", prompts[2][at:at + n])])
            at += n
        pages = runner.cache.kv_groups[0].tensors[min(runner.cache.kv_groups[0].tensors)]
        table = runner.cache.block_table("r", 0)
        codes = pages.codes[table].movedim(3, 1).reshape(48, -1)[:45]
        bits.append((codes, pages.exponents[table]))
    for codes, exponents in bits[1:]:
        assert torch.equal(codes, bits[0][0]) and torch.equal(exponents, bits[0][1])
