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
