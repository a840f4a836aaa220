"""4-bit matrices and 8-bit pages through the engine on the GPU, against the same engine over plain statements in 64 bits."""
import json
import os
import subprocess
import sys

import pytest
import torch

import tiny
from infurnace_b200.engine import Engine, EngineOptions, SamplingParams, StepEntry
from infurnace_b200.engine.loading import build_runner
from low_bit_refs import LowBitReference, round4

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
FORMATS = [("mx4", "dtype"), ("stored", "int8"), ("mx4", "int8")]


@pytest.fixture(scope="module")
def folders(tmp_path_factory):
    root = str(tmp_path_factory.mktemp("m"))
    return {n: tiny.make_model_dir(n, root) for n in ("A", "B")}


def options(device="cuda", **kw):
    return EngineOptions(**{**dict(dtype="float32", device=device, page_size=16, num_pages=48, max_num_seqs=4, max_num_batched_tokens=64), **kw})


def logits(runner, tokens, cuts):
    """The logits of every place of a request that comes in portions."""
    runner.cache.add_request("r")
    at, out = 0, []
    for n in cuts:
        out.append(runner.step([StepEntry("r", tokens[at:at + n], list(range(n)))]).cpu().clone())
        at += n
    runner.cache.free_request("r")
    return torch.cat(out)


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("weight,cache", FORMATS)
def test_float32_logits_are_the_plain_ones(folders, name, weight, cache):
    """The same portions through both engines.  float32 sums differ in their last bits, which moves a number across a rounding step
    of 4 or 8 bits now and then, so single logits may part by such a step; the middle of them may not."""
    tokens = tiny.random_tokens(256, 61, 3)
    cuts = [17, 1, 1, 40, 1, 1]
    fmt = dict(weight_format=weight, cache_format=cache)
    a = logits(build_runner(folders[name], options(**fmt))[2], tokens, cuts)
    b = logits(build_runner(folders[name], options("cpu", **fmt), kernels=LowBitReference(torch.float64))[2], tokens, cuts)
    size = b.abs().max()
    assert (a - b).abs().median() <= 2e-5 * size and (a - b).abs().max() <= 0.1 * size


@pytest.mark.parametrize("weight,cache", FORMATS)
def test_generation_graphs_and_padding(folders, weight, cache):
    """bfloat16: steps replayed from graphs give the tokens of eager steps, in mixed batches of uneven requests."""
    fmt = dict(weight_format=weight, cache_format=cache, dtype="bfloat16")
    prompts = [tiny.random_tokens(256, n, 70 + n) for n in (5, 19, 64)]
    sp = SamplingParams(max_tokens=30, temperature=0.7, seed=3)
    a = Engine.from_model_dir(folders["B"], options(**fmt))
    b = Engine.from_model_dir(folders["B"], options(**fmt))
    b.runner.use_graphs = False
    assert a.generate(prompts, sp) == b.generate(prompts, sp)
    assert a.runner.graph_replays > 0 and b.runner.graph_replays == 0
    a.runner.cache.check()


def test_real_sizes_and_a_prompt_on_tcgen05():
    """Layers of the 0.6B sizes: a prompt whose attention runs on the tcgen05 kernel beside decoding requests.

    The cache: a block of 16 x 128 normal numbers has its largest near 3.6 sigma, a step between that over 128 and over 64, 0.04 sigma
    on average, so a number is off by 1.15 % of sigma (step / sqrt(12)); scores of standard deviation 1 then move the weights by
    1.2 %, and an attention output is off by 1.7 % (both together); three layers, each of which may double what comes in, leave
    the logits within 1.7 % sqrt(3) 2 = 6 % of those over 16-bit pages.

    The matrices: noise d before 4-bit rounding is sqrt(0.8 d) after it (the share of numbers that cross to the next level,
    d / 0.4, times a level's width squared), so logits say nothing; the engine's matrices are compared bit for bit."""
    with open(os.path.join(ROOT, "configs", "qwen3-0.6b.json"), encoding="utf-8") as f:
        cfg = dict(json.load(f), num_hidden_layers=3)
    tokens = tiny.random_tokens(cfg["vocab_size"], 301, 1)
    got, stored = {}, {}
    for weight, cache in [("stored", "dtype")] + FORMATS:
        eng = Engine.from_random(cfg, 5, options(dtype="bfloat16", num_pages=80, max_num_batched_tokens=512, max_model_len=512, weight_format=weight,
                                                 cache_format=cache))
        k = eng.runner.rt.kernels
        before = k.tc_attention_calls
        eng.runner.cache.add_request("short")
        eng.runner.step([StepEntry("short", tokens[:30])])
        eng.runner.cache.add_request("long")
        x = eng.runner.step([StepEntry("short", tokens[30:31], [0]), StepEntry("long", tokens[:300], [10, 299])]).float().cpu()
        y = eng.runner.step([StepEntry("long", tokens[300:], [0]), StepEntry("short", tokens[31:32], [0])]).float().cpu()
        got[weight, cache] = torch.cat((x, y))
        assert k.tc_attention_calls > before and got[weight, cache].isfinite().all()
        k.check_device_errors()
        layer = eng.runner.model.layers[1]
        for name, w in (("qkv", layer.mixer.w_qkv), ("o", layer.mixer.w_o), ("gate_up", layer.ffn.w_gate_up), ("down", layer.ffn.w_down)):
            if weight == "stored":
                stored[name] = round4(w.float().cpu())[2]
            else:
                out = torch.empty(w.shape, dtype=torch.float32, device="cuda")
                assert torch.equal(k.mx4_values(w, out).cpu().double(), stored[name]) and w.gated == (name == "gate_up")
    ref = got["stored", "dtype"]
    assert float((got["stored", "int8"] - ref).norm() / ref.norm()) <= 0.06


def test_command_line(folders):
    args = [sys.executable, "-m", "infurnace_b200", "--model", folders["A"], "--prompt-len", "20", "--max-tokens", "5", "--max-context", "64",
            "--weight-format", "mx4", "--cache-format", "int8", "--json"]
    p = subprocess.run(args, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr
    report = json.loads(p.stdout)
    assert len(report["generated_token_ids"]) == 5
    assert report["execution"]["weight_format"] == "mx4" and report["execution"]["cache_format"] == "int8"
