"""Requests with cuts for a vocabulary larger than the kernels draw from: refused at admission, and no other request is drawn into it."""
import os
import re

import pytest

import tiny
from infurnace_b200.engine import Request, RequestState, SamplingParams, StepEntry
from infurnace_b200.errors import BatchError
from infurnace_b200.kernels.answers import AnswerKernels
from test_answers_cpu import CutKernels, engine, model      # noqa: F401 (model: a fixture)


class SmallKernels(CutKernels):
    """As the device's, which draw under cuts up to a largest vocabulary and raise beyond it."""
    sample_max_vocab = 255

    def sample_filtered(self, logits, *args, **kw):
        assert logits.shape[1] <= self.sample_max_vocab
        super().sample_filtered(logits, *args, **kw)


def test_a_vocabulary_that_is_too_large_is_refused_at_admission(model):      # noqa: F811
    eng = engine(model, SmallKernels())
    prompt = tiny.random_tokens(256, 5, 71)
    for name, options in (("k", dict(top_k=5)), ("p", dict(top_p=0.9)), ("min", dict(min_p=0.1))):
        eng.add_request(Request(name, prompt, SamplingParams(max_tokens=3, temperature=0.9, **options)))
        assert eng.scheduler.get_request(name).state is RequestState.REJECTED
    eng.add_request(Request("plain", prompt, SamplingParams(max_tokens=3, temperature=0.9, seed=4)))
    eng.add_request(Request("scored", prompt, SamplingParams(max_tokens=3, top_k=1, logprobs=True)))
    while not all(eng.scheduler.get_request(n).is_terminal() for n in ("plain", "scored")):
        eng.step()
    plain, scored = (eng.scheduler.get_request(n) for n in ("plain", "scored"))
    assert plain.state is scored.state is RequestState.FINISHED
    assert list(plain.output_token_ids) == engine(model, CutKernels()).generate([prompt], SamplingParams(max_tokens=3, temperature=0.9, seed=4))[0]
    assert len(scored.output_logprobs) == 3
    eng.runner.cache.add_request("step")
    with pytest.raises(BatchError, match="vocabulary"):
        eng.runner.step_and_sample([StepEntry("step", [1], [0])], [0.5], [0.5], cuts=[(5, 1.0, 0.0)])


def test_a_vocabulary_at_the_limit_is_drawn_from(model):      # noqa: F811
    kernels = SmallKernels()
    kernels.sample_max_vocab = 256
    prompt = tiny.random_tokens(256, 5, 72)
    params = SamplingParams(max_tokens=3, temperature=0.9, top_p=0.8, seed=5)
    assert engine(model, kernels).generate([prompt], params) == engine(model, CutKernels()).generate([prompt], params)


def test_the_limit_is_the_kernels():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "infurnace_b200", "csrc", "sampling.cu")
    with open(path, encoding="utf-8") as f:
        text = f.read()
    ctas, size = (int(re.search(rf"constexpr int {name} = (\d+);", text).group(1)) for name in ("SURE_CLUSTER", "SLICE"))
    assert AnswerKernels.sample_max_vocab == ctas * size
