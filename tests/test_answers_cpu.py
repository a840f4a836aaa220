"""What the calls and options of several answers do on the host, without a GPU: refusals, admission, staging."""
import pytest
import torch

import tiny
from infurnace_b200.cache import CacheManager
from infurnace_b200.engine import Engine, EngineOptions, Request, RequestState, SamplingParams, StepEntry
from infurnace_b200.engine.scheduler import Scheduler
from infurnace_b200.errors import BatchError, KernelError
from infurnace_b200.kernels import answers
from infurnace_b200.kernels.answers import AnswerKernels
from infurnace_b200.models import config_from_dict, plan_for
from kernel_refs import ReferenceKernels


class Tensor:
    """What a call looks at of a tensor on a device."""
    def __init__(self, shape, dtype=torch.float32, stride=None, device=0, at=4096):
        self.shape, self.dtype, self.at, self.index = torch.Size(shape), dtype, at, device
        if stride is None:
            stride, step = [], 1
            for n in reversed(shape):
                stride.insert(0, step)
                step *= n
        self._stride = tuple(stride)
        self.device = f"cuda:{device}"

    def stride(self):
        return self._stride

    def dim(self):
        return len(self.shape)

    def numel(self):
        return self.shape.numel()

    def is_contiguous(self):
        return self._stride == Tensor(self.shape)._stride

    def get_device(self):
        return self.index

    def data_ptr(self):
        return self.at


class Library:
    """Stands for the compiled libraries: every call is noted and accepted."""
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append(name)
            return 0
        return call


class Kernels(AnswerKernels):
    _progress, launches, _dev_err_at = None, 0, 0

    def __init__(self):
        self._sampling, self._sampling_max_vocab = Library(), 1000

    def _shared_lib(self, dtype, dim):
        return (lambda packed: 0), (lambda *sizes: 256)


@pytest.fixture
def K(monkeypatch):
    monkeypatch.setattr(answers, "_raw_stream", lambda index: 7)
    monkeypatch.setattr(answers, "_device_of", lambda index: None)
    return Kernels()


I32, BF16 = torch.int32, torch.bfloat16


def cut_args(rows=3, **other):
    args = dict(logits=Tensor((rows, 100)), temperature=Tensor((rows,)), uniform=Tensor((rows,)), out=Tensor((rows,), I32), top_k=Tensor((rows,), I32),
                top_p=Tensor((rows,)), min_p=Tensor((rows,)), logprobs=Tensor((rows,)))
    args.update(other)
    return args


def test_drawing_takes_what_it_documents(K):
    K.sample_filtered(**cut_args())
    K.sample_filtered(**cut_args(top_k=None, top_p=None, min_p=None, logprobs=None))
    K.sample_filtered(**cut_args(logits=Tensor((3, 100), BF16, (128, 1))))
    K.sample_filtered(**cut_args(rows=1, logits=Tensor((1, 100), stride=(7, 1))))
    assert K.launches == 4 and K._sampling.calls == ["ifb_sample_cut"] * 4
    K.sample_filtered(**cut_args(rows=0))
    assert K.launches == 4


@pytest.mark.parametrize("wrong", [
    dict(logits=Tensor((3, 100), torch.float16)), dict(logits=Tensor((3, 100), torch.float64)), dict(logits=Tensor((300,))),
    dict(logits=Tensor((3, 0))), dict(logits=Tensor((3, 100), stride=(200, 2))), dict(logits=Tensor((3, 100), device=-1)),
    dict(logits=Tensor((3, 1001))), dict(temperature=Tensor((2,))), dict(temperature=Tensor((3,), BF16)), dict(uniform=Tensor((3, 1))),
    dict(uniform=Tensor((3,), torch.float64)), dict(top_k=Tensor((3,), torch.int64)), dict(top_k=Tensor((3,))), dict(top_p=Tensor((4,))),
    dict(min_p=Tensor((3,), stride=(2,))), dict(out=Tensor((3,), torch.int64)), dict(out=Tensor((3,), I32, device=1)), dict(logprobs=Tensor((3,), BF16))])
def test_drawing_refuses(K, wrong):
    with pytest.raises(KernelError, match="sample_filtered"):
        K.sample_filtered(**cut_args(**wrong))
    assert not K._sampling.calls and K.launches == 0


@pytest.mark.parametrize("wrong", [
    dict(logits=Tensor((3, 100), torch.float16)), dict(logits=Tensor((3, 100), stride=(1, 3))), dict(tokens=Tensor((3,), torch.int64)), dict(tokens=Tensor((4,), I32)),
    dict(out=Tensor((3,), BF16)), dict(ranks=Tensor((3,))), dict(ranks=Tensor((3,), I32, device=1)), dict(logits=Tensor((3, 100), device=-1))])
def test_scoring_refuses(K, wrong):
    args = dict(logits=Tensor((3, 100)), tokens=Tensor((3,), I32), out=Tensor((3,)), ranks=Tensor((3,), I32))
    K.token_logprobs(**args)
    with pytest.raises(KernelError, match="token_logprobs"):
        K.token_logprobs(**{**args, **wrong})
    assert K.launches == 1


def shared_args(**other):
    args = dict(q=Tensor((5, 8, 64), BF16), kv_pages=Tensor((20, 2, 2, 16, 64), BF16), block_tables=Tensor((4, 6), I32), cu_q=Tensor((5,), I32),
                seq_lens=Tensor((4,), I32), cu_groups=Tensor((3,), I32), shared_lens=Tensor((2,), I32), out=Tensor((5, 8, 64), BF16), scale=0.125, window=0,
                max_q_len=2, max_seq_len=96, room=Tensor((256,), torch.uint8))
    args.update(other)
    return args


def test_shared_attention_takes_what_it_documents(K):
    K.shared_prefix_attention(**shared_args())
    K.shared_prefix_attention(**shared_args(q=Tensor((5, 8, 64), BF16, (768, 64, 1)), kv_pages=Tensor((20, 2, 2, 16, 64), BF16, (8192, 2048, 1024, 64, 1))))
    K.shared_prefix_attention(**shared_args(q=Tensor((5, 8, 64)), kv_pages=Tensor((20, 2, 2, 16, 64)), out=Tensor((5, 8, 64))))
    assert K.launches == 3 + 3 + 2


@pytest.mark.parametrize("wrong", [
    dict(q=Tensor((5, 8, 64), torch.float16)), dict(q=Tensor((5, 512), BF16)), dict(q=Tensor((5, 7, 64), BF16), out=Tensor((5, 7, 64), BF16)),
    dict(q=Tensor((5, 8, 64), BF16, (1024, 128, 1))), dict(q=Tensor((5, 8, 64), BF16, (516, 64, 1))), dict(q=Tensor((5, 8, 64), BF16, at=4104)),
    dict(out=Tensor((5, 8, 64))), dict(out=Tensor((5, 8, 64), BF16, (768, 64, 1))), dict(out=Tensor((4, 8, 64), BF16)),
    dict(kv_pages=Tensor((20, 2, 2, 16, 64))), dict(kv_pages=Tensor((20, 2, 16, 64), BF16)), dict(kv_pages=Tensor((20, 1, 2, 16, 64), BF16)),
    dict(kv_pages=Tensor((20, 2, 2, 16, 128), BF16)), dict(kv_pages=Tensor((20, 2, 2, 16, 64), BF16, (4096, 1024, 2048, 64, 1))),
    dict(kv_pages=Tensor((20, 2, 2, 16, 64), BF16, (2048, 2048, 1024, 64, 1))), dict(kv_pages=Tensor((0, 2, 2, 16, 64), BF16)),
    dict(q=Tensor((5, 8, 40), BF16), out=Tensor((5, 8, 40), BF16), kv_pages=Tensor((20, 2, 2, 16, 40), BF16)),
    dict(q=Tensor((5, 8, 272), BF16), out=Tensor((5, 8, 272), BF16), kv_pages=Tensor((20, 2, 2, 16, 272), BF16)),
    dict(q=Tensor((5, 130, 64), BF16), out=Tensor((5, 130, 64), BF16)), dict(cu_q=Tensor((4,), I32)), dict(cu_q=Tensor((5,), torch.int64)),
    dict(seq_lens=Tensor((4,), torch.int64)), dict(cu_groups=Tensor((2,), I32)), dict(shared_lens=Tensor((2,), I32, (2,))), dict(shared_lens=Tensor((2,), I32, device=1)),
    dict(block_tables=Tensor((3, 6), I32)), dict(block_tables=Tensor((4, 6), torch.int64)), dict(block_tables=Tensor((4, 6), I32, (1, 4))),
    dict(max_seq_len=97), dict(max_q_len=0), dict(window=-1), dict(kv_pages=Tensor((20, 2, 2, 16, 64), BF16, device=1)),
    dict(room=Tensor((255,), torch.uint8)), dict(room=Tensor((256,), torch.int8)), dict(room=Tensor((256,), torch.uint8, at=4104)),
    dict(seq_lens=Tensor((2047,), I32), cu_q=Tensor((2048,), I32), block_tables=Tensor((2047, 6), I32))])
def test_shared_attention_refuses(K, wrong):
    with pytest.raises(KernelError, match="shared_prefix_attention"):
        K.shared_prefix_attention(**shared_args(**wrong))
    assert K.launches == 0


# ------------------------------------------------------------------------------------------------ options
@pytest.mark.parametrize("options,alone,with_cuts", [
    (dict(top_k=5), False, True), (dict(top_p=0.9), False, True), (dict(min_p=0.1), False, True), (dict(logprobs=True), False, True),
    (dict(top_k=1), True, True), (dict(top_k=-1), False, False), (dict(top_k=2.5), False, False), (dict(top_p=1.1), False, False),
    (dict(top_p=-0.1), False, False), (dict(top_p=float("nan")), False, False), (dict(min_p=1.5), False, False), (dict(min_p=float("nan")), False, False),
    (dict(top_k=1 << 31), False, False), (dict(temperature=-1.0), False, False), (dict(top_p=0.0, min_p=1.0, top_k=7), False, True)])
def test_what_is_admitted(options, alone, with_cuts):
    plan = plan_for(config_from_dict(tiny.TINY["A"]["config"]))
    for cuts, want in ((False, alone), (True, with_cuts)):
        cache = CacheManager(plan, tiny.TINY["A"]["page_size"], 8, 2, allocate_tensors=False)
        s = Scheduler(cache, 2, 32, 64, cuts=cuts)
        s.add_request(Request("a", [1, 2, 3], SamplingParams(max_tokens=2, **{"temperature": 0.8, **options})))
        assert (s.get_request("a").state is RequestState.WAITING) == want


def test_which_requests_are_drawn_under_cuts():
    assert SamplingParams(temperature=0.8).cuts is None
    assert SamplingParams(top_k=5).cuts is None                                  # greedy
    assert SamplingParams(temperature=0.8, top_k=1, top_p=0.5).cuts is None      # greedy too
    assert SamplingParams(temperature=0.8, top_k=5).cuts == (5, 1.0, 0.0)
    assert SamplingParams(temperature=0.8, top_p=0.5, min_p=0.25).cuts == (0, 0.5, 0.25)


class CutKernels(ReferenceKernels):
    """The reference kernels with the calls that draw under cuts and score, stated plainly."""
    def sample_filtered(self, logits, temperature, uniform, out, top_k=None, top_p=None, min_p=None, logprobs=None):
        from answer_refs import sample_row
        for r in range(logits.shape[0]):
            t = float(temperature[r])
            if t == t:
                out[r] = sample_row(logits[r], t, float(uniform[r]), int(top_k[r]), float(top_p[r]), float(min_p[r]))[0]

    def token_logprobs(self, logits, tokens, out, ranks=None):
        from answer_refs import logprob_row
        for r in range(logits.shape[0]):
            out[r] = logprob_row(logits[r], int(tokens[r]))[0]


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    return tiny.make_model_dir("A", str(tmp_path_factory.mktemp("models")))


def engine(model, kernels, **kw):
    opts = dict(dtype="float32", device="cpu", page_size=tiny.TINY["A"]["page_size"], num_pages=40, max_num_seqs=4, max_num_batched_tokens=32)
    opts.update(kw)
    return Engine.from_model_dir(model, EngineOptions(**opts), kernels=kernels)


def test_an_engine_draws_under_cuts_and_keeps_log_probabilities(model):
    import math

    import plain_qwen3 as P
    cfg, w = P.read_model(model)
    prompts = [tiny.random_tokens(256, n, 40 + n) for n in (5, 9, 3)]
    params = [SamplingParams(max_tokens=6, temperature=0.9, seed=1, top_k=20, top_p=0.8, logprobs=True), SamplingParams(max_tokens=6, temperature=0.7, seed=2),
              SamplingParams(max_tokens=6, temperature=1.2, seed=3, min_p=0.1)]
    eng = engine(model, CutKernels())
    together = eng.generate(prompts, params)
    alone = [engine(model, CutKernels()).generate([p], sp)[0] for p, sp in zip(prompts, params)]
    assert together == alone
    assert alone[1] == engine(model, ReferenceKernels()).generate([prompts[1]], params[1])[0]      # drawn as ever
    kept = eng.scheduler.get_request("gen-1").output_logprobs
    assert len(kept) == 6 and eng.scheduler.get_request("gen-2").output_logprobs == ()
    seq = list(prompts[0])
    for token, logprob in zip(together[0], kept):
        logits = P.forward(cfg, w, seq)[-1].double()
        assert abs(float(torch.log_softmax(logits, 0)[token]) - logprob) < 1e-4      # (a float32 model's logits, off by some 1e-5)
        assert (logits > logits[token]).sum() < 20                                 # top_k
        seq.append(token)
    assert not any(math.isnan(x) for x in kept)


def test_an_engine_without_such_kernels_refuses(model):
    eng = engine(model, ReferenceKernels())
    eng.add_request(Request("a", [1, 2, 3], SamplingParams(max_tokens=2, temperature=0.5, top_p=0.5)))
    assert eng.scheduler.get_request("a").state is RequestState.REJECTED
    eng.runner.cache.add_request("b")
    with pytest.raises(BatchError, match="cuts"):
        eng.runner.step_and_sample([StepEntry("b", [1], [0])], [0.5], [0.5], cuts=[(5, 1.0, 0.0)])
    with pytest.raises(BatchError, match="logprobs"):
        eng.runner.step_and_sample([StepEntry("b", [1], [0])], [0.5], [0.5], logprobs=True)
    with pytest.raises(BatchError, match="cuts"):
        eng.runner.step_and_sample([StepEntry("b", [1], [0])], [0.5], [0.5], cuts=[])


def test_rows_without_cuts_and_padding_are_not_drawn_anew(model):
    eng = engine(model, CutKernels())
    run, cache = eng.runner, eng.runner.cache
    for rid in "abc":
        cache.add_request(rid)
        run.step([StepEntry(rid, [1, 2, 3])])
    entries = [StepEntry(rid, [5], [0]) for rid in "abc"]
    run.validate(entries, sampled=True)
    run._reserve(entries)
    ctx = run._build_context(entries, temperatures=[0.7, 0.0, 0.5], uniforms=[0.5] * 3, pad_to=4, seq_bucket=256, cuts=[None, (4, 0.5, 0.0), (3, 0.9, 0.25)])
    k, p, least, t = ctx.cuts
    assert t.isnan().tolist() == [True, True, False, True]
    assert (int(k[2]), float(p[2]), float(least[2]), float(t[2])) == (3, pytest.approx(0.9), 0.25, 0.5)
    views = [ctx.temperatures, ctx.uniforms, *ctx.cuts]
    spans = sorted((v.data_ptr(), v.data_ptr() + v.numel() * 4) for v in views)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
    assert spans[-1][1] <= run._dev_tables.data_ptr()
