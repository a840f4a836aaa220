"""Several answers to one prompt on the device: the calls together as a program uses them, and the engine's options."""
import json
import math
import os
import subprocess
import sys
import threading

import pytest
import torch

import plain_qwen3 as P
import tiny
from answer_refs import attention, logprob_row, sample_row
from infurnace_b200.engine import Engine, EngineOptions, Request, RequestState, SamplingParams
from infurnace_b200.sampling import Sampler, uniform

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


@pytest.fixture(scope="module")
def models(tmp_path_factory):
    root = str(tmp_path_factory.mktemp("models"))
    return {n: tiny.make_model_dir(n, root) for n in ("A", "B")}


def test_a_row_of_nan_temperature_stays_as_it_is(K):
    logits = torch.randn((6, 151936), generator=torch.Generator().manual_seed(1)).cuda()
    t = torch.tensor([math.nan, 1.0, math.nan, 0.0, 0.7, math.nan], device="cuda")
    u = torch.full((6,), 0.3, device="cuda")
    out = torch.full((6,), -9, dtype=torch.int32, device="cuda")
    logprobs = torch.full((6,), 5.0, device="cuda")
    K.sample_filtered(logits, t, u, out, top_p=torch.full((6,), 0.9, device="cuda"), logprobs=logprobs)
    assert (out == -9).tolist() == [True, False, True, False, False, True] == (logprobs == 5.0).tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_answers_to_one_prompt(K, dtype):
    """Five answers to a prompt whose keys lie in pages once: a step stores the new tokens' keys and values, attends over shared and own pages, draws
    each answer's next token and scores it.  Attention is held against 64 bits, tokens against the definition on the step's own logits."""
    g = torch.Generator().manual_seed(5)
    n, prompt, page, kv_heads, group, dim, vocab, steps = 5, 75, 16, 2, 2, 64, 997, 20
    heads, width = kv_heads * group, 48
    common, own = prompt // page, -(-(prompt + steps) // page) - prompt // page
    embed = torch.randn((vocab, width), generator=g)
    wq, wkv = (torch.randn((width, x), generator=g) * width ** -0.5 for x in (heads * dim, 2 * kv_heads * dim))
    head = (torch.randn((heads * dim, vocab), generator=g) * 2 * (heads * dim) ** -0.5).cuda()
    pages = torch.zeros((common + n * own, 2, kv_heads, page, dim), dtype=dtype, device="cuda")
    tables = torch.tensor([list(range(common)) + list(range(common + r * own, common + (r + 1) * own)) for r in range(n)], dtype=torch.int32, device="cuda")

    def store(r, position, tokens):
        kv = (embed[tokens] @ wkv).view(-1, 2, kv_heads, dim).to(dtype).cuda()
        for i, x in enumerate(kv):
            pages[int(tables[r, (position + i) // page]), :, :, (position + i) % page] = x

    words = torch.randint(0, vocab, (prompt,), generator=g)
    for r in range(n):
        store(r, 0, words)                       # (the shared pages are the same for all)
    answers, scores = [[int(words[-1])] for _ in range(n)], [0.0] * n
    one = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device="cuda")
    cu_q, cu_groups, shared = one(list(range(n + 1))), one([0, n]), one([common * page])
    k, p, least = one([0, 40, 0, 9, 0]), one([0.9, 1.0, 1.0, 0.8, 1.0], torch.float32), one([0.0, 0.0, 0.05, 0.0, 0.0], torch.float32)
    t = one([0.8, 1.1, 0.9, 0.7, 0.0], torch.float32)
    out, logprobs, drawn = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    ranks = torch.empty(n, dtype=torch.int32, device="cuda")
    for step in range(steps):
        lens = [prompt + step] * n
        if step:
            for r in range(n):
                store(r, prompt + step - 1, torch.tensor([answers[r][-1]]))
        q = (embed[[a[-1] for a in answers]] @ wq).view(n, heads, dim).to(dtype).cuda()
        y = torch.empty_like(q)
        K.shared_prefix_attention(q, pages, tables, cu_q, one(lens), cu_groups, shared, y, dim ** -0.5, 0, 1, max(lens))
        if step % 7 == 0:
            want, size = attention(q.float().cpu(), pages.float().cpu(), tables.cpu(), list(range(n + 1)), lens, [0, n], [common * page], dim ** -0.5, 0)
            # (derived in test_shared_prefix_gpu.py: scores, weights, sums, and the output's half step)
            norm = float(q.float().norm(dim=2).max() * pages[:, 0].float().norm(dim=3).max()) * dim ** -0.5
            wide = 2 * dim * 2.0 ** -24 * norm + 2.0 ** -20 + 2 * max(lens) * 2.0 ** -24 + (2.0 ** -16 if dtype == torch.bfloat16 else 0.0)
            assert ((y.double().cpu() - want).abs() <= wide * size + torch.finfo(dtype).eps / 2 * want.abs()).all()
        logits = y.float().view(n, -1) @ head
        u = torch.tensor([uniform(r, step) for r in range(n)], dtype=torch.float32)
        K.sample_filtered(logits, t, u.cuda(), out, top_k=k, top_p=p, min_p=least, logprobs=drawn)
        K.token_logprobs(logits, out, logprobs, ranks)
        for r in range(n):
            token, logprob = sample_row(logits[r].cpu(), float(t[r]), float(u[r]), int(k[r]), float(p[r]), float(least[r]))
            assert int(out[r]) == token
            assert abs(float(drawn[r]) - logprob) <= 2.0 ** -23 * abs(logprob) + 2.0 ** -35
            assert int(ranks[r]) == logprob_row(logits[r].cpu(), token)[1]
            answers[r].append(token)
            scores[r] += float(logprobs[r])
    assert answers[0] != answers[1] and all(math.isfinite(x) and x < 0 for x in scores)


def test_threads_that_call_on_one_stream(K):
    """Three host threads on one stream, so that the launches of their calls come in any order between one another: what each gets is what it gets alone."""
    g = torch.Generator(device="cuda").manual_seed(3)
    one = lambda x, t=torch.int32: torch.tensor(x, dtype=t, device="cuda")
    pages = torch.randn((400, 2, 2, 16, 64), generator=g, device="cuda").to(torch.bfloat16)
    groups, members = 3, 12
    tables = torch.stack([torch.cat((torch.arange(20) + 20 * (r // members), 60 + 9 * r + torch.arange(9))) for r in range(groups * members)]).to(torch.int32).cuda()
    cu_groups, shared = one([members * j for j in range(groups + 1)]), one([320] * groups)

    def attend(seed):
        tokens = [1 + (r + seed) % 3 if r % 5 else 9 for r in range(groups * members)]
        cu_q, lens = one([sum(tokens[:r]) for r in range(len(tokens) + 1)]), one([330 + (7 * r + seed) % 130 for r in range(len(tokens))])
        q = torch.randn((sum(tokens), 8, 64), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(torch.bfloat16)
        return lambda: K.shared_prefix_attention(q, pages, tables, cu_q, lens, cu_groups, shared, torch.empty_like(q), 0.125, 0, 9, 464)

    def draw(seed):
        x = 3 * torch.randn((220, 20011), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
        u = torch.rand(220, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
        t, p = torch.ones(220, device="cuda"), one([0.9, 1.0] * 110, torch.float32)
        return lambda: K.sample_filtered(x, t, u, torch.empty(220, dtype=torch.int32, device="cuda"), top_p=p)

    calls = [attend(1), attend(2), draw(3)]
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    results = [[], [], []]

    def work(i):
        for _ in range(40):
            results[i].append(calls[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(3):
        assert len(results[i]) == 40 and all(torch.equal(x, alone[i]) for x in results[i])
    K.check_device_errors()


def engine(model_dir, name, dtype, **kw):
    opts = dict(dtype=dtype, page_size=tiny.TINY[name]["page_size"], num_pages=64, max_num_seqs=4, max_num_batched_tokens=64)
    opts.update(kw)
    return Engine.from_model_dir(model_dir, EngineOptions(**opts))


PARAMS = [dict(temperature=0.9, seed=1, top_k=20, top_p=0.8, logprobs=True), dict(temperature=0.7, seed=2), dict(temperature=1.2, seed=3, min_p=0.1),
          dict(), dict(temperature=1.0, seed=5, top_p=0.6, logprobs=True)]


@pytest.mark.parametrize("name", ["A", "B"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_cuts_in_the_engine(models, name, dtype):
    """A request's tokens do not depend on what else is in the batch, on graphs or on steps launched ahead; requests without cuts have the tokens that
    they had; log probabilities are the model's."""
    cfg, w = P.read_model(models[name])
    prompts = [tiny.random_tokens(cfg["vocab_size"], n, 30 + n) for n in (5, 12, 3, 7, 9)]
    params = [SamplingParams(max_tokens=9, **x) for x in PARAMS]
    eng = engine(models[name], name, dtype)
    together = eng.generate(prompts, params)
    kept = [eng.scheduler.get_request(f"gen-{i + 1}").output_logprobs for i in range(5)]
    assert [len(x) for x in kept] == [9, 0, 0, 0, 9]
    plain = engine(models[name], name, dtype)
    assert [together[1], together[3]] == plain.generate([prompts[1], prompts[3]], [params[1], params[3]])
    slow = engine(models[name], name, dtype)
    slow.overlap_decode = False
    slow.runner.use_graphs = False
    assert slow.generate(prompts, params) == together
    if dtype == "float32":
        alone = [engine(models[name], name, dtype).generate([p], sp)[0] for p, sp in zip(prompts, params)]
        assert alone == together
        for i in (0, 4):
            seq = list(prompts[i])
            for token, logprob in zip(together[i], kept[i]):
                logits = P.forward(cfg, w, seq)[-1].double()
                assert abs(float(torch.log_softmax(logits, 0)[token]) - logprob) < 1e-4      # (the model's own float32 error, some 1e-5)
                seq.append(token)


def test_the_narrowest_cuts_are_greedy(models):
    prompts = [tiny.random_tokens(256, n, 60 + n) for n in (4, 11)]
    want = engine(models["A"], "A", "float32").generate(prompts, SamplingParams(max_tokens=8))
    for cut in (dict(top_p=0.0), dict(min_p=1.0), dict(top_k=1), dict(top_k=3, top_p=0.0, min_p=1.0)):
        assert engine(models["A"], "A", "float32").generate(prompts, SamplingParams(max_tokens=8, temperature=1.3, seed=4, **cut)) == want


def test_the_sampler_draws_under_cuts(K):
    logits = (3 * torch.randn((4, 5003), generator=torch.Generator().manual_seed(3))).cuda()
    cuts = [(50, 1.0, 0.0), None, (0, 0.7, 0.02), (5, 0.5, 0.0)]
    temps, seeds = [0.8, 0.9, 1.2, 0.0], [3, 4, 5, 6]
    got = Sampler(K, "cuda").sample(logits, temps, seeds, [7] * 4, cuts=cuts)
    assert got[1] == Sampler(K, "cuda").sample(logits, temps, seeds, [7] * 4)[1]
    for r in (0, 2, 3):
        k, p, least = (float(torch.tensor(x)) for x in cuts[r])
        assert got[r] == sample_row(logits[r].cpu(), float(torch.tensor(temps[r])), uniform(seeds[r], 7), int(k), p, least)[0]


def test_preempted_requests_keep_their_tokens_and_scores(models):
    """Too few pages for all: requests give way and are computed anew, and have what they have alone."""
    prompts = [tiny.random_tokens(256, 10, 90 + i) for i in range(4)]
    params = [SamplingParams(max_tokens=12, temperature=0.9, seed=i, top_p=0.8, logprobs=True) for i in range(4)]
    eng = engine(models["A"], "A", "float32", num_pages=max(4, 60 // tiny.TINY["A"]["page_size"]))
    got = eng.generate(prompts, params)
    for i in range(4):
        alone = engine(models["A"], "A", "float32")
        assert alone.generate([prompts[i]], params[i])[0] == got[i]
        mine, want = eng.scheduler.get_request(f"gen-{i + 1}").output_logprobs, alone.scheduler.get_request("gen-1").output_logprobs
        assert len(mine) == 12 and all(abs(a - b) < 1e-5 for a, b in zip(mine, want))


def test_the_command_line_draws_under_cuts(models):
    cmd = [sys.executable, "-m", "infurnace_b200", "--model", models["A"], "--dtype", "float32", "--prompt-ids", "5,6,7", "--max-tokens", "5", "--temperature", "0.9",
           "--top-k", "12", "--top-p", "0.9", "--min-p", "0.01", "--logprobs", "--seed", "3", "--page-size", str(tiny.TINY["A"]["page_size"]), "--json"]
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    run = subprocess.run(cmd, capture_output=True, text=True, cwd=root, timeout=300)
    assert run.returncode == 0, run.stderr
    report = json.loads(run.stdout)
    want = engine(models["A"], "A", "float32").generate([[5, 6, 7]], SamplingParams(max_tokens=5, temperature=0.9, top_k=12, top_p=0.9, min_p=0.01, seed=3))[0]
    assert report["generated_token_ids"] == want and len(report["logprobs"]) == 5 and all(x <= 0 for x in report["logprobs"])
    bad = subprocess.run(cmd + ["--top-p", "1.5"], capture_output=True, text=True, cwd=root, timeout=300)
    assert bad.returncode == 1 and "top_p 1.5" in bad.stderr


def test_a_wrong_option_is_refused_by_the_engine(models):
    eng = engine(models["A"], "A", "float32")
    eng.add_request(Request("a", [1, 2], SamplingParams(max_tokens=2, temperature=0.5, top_p=2.0)))
    assert eng.scheduler.get_request("a").state is RequestState.REJECTED
