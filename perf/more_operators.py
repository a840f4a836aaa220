"""The work by which the operators of several answers to one prompt are judged: drawing a token under top-k, top-p and min-p,
the log probabilities of what was drawn, and attention over pages that requests share.

Each case is one call:

* ``sample``: a token for each row of logits, from softmax(logits / temperature) cut by top-k, then top-p, then min-p, with one
  given uniform number a row, and its log probability under what the cuts left (0 where it was certain).  Rows have parameters of
  their own; a temperature of 0 is greedy.
* ``logprobs``: the log probability of a given token in each row of logits, and its rank (how many tokens come before it).
* ``attend``: causal attention of a step's queries over pages of keys and values, where the requests of a group have the pages of
  their first keys in common: samples of one prompt that decode, and questions to one document.

``prepare`` makes inputs and pages with torch; ``run`` is the call, in its plain form or (``own``) through the package's kernels;
``exact`` states the same in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    def sample(name, rows, vocab, cuts, dtype="float32", masked=0.0):
        """``cuts``: what the rows have, one after the other, of "greedy", "plain", "k", "p", "min", "kp" and "all"."""
        return dict(name=name, kind="sample", rows=rows, vocab=vocab, cuts=cuts, dtype=dtype, masked=masked)

    def logprobs(name, rows, vocab, dtype="float32"):
        return dict(name=name, kind="logprobs", rows=rows, vocab=vocab, dtype=dtype)

    def attend(name, groups, members, shared, shortest, longest, tokens=1, page=16, kv_heads=8, group=4, dim=128, window=0, dtype="bfloat16"):
        """``groups`` of 1 to ``members`` requests (the first has them all) that share ``shared`` keys or less (the first: all);
        each request has ``shortest`` to ``longest`` keys of its own and brings ``tokens`` queries."""
        return dict(name=name, kind="attend", groups=groups, members=members, shared=shared, shortest=shortest, longest=longest, tokens=tokens,
                    page=page, kv_heads=kv_heads, group=group, dim=dim, window=window, dtype=dtype)

    return [
        # one chat with the usual top-p: what a user waits for behind every token
        sample("sample-1-p", 1, 151936, "p"),
        # a step of 64 requests, each with options of its own
        sample("sample-64-mixed", 64, 151936, "greedy k p min kp all plain p"),
        # a full batch of creative writing: nothing is cut
        sample("sample-256-plain", 256, 151936, "plain"),
        # samples under a grammar that forbids nine tokens in ten, a small odd vocabulary, logits of 16 bits
        sample("sample-37-masked-bf16", 37, 32749, "kp p all", dtype="bfloat16", masked=0.9),
        # the log probabilities of a step's eight tokens
        logprobs("logprobs-8", 8, 151936),
        # a document scored token by token
        logprobs("logprobs-prompt-2043", 2043, 151936),
        # the same for a smaller vocabulary, logits of 16 bits
        logprobs("logprobs-prompt-1000-bf16", 1000, 32768, dtype="bfloat16"),
        # four answers to a short prompt (0.6B heads): latency counts
        attend("attend-4-short", 1, 4, 480, 3, 40, group=2),
        # 64 answers to a long prompt (8B heads)
        attend("attend-64-long", 1, 64, 8000, 20, 300),
        # several conversations behind a few system prompts of unequal length, pages of 32, odd sizes
        attend("attend-groups", 7, 19, 3008, 1, 1500, page=32),
        # questions of 230 tokens to one document
        attend("attend-questions", 1, 8, 6000, 230, 240, tokens=230),
        # samples in the 32-bit mode
        attend("attend-9-fp32", 2, 9, 1296, 5, 200, kv_heads=4, group=3, dim=64, dtype="float32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["sample", "sample", "sample", "logprobs", "logprobs", "attend", "attend", "attend", "attend"])
    dtype = "float32" if rng.random() < (0.2 if kind == "attend" else 0.6) else "bfloat16"
    if kind != "attend":
        vocab = _log(rng, 200, 200_000)
        rows = _log(rng, 1, min(256 if kind == "sample" else 2000, 38_000_000 // vocab if kind == "sample" else 300_000_000 // vocab))
        if kind == "logprobs":
            return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype)
        cuts = " ".join(rng.choice(["greedy", "plain", "k", "k", "p", "p", "p", "min", "min", "kp", "kp", "all"]) for _ in range(rng.randint(1, 6)))
        return dict(kind=kind, rows=rows, vocab=vocab, cuts=cuts, dtype=dtype, masked=rng.choice([0.0, 0.0, 0.5, 0.97]))
    c = dict(kind=kind, page=rng.choice([16, 16, 32, 64]), kv_heads=rng.choice([1, 2, 4, 8]), group=rng.choice([1, 2, 3, 4, 5, 8]),
             dim=rng.choice([64, 128, 128, 128, 96, 256]), dtype=dtype, tokens=1, window=0, groups=rng.choice([1, 1, 2, 5]))
    heads = c["kv_heads"] * c["group"]
    if rng.random() < 0.7:
        c["members"] = _log(rng, 2, 64 if c["groups"] == 1 else 16)
        c["longest"] = _log(rng, 1, 1000)
        if rng.random() < 0.2:
            c["window"] = _log(rng, 16, 4000)
    else:
        c["members"] = rng.randint(2, 6)
        c["tokens"] = _log(rng, 2, 200)
        c["longest"] = c["tokens"] + rng.randint(0, 100)
    c["shared"] = c["page"] * _log(rng, 1, 6000 // c["page"])
    if dtype == "float32":
        c["shared"] = min(c["shared"], c["page"] * max(1, 40_000_000 // (c["groups"] * c["members"] * c["tokens"] * heads * c["dim"]) // c["page"]))
    c["shortest"] = rng.randint(c["tokens"], c["longest"])
    return c


def _layout(case):
    """(requests of each group, keys that each group shares, all keys of each request)."""
    n, m, page = case["groups"], case["members"], case["page"]
    members = [max(1, m - (m * g) // n) for g in range(n)]
    shared = [(case["shared"] - (case["shared"] * g) // (2 * n)) // page * page for g in range(n)]
    lens, total, at = [], sum(members), 0
    for count, keys in zip(members, shared):
        for _ in range(count):
            lens.append(keys + case["longest"] - (case["longest"] - case["shortest"]) * at // max(1, total - 1))
            at += 1
    return members, shared, lens


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, scale=1.0):
    return torch.randn(shape, generator=g, device=DEV) * scale


def _logits(g, rows, vocab, dtype):
    """Rows as a head gives them: most tokens far below a few, some rows sure of theirs and some not."""
    spread = 1.5 + 2.0 * torch.rand((rows, 1), generator=g, device=DEV)
    x = _normal(g, (rows, vocab)).mul_(spread)
    best = torch.randint(0, vocab, (rows, 5), generator=g, device=DEV)
    x.scatter_add_(1, best, 6.0 * torch.rand((rows, 5), generator=g, device=DEV) * spread)
    return x.to(dtype)


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case=case, dtype=dtype)
    if case["kind"] == "attend":
        _prepare_pages(case, s, g)
    else:
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = _logits(g, rows, vocab, dtype)
        if case["kind"] == "logprobs":
            # tokens as they come: mostly likely ones
            likely = s["logits"].float().argmax(dim=1)
            other = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
            s["tokens"] = torch.where(torch.rand(rows, generator=g, device=DEV) < 0.5, likely, other).to(torch.int32)
        else:
            _prepare_cuts(case, s, g)
    if own:
        from infurnace_b200.kernels import load_cuda_kernels
        s["kernels"] = load_cuda_kernels()
    return s


def _prepare_cuts(case, s, g):
    rows, vocab = case["rows"], case["vocab"]
    if case["masked"]:
        keep = torch.rand((rows, vocab), generator=g, device=DEV) >= case["masked"]
        keep[:, vocab // 2] = True
        s["logits"].masked_fill_(~keep, -math.inf)
    cuts = case["cuts"].split()
    names = [cuts[r % len(cuts)] for r in range(rows)]
    rand = torch.rand((4, rows), generator=g, device=DEV)

    def where(kinds, value, off):
        on = torch.tensor([n in kinds for n in names], device=DEV)
        return torch.where(on, value, off)

    s["temperature"] = where(("greedy",), torch.zeros(rows, device=DEV), 0.5 + 0.8 * rand[0])
    s["top_k"] = where(("k", "kp", "all"), (1 + 100 * rand[1] ** 2).to(torch.int32), torch.zeros(rows, dtype=torch.int32, device=DEV))
    s["top_p"] = where(("p", "kp", "all"), 0.7 + 0.29 * rand[2], torch.ones(rows, device=DEV))
    s["min_p"] = where(("min", "all"), 0.02 + 0.1 * rand[3], torch.zeros(rows, device=DEV))
    s["uniform"] = torch.rand(rows, generator=g, device=DEV)


def _prepare_pages(case, s, g):
    page, heads, dim, dtype = case["page"], case["kv_heads"], case["dim"], s["dtype"]
    members, shared, lens = _layout(case)
    requests, tokens = len(lens), case["tokens"]
    common = [n // page for n in shared]
    owner = [j for j, n in enumerate(members) for _ in range(n)]
    held = [-(-n // page) for n in lens]
    pages = sum(common) + sum(h - common[j] for h, j in zip(held, owner)) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    tables = torch.full((requests, max(held)), -1, dtype=torch.int32, device=DEV)
    at, firsts = 0, []
    for n in common:
        firsts.append(order[at:at + n])
        at += n
    for r, (n, j) in enumerate(zip(held, owner)):
        tables[r, :common[j]] = firsts[j]
        tables[r, common[j]:n] = order[at:at + n - common[j]]
        at += n - common[j]
    # keys of uneven size by head and feature
    size = torch.exp(0.4 * _normal(g, (2, heads, 1, 1)))
    feature = torch.stack((torch.exp(0.3 * _normal(g, (heads, 1, dim))), torch.ones((heads, 1, dim), device=DEV)))
    s["pages"] = torch.empty((pages, 2, heads, page, dim), dtype=dtype, device=DEV)
    for a in range(0, pages, 256):
        part = s["pages"][a:a + 256]
        part.copy_(_normal(g, part.shape) * (size * feature))
    s["q"] = _normal(g, (requests * tokens, heads * case["group"], dim)).to(dtype)
    starts = [0]
    for n in members:
        starts.append(starts[-1] + n)

    def whole(x):
        return torch.tensor(x, dtype=torch.int32, device=DEV)

    s.update(tables=tables, cu_q=whole([tokens * r for r in range(requests + 1)]), seq_lens=whole(lens), cu_groups=whole(starts),
             shared_lens=whole(shared), scale=dim ** -0.5, longest=max(lens), layout=(members, shared, lens))


# ------------------------------------------------------------------------------------------------ the plain forms
def _plain_sample(s):
    x = s["logits"].float()
    vocab = x.shape[1]
    # 64 bits: the borders between tokens lie closer than a sum's rounding in 32
    t = torch.where(s["temperature"] > 0, s["temperature"], 1.0).double()[:, None]
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    weight = torch.exp((value.double() - value[:, :1].double()) / t)
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    weight = torch.where(torch.arange(vocab, device=DEV) < k, weight, 0.0)
    p = s["top_p"].double()[:, None]
    before = torch.cumsum(weight, dim=1)
    goal = p * before[:, -1:]
    before = torch.cat((torch.zeros_like(goal), before[:, :-1]), dim=1)
    weight = torch.where((p >= 1) | (before < goal), weight, 0.0)
    weight = torch.where(weight >= s["min_p"].double()[:, None], weight, 0.0)
    weight = torch.zeros_like(weight).scatter_(1, index, weight)
    run = torch.cumsum(weight, dim=1)
    drawn = (run <= s["uniform"].double()[:, None] * run[:, -1:]).sum(dim=1)
    drawn = torch.where(s["temperature"] > 0, drawn, index[:, 0])
    logprob = torch.log(torch.gather(weight, 1, drawn[:, None])[:, 0] / run[:, -1])
    return drawn.to(torch.int32), torch.where(s["temperature"] > 0, logprob, 0.0).float()


def _plain_logprobs(s):
    token = s["tokens"].long()[:, None]
    x = s["logits"].float()
    own_value = torch.gather(x, 1, token)
    top = x.amax(dim=1, keepdim=True)
    logprob = own_value - top - torch.log(torch.exp(x - top).sum(dim=1, keepdim=True))
    index = torch.arange(x.shape[1], device=DEV)
    rank = ((x > own_value) | ((x == own_value) & (index < token))).sum(dim=1)
    return logprob[:, 0], rank.to(torch.int32)


def _keys(pages, rows, heads, page):
    """Keys and values of tables ``rows`` [..., n] as float32 [2, ..., heads, n * page, dim]."""
    kv = pages[rows.long()].float()                                     # [..., n, 2, heads, page, dim]
    lead = rows.dim() - 1
    kv = kv.permute(lead + 1, *range(lead), lead + 2, lead, lead + 3, lead + 4)
    return kv.reshape(2, *rows.shape[:-1], heads, -1, kv.shape[-1])


def _plain_attend(s):
    case = s["case"]
    heads, group, dim, page, tokens = case["kv_heads"], case["group"], case["dim"], case["page"], case["tokens"]
    members, shared, lens = s["layout"]
    out, first = [], 0
    for count, common in zip(members, shared):
        most = max(lens[first:first + count])
        tables = s["tables"][first:first + count, common // page:-(-most // page)].clamp(min=0)
        kp, vp = _keys(s["pages"], s["tables"][first, :common // page], heads, page)         # [heads, common, dim]
        ko, vo = _keys(s["pages"], tables, heads, page)                                      # [count, heads, own, dim]
        q = s["q"][first * tokens:(first + count) * tokens].float().reshape(count, tokens, heads, group, dim)
        rows = q.permute(0, 2, 3, 1, 4).reshape(count, heads, group * tokens, dim)
        together = rows.permute(1, 0, 2, 3).reshape(heads, -1, dim)
        scores = torch.cat(((together @ kp.transpose(1, 2)).reshape(heads, count, group * tokens, -1).transpose(0, 1),
                            rows @ ko.transpose(2, 3)), dim=3) * s["scale"]
        position = s["seq_lens"][first:first + count, None] - tokens + torch.arange(tokens, device=DEV)
        key = torch.arange(scores.shape[3], device=DEV)
        seen = key <= position[..., None]
        if case["window"]:
            seen &= key > position[..., None] - case["window"]
        scores = scores.reshape(count, heads, group, tokens, -1).masked_fill(~seen[:, None, None], -math.inf)
        weight = torch.exp(scores - scores.amax(dim=4, keepdim=True))
        weight = (weight / weight.sum(dim=4, keepdim=True)).reshape(count, heads, group * tokens, -1)
        y = (weight[..., :common].transpose(0, 1).reshape(heads, -1, common) @ vp).reshape(heads, count, group * tokens, dim).transpose(0, 1)
        y = y + weight[..., common:] @ vo
        out.append(y.reshape(count, heads, group, tokens, dim).permute(0, 3, 1, 2, 4).reshape(count * tokens, heads * group, dim))
        first += count
    return torch.cat(out).to(s["dtype"])


# ------------------------------------------------------------------------------------------------ the package's kernels
def _own_sample(s):
    rows = s["case"]["rows"]
    out = torch.empty(rows, dtype=torch.int32, device=DEV)
    logprobs = torch.empty(rows, dtype=torch.float32, device=DEV)
    s["kernels"].sample_filtered(s["logits"], s["temperature"], s["uniform"], out, top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"],
                                 logprobs=logprobs)
    return out, logprobs


def _own_logprobs(s):
    rows = s["case"]["rows"]
    out = torch.empty(rows, dtype=torch.float32, device=DEV)
    ranks = torch.empty(rows, dtype=torch.int32, device=DEV)
    s["kernels"].token_logprobs(s["logits"], s["tokens"], out, ranks=ranks)
    return out, ranks


def _own_attend(s):
    out = torch.empty_like(s["q"])
    s["kernels"].shared_prefix_attention(s["q"], s["pages"], s["tables"], s["cu_q"], s["seq_lens"], s["cu_groups"], s["shared_lens"], out,
                                         s["scale"], s["case"]["window"], s["case"]["tokens"], s["longest"])
    return out


def run(state):
    forms = (dict(sample=_own_sample, logprobs=_own_logprobs, attend=_own_attend) if own else
             dict(sample=_plain_sample, logprobs=_plain_logprobs, attend=_plain_attend))
    return forms[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    width = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "sample":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * width + 28 * case["rows"], flops=3 * n)
    if case["kind"] == "logprobs":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * width + 12 * case["rows"], flops=4 * n)
    members, shared, lens = _layout(case)
    heads, dim, tokens, w = case["kv_heads"], case["dim"], case["tokens"], case["window"]
    owner = [j for j, n in enumerate(members) for _ in range(n)]
    pairs = read = 0
    reach = list(shared)                                                # the first key of a group that some query sees
    for n, j in zip(lens, owner):
        first = max(0, n - tokens - w + 1) if w else 0
        reach[j] = min(reach[j], first)
        read += n - max(first, shared[j])
        pairs += sum(min(p + 1, w) if w else p + 1 for p in range(n - tokens, n))
    read += sum(n - first for n, first in zip(shared, reach))
    rows = len(lens) * tokens * heads * case["group"]
    return dict(bytes=(read * 2 * heads * dim + 2 * rows * dim) * width, flops=4 * pairs * heads * case["group"] * dim)


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "sample":
        return _exact_sample(s)
    if case["kind"] == "logprobs":
        logprob, rank = [], []
        for x, token in zip(s["logits"], s["tokens"].tolist()):
            row = x.double()
            logprob.append(torch.log_softmax(row, dim=0)[token])
            rank.append((row > row[token]).sum() + (row[:token] == row[token]).sum())
        return torch.stack(logprob), torch.stack(rank).to(torch.int32)
    return _exact_attend(case, s)


def _exact_sample(s):
    """Row by row: the tokens that can be drawn are taken one after the other, the best first, until a cut stops them."""
    out, logprob = [], []
    for r in range(s["logits"].shape[0]):
        row = s["logits"][r].double()
        t, k, p, least, u = (s[n][r].double().item() for n in ("temperature", "top_k", "top_p", "min_p", "uniform"))
        best = int(torch.nonzero(row == row.max())[0])
        if t == 0:
            out.append(best)
            logprob.append(torch.zeros((), dtype=torch.float64, device=DEV))
            continue
        prob = torch.softmax(row / t, dim=0)
        order = torch.argsort(row, descending=True, stable=True)
        if k >= 1:
            order = order[:int(k)]
        if p < 1:
            kept = prob[order] / prob[order].sum()
            reached = torch.nonzero(torch.cumsum(kept, dim=0) >= p)
            order = order[:int(reached[0]) + 1] if len(reached) else order
        order = order[prob[order] >= least * prob[best]]
        order = torch.sort(order)[0]
        run = torch.cumsum(prob[order], dim=0)
        out.append(int(order[torch.searchsorted(run, u * run[-1], right=True)]))
        logprob.append(torch.log(prob[out[-1]]) - torch.log(run[-1]))
    return torch.tensor(out, dtype=torch.int32, device=DEV), torch.stack(logprob)


def _exact_attend(case, s):
    heads, group, page, m = case["kv_heads"], case["group"], case["page"], case["tokens"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
    for r, n in enumerate(s["layout"][2]):
        kv = s["pages"][s["tables"][r, :-(-n // page)].long()].double()                      # [pages, 2, heads, page, dim]
        p = torch.arange(n - m, n, device=DEV)[:, None]
        key = torch.arange(n, device=DEV)[None]
        hidden = key > p
        if case["window"]:
            hidden |= key + case["window"] <= p
        for h in range(heads):
            k, v = (kv[:, i, h].reshape(-1, case["dim"])[:n] for i in range(2))
            q = s["q"][r * m:(r + 1) * m, h * group:(h + 1) * group].double()
            score = (torch.einsum("tgd,kd->gtk", q, k) * s["scale"]).masked_fill(hidden, -math.inf)
            out[r * m:(r + 1) * m, h * group:(h + 1) * group] = torch.einsum("gtk,kd->tgd", torch.softmax(score, dim=2), v)
    return out
