"""Drawing under cuts, log probabilities of tokens and attention over shared pages, stated in 64 bits."""
import math
from fractions import Fraction

import torch


def sample_row(logits, temperature, uniform, k=0, p=1.0, least=0.0):
    """(token, log probability under what the cuts left) of one row; ``uniform`` in [0, 1)."""
    x = logits.double().cpu()
    x = torch.where(x.isnan(), -math.inf, x) + 0.0
    m = x.max().item()
    if m == -math.inf:
        return 0, math.nan
    best = int((x == m).nonzero()[0])
    if not temperature > 0:
        return best, 0.0
    w = torch.exp((x - m) / temperature)
    w = torch.where(x == m, 1.0, torch.where(w.isnan(), 0.0, w))
    order = torch.sort(x, descending=True, stable=True)[1]
    whole = torch.round(w * 2.0 ** 44).to(torch.int64)              # weights count in units of 2^-44 of the largest
    if 1 <= k < len(x):
        order = order[:k]
    if p < 1:
        run = torch.cumsum(whole[order], 0)
        goal = max(1, math.ceil(Fraction(p) * int(run[-1])))
        order = order[run - whole[order] < goal]
    order = order[(w[order] >= least) | (x[order] == m)].sort()[0]
    run = torch.cumsum(whole[order], 0)
    total = int(run[-1])
    token = int(order[int((run <= math.floor(Fraction(uniform) * total)).sum())])
    return token, (0.0 if x[token] == m else (x[token].item() - m) / temperature) - math.log(total / 2.0 ** 44)


def logprob_row(logits, token):
    """(log probability, rank) of one row's token."""
    x = logits.double().cpu()
    if not 0 <= token < len(x):
        return math.nan, -1
    rank = int((x > x[token]).sum() + (x[:token] == x[token]).sum())
    if x.isnan().any() or (x == math.inf).any() or x.max() == -math.inf:
        return math.nan, rank
    rest = torch.sort(x, descending=True)[0]
    return (x[token] - rest[0] - torch.log1p(torch.exp(rest[1:] - rest[0]).sum())).item(), rank


def attention(q, pages, tables, cu_q, seq_lens, cu_groups, shared_lens, scale, window):
    """Each request by itself, over the keys of its own table but for those that its group shares, which are its first request's."""
    n, heads, dim = q.shape
    _, _, kv_heads, page, _ = pages.shape
    group = heads // kv_heads
    out = torch.zeros((n, heads, dim), dtype=torch.float64)
    weight_sum = torch.zeros((n, heads, dim), dtype=torch.float64)          # sum of |weight value|, for tolerances
    for r, length in enumerate(seq_lens):
        rows = range(cu_q[r], cu_q[r + 1])
        if length == 0 or not len(rows):
            continue
        g = next((g for g in range(len(shared_lens)) if cu_groups[g] <= r < cu_groups[g + 1]), None)
        slots = [int(tables[r if g is None or i >= shared_lens[g] else cu_groups[g], i // page]) * page + i % page for i in range(length)]
        slots = torch.tensor(slots)
        kv = pages[slots // page, :, :, slots % page].double()               # [keys, 2, kv_heads, dim]
        for i, row in enumerate(rows):
            p = length - len(rows) + i
            lo = max(0, p - window + 1) if window else 0
            if p < lo:
                continue
            for h in range(heads):
                k, v = kv[lo:p + 1, 0, h // group], kv[lo:p + 1, 1, h // group]
                w = torch.softmax(k @ q[row, h].double() * scale, 0)
                out[row, h] = w @ v
                weight_sum[row, h] = w @ v.abs()
    return out, weight_sum
