"""Drawing under cuts where numbers end (infinities, the smallest temperatures, many rows at once), against the definition in 64 bits."""
import math

import pytest
import torch

from answer_refs import sample_row
from test_sampling_gpu import K, check, draw, logits_of      # noqa: F401 (K: a fixture)

pytestmark = pytest.mark.gpu


def f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


@pytest.mark.parametrize("vocab", [7, 5000, 40001])
def test_infinities_in_many_rows(K, vocab):      # noqa: F811
    """More rows than find room at once (the kernel that keeps none of a row): what a row has does not depend on the batch."""
    rows = 320
    x = logits_of(rows, vocab, 51, torch.float32)
    for r in range(rows):
        if r % 6 == 1:
            x[r, [r % vocab, (r * 7 + 3) % vocab]] = math.inf
        elif r % 6 == 2:
            x[r] = -math.inf
        elif r % 6 == 3:
            x[r, ::2] = math.nan
        elif r % 6 == 4:
            x[r, r % vocab] = 3e38 if r % 4 else -3e38
        elif r % 6 == 5:
            x[r, r % vocab] = math.inf
            x[r, 1::3] = -math.inf if r % 4 else math.nan
    u = torch.rand(rows, generator=torch.Generator().manual_seed(52)).tolist()
    t = [(0.8, 1.0, 0.0, 2.5, math.inf)[r % 5] for r in range(rows)]
    for least in ([0.0] * rows, [(0.05, 1.0, 0.0, 0.5)[r % 4] for r in range(rows)]):
        tokens, logprobs = draw(K, x, t, u, least=least)
        for r in range(rows):
            want, logprob = sample_row(x[r], f32(t[r]), f32(u[r]), 0, 1.0, f32(least[r]))
            assert tokens[r] == want, (r, t[r], least[r])
            if math.isnan(logprob):
                assert math.isnan(logprobs[r])
            else:
                # one rounding to float32 of a difference whose sum of weights is right to 2^-45 times the tokens
                assert abs(logprobs[r] - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -45 * vocab, r
        for part in (list(range(0, 8)), [85, 31, 7], [5]):
            got = draw(K, x[part], [t[r] for r in part], [u[r] for r in part], least=[least[r] for r in part])
            assert got[0] == [tokens[r] for r in part]
            assert all(a == b or (math.isnan(a) and math.isnan(b)) for a, b in zip(got[1], (logprobs[r] for r in part)))


@pytest.mark.parametrize("infinities", [0, 1, 2, 3])
@pytest.mark.parametrize("vocab", [700, 5000, 60001])
def test_infinite_temperatures_under_top_k(K, vocab, infinities):      # noqa: F811
    """Of finite logits each is as likely as the other, beside an infinite one none has a weight: what the first k's list holds is what was counted."""
    rows = 24
    x = logits_of(rows, vocab, 53, torch.float32)
    at = torch.randperm(vocab, generator=torch.Generator().manual_seed(54))[:infinities]
    x[:, at] = math.inf
    x[::4, 1::5] = -math.inf
    x[1::4, ::7] = math.nan
    x[:, at] = math.inf
    u = [(0.0, 0.3, 0.6, 0.95)[r // 6] for r in range(rows)]
    ks = [(1, 2, 3, 50, 511, 512)[r % 6] for r in range(rows)]
    for ps in (None, [(1.0, 0.9, 0.4, 0.0)[r % 4] for r in range(rows)]):
        for t in (math.inf, 3e38, 1e30):
            check(K, x, [t] * rows, u, ks, ps)


@pytest.mark.parametrize("rows", [6, 320])
@pytest.mark.parametrize("vocab", [700, 5000, 60001])
def test_the_smallest_temperatures(K, vocab, rows):      # noqa: F811
    """Below the smallest normal number 1 / T passes what 32 bits hold; logits around zero, differences of ordinary size and of the smallest numbers' size."""
    t = [(1e-45, 1e-43, 1e-41, 1e-40, 3e-39, 1e-38)[r % 6] for r in range(rows)]
    g = torch.Generator().manual_seed(55)
    u = torch.rand(rows, generator=g).tolist()
    x = -torch.rand((rows, vocab), generator=g) - 1e-3
    x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] = 0.0
    y = torch.rand((rows, vocab), generator=g) * torch.tensor(t)[:, None] * 40.0
    y[::2, ::3] = -1.0
    for logits in (x, y - 1e-38):
        check(K, logits, t, u)
        check(K, logits, t, u, least=[(0.0, 0.1, 1.0, 0.5)[r % 4] for r in range(rows)])
        check(K, logits, t, u, k=[(50, 0, 600, 3)[r % 4] for r in range(rows)], p=[(0.9, 0.5, 1.0, 0.97, 0.0)[r % 5] for r in range(rows)])


def test_the_largest_vocabulary_is_what_admission_goes_by(K):      # noqa: F811
    assert K.sample_max_vocab == int(K._sampling_lib().ifb_sample_cut_max_vocab())
