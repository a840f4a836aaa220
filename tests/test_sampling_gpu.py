"""Drawing under top-k, top-p and min-p and log probabilities of tokens on the device against their statement in 64 bits (tests/answer_refs.py)."""
import math

import pytest
import torch

from answer_refs import logprob_row, sample_row

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


def logits_of(rows, vocab, seed, dtype, spread=2.5):
    g = torch.Generator().manual_seed(seed)
    return (spread * torch.randn((rows, vocab), generator=g)).to(dtype)


def draw(K, logits, temperature, uniform, k=None, p=None, least=None):
    """Tokens and log probabilities, as lists; parameters are lists or None."""
    rows = logits.shape[0]
    dev = logits if logits.is_cuda else logits.cuda()
    out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    logprobs = torch.full((rows,), 7.0, device="cuda")

    def on(x, dtype):
        return None if x is None else torch.tensor(x, dtype=dtype, device="cuda")

    K.sample_filtered(dev, on(temperature, torch.float32), on(uniform, torch.float32), out, on(k, torch.int32), on(p, torch.float32),
                      on(least, torch.float32), logprobs)
    return out.tolist(), logprobs.tolist()


def check(K, logits, temperature, uniform, k=None, p=None, least=None):
    tokens, logprobs = draw(K, logits, temperature, uniform, k, p, least)
    f32 = lambda x: float(torch.tensor(x, dtype=torch.float32))      # parameters as the kernel gets them
    for r in range(logits.shape[0]):
        want, logprob = sample_row(logits[r], f32(temperature[r]), f32(uniform[r]), k[r] if k else 0, f32(p[r]) if p else 1.0,
                                   f32(least[r]) if least else 0.0)
        assert tokens[r] == want, (r, temperature[r], uniform[r], k and k[r], p and p[r], least and least[r])
        if math.isnan(logprob):
            assert math.isnan(logprobs[r])
        else:
            # one rounding to float32 (2^-24) of a difference in 64 bits whose sum of weights is right to 2^-45 times the tokens
            assert abs(logprobs[r] - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -45 * logits.shape[1], (r, logprobs[r], logprob)


VOCABS = [1, 2, 5, 31, 257, 1000, 4099, 20481, 49999, 151936]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_every_cut_is_the_definitions(K, vocab, dtype):
    """Rows with every combination of cuts, off and at their ends."""
    cuts = [(k, p, least) for k in (0, 1, 3, 50, 700, vocab, vocab + 9) for p in (1.0, 0.0, 0.3, 0.95) for least in (0.0, 0.05, 1.0)]
    cuts = cuts[::1 if vocab < 30000 else 3]
    g = torch.Generator().manual_seed(vocab)
    n = len(cuts)
    u = torch.rand(n, generator=g).tolist()
    t = [(0.0, 0.3, 1.0, 1.7)[i % 4] if i % 7 == 0 else 0.4 + 0.1 * (i % 11) for i in range(n)]
    check(K, logits_of(n, vocab, vocab + 1, dtype), t, u, [c[0] for c in cuts], [c[1] for c in cuts], [c[2] for c in cuts])


@pytest.mark.parametrize("vocab", [1, 1000, 151936])
def test_cuts_that_are_absent(K, vocab):
    x = logits_of(6, vocab, 5, torch.float32)
    u = [0.0, 0.1, 0.5, 0.9, 0.999, 1.0 - 2.0 ** -24]
    t = [1.0, 0.7, 2.0, 1.3, 1.0, 1.0]
    check(K, x, t, u)
    check(K, x, t, u, k=[40] * 6)
    check(K, x, t, u, p=[0.9] * 6)
    check(K, x, t, u, least=[0.1] * 6)


def test_the_largest_vocabulary_and_the_one_beyond(K):
    from infurnace_b200.errors import KernelError
    top = int(K._sampling_lib().ifb_sample_cut_max_vocab())
    x = logits_of(2, top, 6, torch.float32)
    check(K, x, [1.0, 1.0], [0.4, 0.8], p=[0.9, 1.0], k=[0, 5000])
    with pytest.raises(KernelError, match="at most"):
        draw(K, torch.zeros((1, top + 1)), [1.0], [0.5])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("distinct", [1, 2, 7, 200])
@pytest.mark.parametrize("vocab", [40, 3000, 60001])
def test_ties_go_by_index(K, vocab, distinct, dtype):
    """Few distinct logits, so that cuts run through thousands of equal ones."""
    g = torch.Generator().manual_seed(distinct)
    x = (torch.randint(0, distinct, (24, vocab), generator=g).float() / 8).to(dtype)
    u = torch.rand(24, generator=g).tolist()
    ks = [0, 1, 17, vocab // 3, vocab - 1, 0] * 4
    ps = [1.0, 1.0, 1.0, 0.6, 1.0, 0.37, 0.5, 0.9] * 3
    check(K, x, [1.0, 0.5, 3.0] * 8, u, ks, ps, [0.0, 0.0, 0.9, 0.0] * 6)


def test_many_values_within_a_part_of_a_bin(K):
    """More than a list of values that differ in their last bits only: a cut is found by halving."""
    base = torch.full((8, 30000), 3.0)
    g = torch.Generator().manual_seed(9)
    x = (base.view(torch.int32) + torch.randint(0, 37, base.shape, generator=g, dtype=torch.int32)).view(torch.float32)
    x[:, ::3] = -4.0
    u = torch.rand(8, generator=g).tolist()
    check(K, x, [1.0] * 8, u, [0, 9000, 1, 19999, 0, 300, 0, 12345], [0.5, 1.0, 1.0, 0.8, 0.01, 1.0, 0.999, 0.3])


@pytest.mark.parametrize("vocab", [6, 5000, 151936])
def test_infinities_and_nan(K, vocab):
    x = logits_of(8, vocab, 8, torch.float32)
    x[0, 1:] = -math.inf                      # one token is left
    x[1, :] = -math.inf                       # none
    x[2, :] = math.nan
    x[3, ::2] = math.nan
    x[4, 3] = x[4, 5] = math.inf              # two infinities share all
    x[5, :vocab // 2] = -math.inf
    x[6, 2] = 3e38
    x[7, :] = -3e38
    for u in (0.0, 0.3, 0.75, 0.99):
        check(K, x, [1.0] * 8, [u] * 8)
        check(K, x, [0.8] * 8, [u] * 8, [0, 0, 3, 3, 1, 3, 0, 2], [0.9, 0.9, 0.9, 1.0, 1.0, 0.5, 0.9, 0.7], [0.0] * 4 + [0.1] * 4)
        check(K, x, [0.0] * 8, [u] * 8)


def test_ends_of_temperature_and_of_the_numbers(K):
    x = logits_of(8, 3001, 11, torch.float32)
    t = [1e-38, 1e-20, 1e-3, 1e3, 1e30, math.inf, -1.0, 0.0]
    for u in (0.0, 0.2, 1.0 - 2.0 ** -24):
        check(K, x, t, [u] * 8)
        check(K, x, t, [u] * 8, [0, 5, 0, 2000, 0, 1500, 3, 3], [0.5, 1.0, 0.9, 0.9, 0.3, 0.7, 0.9, 0.9])
    # numbers outside [0, 1) stay inside the vocabulary
    tokens, _ = draw(K, x, [1.0] * 8, [1.0, 2.0, -1.0, math.nan, math.inf, -math.inf, 1.5, 1e30], p=[0.9] * 8)
    assert all(0 <= tok < 3001 for tok in tokens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,offset,pitch", [(999, 0, 1024), (1000, 1, 1003), (8190, 3, 8197), (151935, 5, 151999)])
def test_rows_that_lie_apart(K, vocab, offset, pitch, dtype):
    whole = logits_of(1, 5 * pitch + offset, 12, dtype)[0]
    rows = whole[offset:offset + 5 * pitch].view(5, pitch)[:, :vocab]
    dev = whole.cuda()[offset:offset + 5 * pitch].view(5, pitch)[:, :vocab]
    u = [0.1, 0.35, 0.6, 0.85, 0.97]
    got = draw(K, dev, [0.9] * 5, u, [0, 0, 20, 0, 90], [1.0, 0.9, 1.0, 0.8, 0.9])
    assert got[0] == [sample_row(rows[i], float(torch.tensor(0.9)), float(torch.tensor(u[i])), [0, 0, 20, 0, 90][i],
                                 float(torch.tensor([1.0, 0.9, 1.0, 0.8, 0.9][i])))[0] for i in range(5)]
    same = rows[:1].expand(5, vocab)
    one = dev[:1].expand(5, vocab)                                             # rows of pitch 0
    assert draw(K, one, [0.9] * 5, u)[0] == draw(K, same.contiguous(), [0.9] * 5, u)[0]


@pytest.mark.parametrize("vocab", [5000, 151936])
def test_a_row_does_not_depend_on_the_others(K, vocab):
    """Bits of a row alone, in a small batch and in one that has other numbers of CTAs a row."""
    x = logits_of(300, vocab, 13, torch.float32).cuda()
    u = torch.rand(300, generator=torch.Generator().manual_seed(1)).tolist()
    ps = [0.9, 1.0, 0.95] * 100
    ks = [0, 0, 50, 900, 0] * 60
    whole = draw(K, x, [1.0] * 300, u, ks, ps)
    for rows in ([0], [1], [4, 5, 6], list(range(37, 80))):
        part = draw(K, x[rows], [1.0] * len(rows), [u[i] for i in rows], [ks[i] for i in rows], [ps[i] for i in rows])
        assert part[0] == [whole[0][i] for i in rows] and part[1] == [whole[1][i] for i in rows]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("left", [1, 2, 31, 33, 511, 512, 513, 600])
@pytest.mark.parametrize("vocab", [700, 50000])
def test_what_a_grammar_leaves(K, vocab, left, dtype):
    """Few tokens above -inf, about as many as a list holds, some of them far below the others; among them infinities and the largest numbers."""
    g = torch.Generator().manual_seed(left)
    x = torch.full((16, vocab), -math.inf)
    for r in range(16):
        at = torch.randperm(vocab, generator=g)[:left]
        x[r, at] = (1.0, 30.0, 1e4, 0.01)[r % 4] * torch.randn(left, generator=g)
        if r == 13:
            x[r, at[:(left + 1) // 2]] = math.inf
        if r == 14:
            x[r, at] = torch.where(torch.rand(left, generator=g) < 0.5, 3e38, -3e38)
        if r == 15:
            x[r, at] = math.nan if left < 3 else 0.0
    u = torch.rand(16, generator=g).tolist()
    ks = [0, 1, 5, left, 0, max(1, left - 1), left + 1, 50] * 2
    check(K, x.to(dtype), [1.0, 0.2, 5.0, 1.0] * 4, u, ks, [0.9, 1.0, 0.5, 0.99, 0.0, 1.0, 0.7, 1.0] * 2, [0.0, 0.0, 0.1, 0.0] * 4)


@pytest.mark.parametrize("vocab", [40000, 97477])
def test_a_row_of_16_bits_does_not_depend_on_the_others(K, vocab):
    """Many rows have half the CTAs each that few have."""
    x = logits_of(150, vocab, 15, torch.bfloat16)
    u = torch.rand(150, generator=torch.Generator().manual_seed(2)).tolist()
    ps, ks = [0.9, 1.0, 0.95] * 50, [0, 0, 50, 900, 0] * 30
    whole = draw(K, x, [1.0] * 150, u, ks, ps)
    for rows in ([7], [4, 5, 6], list(range(100, 130))):
        part = draw(K, x[rows], [1.0] * len(rows), [u[i] for i in rows], [ks[i] for i in rows], [ps[i] for i in rows])
        assert part[0] == [whole[0][i] for i in rows] and part[1] == [whole[1][i] for i in rows]
    check(K, x[:9], [1.0] * 9, u[:9], ks[:9], ps[:9])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_a_high_temperature_puts_many_values_into_a_part_of_a_bin(K, sign, dtype):
    """Thousands of tokens of some hundred neighbouring values: found by halving, of 16-bit logits by their upper halves."""
    g = torch.Generator().manual_seed(12)
    x = (sign * (3.0 + torch.randint(0, 128, (8, 40000), generator=g).float() / 128)).to(dtype)
    u = torch.rand(8, generator=g).tolist()
    check(K, x, [1e4, 3e4, 1e5, 1e4] * 2, u, [0, 30001, 0, 777, 39999, 0, 20000, 1], [0.5, 1.0, 0.97, 0.6, 0.3, 0.0, 1.0, 0.2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,offset", [(3, 1), (20001, 0), (20002, 3), (20003, 6)])
def test_many_rows_without_cuts_that_begin_anywhere(K, vocab, offset, dtype):
    """More rows than find room at once: the kernel that keeps none of a row, from every place within 16 bytes."""
    rows = 320
    wide = torch.full((rows, vocab + 7 + vocab % 2), 50.0).to(dtype)      # an odd pitch; what lies beside a row is larger than all of it
    wide[:, offset:offset + vocab] = logits_of(rows, vocab, 13, dtype)
    held = wide.cuda()[:, offset:offset + vocab]
    u = torch.rand(rows, generator=torch.Generator().manual_seed(14)).tolist()
    t = [(0.0, 0.8, 1.0, 2.5)[r % 4] for r in range(rows)]
    tokens, logprobs = draw(K, held, t, u)
    narrow, least = draw(K, held, t, u, least=[0.05 * (r % 3) for r in range(rows)])
    f32 = lambda x: float(torch.tensor(x, dtype=torch.float32))
    for r in range(rows):
        for got, scores, min_p in ((tokens, logprobs, 0.0), (narrow, least, f32(0.05 * (r % 3)))):
            want, logprob = sample_row(wide[r, offset:offset + vocab], f32(t[r]), f32(u[r]), 0, 1.0, min_p)
            assert got[r] == want, r
            assert abs(scores[r] - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -45 * vocab


def test_no_rows_is_nothing(K):
    assert draw(K, torch.zeros((0, 10)), [], [], [], [], []) == ([], [])
    empty = torch.empty(0, device="cuda")
    K.token_logprobs(torch.zeros((0, 10), device="cuda"), empty.int(), empty)


# ------------------------------------------------------------------------------------------------ log probabilities
def score(K, logits, tokens):
    dev = logits if logits.is_cuda else logits.cuda()
    out = torch.full((len(tokens),), 7.0, device="cuda")
    ranks = torch.full((len(tokens),), -7, dtype=torch.int32, device="cuda")
    K.token_logprobs(dev, torch.tensor(tokens, dtype=torch.int32, device="cuda"), out, ranks)
    return out.tolist(), ranks.tolist()


def check_scores(K, logits, tokens):
    got, ranks = score(K, logits, tokens)
    for r, token in enumerate(tokens):
        want, rank = logprob_row(logits[r], token)
        assert ranks[r] == rank, (r, token)
        if math.isnan(want) or math.isinf(want):
            assert got[r] == want or (math.isnan(want) and math.isnan(got[r])), (r, got[r], want)
            continue
        # A term e^(l - m): two roundings of its exponent, d = l - m and d log2 e (2^-24 of |d| log2 e each, for the terms that count |d| <= 40:
        # 2^-24 * 2 * 40), ex2.approx (2^-22) and the additions of a thread (at most 2^12 of them, 2^-24 each at worst, of random sign: 2^-18
        # bounds them): below 2^-16 of the sum's logarithm's slope s / (1 + s) <= min(1, s), s the sum itself; and one rounding at the end.
        x = logits[r].double()
        top = x.max()
        s = math.expm1(-(top - top - torch.log1p(torch.exp(torch.sort(x, descending=True)[0][1:] - top).sum())).item())
        assert abs(got[r] - want) <= 2.0 ** -24 * abs(want) + 2.0 ** -16 * min(1.0, s), (r, got[r], want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", VOCABS)
def test_scores_are_the_definitions(K, vocab, dtype):
    x = logits_of(9, vocab, vocab, dtype)
    x[8] *= 12                                # rows that are sure
    check_scores(K, x, [0, vocab - 1, vocab // 2, int(x[3].float().argmax()), int(x[4].float().argmin()), vocab // 3, max(0, vocab - 2), -1,
                        int(x[8].float().argmax())])
    check_scores(K, x[:1], [vocab // 2])


def test_scores_of_many_rows(K):
    x = logits_of(1500, 2003, 3, torch.float32)
    tokens = torch.randint(0, 2003, (1500,), generator=torch.Generator().manual_seed(1)).tolist()
    check_scores(K, x, tokens)


def test_a_certain_token_keeps_its_digits(K):
    x = torch.full((1, 1000), -20.0)
    x[0, 17] = 5.0
    got, _ = score(K, x, [17])
    want = -math.log1p(999 * math.exp(-25.0))
    assert abs(got[0] - want) <= 2.0 ** -15 * abs(want)


@pytest.mark.parametrize("vocab", [7, 5000, 151936])
def test_scores_of_infinities_and_nan_and_ties(K, vocab):
    x = logits_of(8, vocab, 21, torch.float32)
    x[0, :] = -math.inf
    x[1, 3] = math.nan
    x[2, 4] = math.inf
    x[3, 1:] = -math.inf
    x[4, :] = 2.5
    x[5, ::2] = -math.inf
    x[6, :] = math.nan
    check_scores(K, x, [1, 2, 4, 1, vocab // 2, 2, 0, vocab])
    check_scores(K, x, [0, 3, 0, 0, vocab - 1, 1, 3, -5])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,offset,pitch", [(999, 0, 1024), (1000, 1, 1003), (8190, 3, 8197), (151935, 5, 151999)])
def test_scores_of_rows_that_lie_apart(K, vocab, offset, pitch, dtype):
    whole = logits_of(1, 5 * pitch + offset, 12, dtype)[0]
    rows = whole[offset:offset + 5 * pitch].view(5, pitch)[:, :vocab]
    dev = whole.cuda()[offset:offset + 5 * pitch].view(5, pitch)[:, :vocab]
    tokens = [0, vocab - 1, 1, vocab // 2, 7]
    assert score(K, dev, tokens) == score(K, rows.contiguous(), tokens)
    check_scores(K, rows, tokens)


# ------------------------------------------------------------------------------------------------ as a program uses them
def test_drawn_tokens_are_scored_in_a_graph_and_on_another_stream(K):
    """What is drawn is scored, recorded and replayed with new logits, and on a stream of its own."""
    rows, vocab = 5, 4099
    x = logits_of(rows, vocab, 31, torch.float32).cuda()
    t, u, p = (torch.full((rows,), v, device="cuda") for v in (0.9, 0.4, 0.9))
    out = torch.empty(rows, dtype=torch.int32, device="cuda")
    logprobs, ranks = torch.empty(rows, device="cuda"), torch.empty(rows, dtype=torch.int32, device="cuda")

    def both():
        K.sample_filtered(x, t, u, out, top_p=p)
        K.token_logprobs(x, out, logprobs, ranks)

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
    for seed in (41, 42):
        x.copy_(logits_of(rows, vocab, seed, torch.float32))
        graph.replay()
        torch.cuda.synchronize()
        replayed = (out.tolist(), logprobs.tolist(), ranks.tolist())
        side = torch.cuda.Stream()
        out.zero_()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            both()
        torch.cuda.synchronize()
        assert replayed == (out.tolist(), logprobs.tolist(), ranks.tolist())
        f = float(torch.tensor(0.9))
        assert replayed[0] == [sample_row(x[i].cpu(), f, float(torch.tensor(0.4)), 0, f)[0] for i in range(rows)]
        assert replayed[2] == [logprob_row(x[i].cpu(), replayed[0][i])[1] for i in range(rows)]
