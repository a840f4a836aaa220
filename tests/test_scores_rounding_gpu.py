"""What log probabilities lose by rounding where a row's best tokens come late, far above what a thread saw first."""
import pytest
import torch

from test_sampling_gpu import K, check_scores, score      # noqa: F401 (K: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1500, 4000), (40, 8001), (700, 9999), (60, 60000)])
@pytest.mark.parametrize("above", [3.0, 17.0, 37.0, 39.0, 45.0])
def test_near_equal_tokens_far_above_the_others(K, rows, vocab, above, dtype):      # noqa: F811
    """Three of them: the one that is scored, and two side by side, which one thread has."""
    g = torch.Generator().manual_seed(61)
    low = (8.0 * torch.rand((rows, 1), generator=g)).to(dtype).float()
    top = (low + above + 0.5 * torch.rand((rows, 3), generator=g)).to(dtype).float()
    x = low.expand(rows, vocab).clone()
    pair = vocab // 2 + 16 * torch.randint(0, vocab // 32 - 1, (rows, 1), generator=g)
    at = torch.cat((torch.randint(0, vocab // 2, (rows, 1), generator=g), pair, pair + 1), dim=1)
    x.scatter_(1, at, top)
    got, ranks = score(K, x.to(dtype), at[:, 0].tolist())
    y = x.double()
    want = torch.log_softmax(y, dim=1).gather(1, at[:, :1])[:, 0]
    assert ranks == [sum(b > a for b in (b1, b2)) for a, b1, b2 in top.tolist()]
    # s: the sum over all but the best.  A term d below the best: d rounded (2^-24 of it), times log2 e (that number's own rounding 2^-25, the product's 2^-24),
    # ex2.approx (2^-22), and as much once more where its sum is brought from one best to the next (of three there are two steps, together d); four roundings where it is
    # added and multiplied: (2.5 d + 3 * 4 + 4) 2^-24.  The small ones, n of them `above` below, meet in sums of at most n / 256 + 40 additions of 2^-24 each besides.
    # Both through the slope of log(1 + s), 1 / (1 + s); one rounding at the end.
    d = y.max(dim=1, keepdim=True)[0] - top.double()
    near = torch.exp(-d)
    others = near.sum(dim=1) - 1
    small = (vocab - 3) * torch.exp(low[:, 0].double() - y.max(dim=1)[0])
    error = (near * (2.5 * d + 16)).sum(dim=1) - 16 + small * (2.5 * above + 2.5 + 16 + vocab / 256 + 40)
    bound = 2.0 ** -24 * (want.abs() + error / (1 + others + small))
    off = (torch.tensor(got, dtype=torch.float64) - want).abs()
    print("largest share of the bound %.2f, off %.2g" % ((off / bound).max(), off.max()))
    assert (off <= bound).all(), ((off / bound).max(), off.max())


def test_scores_of_rows_that_rise_and_fall(K):      # noqa: F811
    """A largest number that grows with every vector, or never; -inf first, and steps beyond what an exponential in 32 bits reaches."""
    n = 30011
    ramp = torch.arange(n, dtype=torch.float32)
    rows = [ramp * 1e-3, ramp * 0.5, -ramp * 0.5, ramp * 1e30, torch.where(ramp < n // 2, -float("inf"), ramp * 1e-3), (ramp % 977) * 0.3,
            torch.where(ramp % 2 == 0, -3e38, 3e38), torch.where(ramp == n - 1, 100.0, -float("inf"))]
    x = torch.stack(rows)
    check_scores(K, x, [n - 1, n - 1, 0, n - 1, n - 1, 976, 1, n - 1])
    other = [0, n - 2, 1, 7, n - 3, 975, 0, n - 1]
    check_scores(K, x[[0, 1, 2, 3, 4, 5, 7]], other[:6] + other[7:])
    assert score(K, x, other)[0][6] == -float("inf")      # -6e38 is more than 32 bits hold
