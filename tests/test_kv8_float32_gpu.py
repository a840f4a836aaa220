"""How close attention over 8-bit pages in float32 comes to 64 bits for keys, values and queries of ordinary size."""
import pytest
import torch

from low_bit_refs import attention8
from test_kv8_gpu import on_device

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


@pytest.mark.parametrize("q_lens,lens", [([1, 1, 1], [1500, 900, 333]), ([70], [600]), ([200, 1], [200, 40])])
@pytest.mark.parametrize("dim", [64, 128])
def test_float32_keeps_the_bits_of_three_bytes(K, q_lens, lens, dim):
    """The roundings, as independent errors.  Scores of standard deviation 1 (the largest seen 4, 6 in log2): four float32 roundings of
    2^-25 of them each, and queries off by 2^-24 of the row's largest (3.5) along keys of size 1, leave a weight off by 2e-7.  A weight is
    rounded to 2^-25 of the largest of 32 keys; its exponential is off by 2^-22.5 (twice: weights and their unit), 2.4e-7; the unit's
    exponent, near 100, is rounded to 2^-19 at most for all keys of a tile alike, 6.6e-7 at the very most and half of it in the mean.  Together
    some 5e-7 of the output; twice that is the bound.  (Queries and weights of two half-precision terms: 1.4e-6 and more.)"""
    g = torch.Generator().manual_seed(dim + len(lens))
    heads, group, ps = 2, 4, 16
    held = [-(-n // ps) for n in lens]
    codes = torch.zeros((sum(held), 2, heads, ps, dim), dtype=torch.int8)
    fields = torch.zeros((sum(held), 2, heads), dtype=torch.uint8)
    pages = on_device(codes, fields)
    tables = torch.full((len(lens), max(held)), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(lens):
        tables[r, :held[r]] = torch.arange(at, at + held[r])
        k, v = torch.randn((2, n, heads, dim), generator=g).cuda()
        K.kv8_store(k, v, torch.arange(at * ps, at * ps + n, dtype=torch.int32, device="cuda"), pages)
        at += held[r]
    cu = torch.tensor([0] + q_lens).cumsum(0).to(torch.int32)
    seq = torch.tensor(lens, dtype=torch.int32)
    q = torch.randn((int(cu[-1]), heads * group, dim), generator=g)
    out = torch.empty(q.shape, device="cuda")
    K.kv8_attention(q.cuda(), pages, tables.cuda(), cu.cuda(), seq.cuda(), out, dim ** -0.5, 0, max(q_lens), max(lens))
    ref = attention8(q, pages.codes.cpu(), pages.exponents.cpu(), tables, cu, seq, dim ** -0.5)[0]
    assert float((out.cpu().double() - ref).norm() / ref.norm()) <= 1e-6
