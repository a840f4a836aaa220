"""A tensor of one row (or one column) has a stride that leads nowhere: whatever it is, the calls take it."""
import pytest
import torch

from test_kv8_gpu import on_device, scene

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_row_of_a_product(K, dtype):
    from infurnace_b200.kernels import Mx4Matrix
    x = torch.randn((1, 96), device="cuda").to(dtype)
    odd = x.as_strided((1, 96), (97, 1))
    w = K.mx4_matrix(torch.randn((40, 96), device="cuda"))
    a, b = (torch.empty((1, 40), dtype=dtype, device="cuda") for _ in range(2))
    assert torch.equal(K.mx4_linear(x, w, a), K.mx4_linear(odd, w, b))
    p, q = K.mx4_quantize(x, Mx4Matrix.empty(1, 96)), K.mx4_quantize(odd, Mx4Matrix.empty(1, 96))
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [1, 2])
def test_one_token_and_one_page(K, dtype, heads):
    q, codes, fields, tables, cu, seq = (t.cuda() for t in scene([1], [9], heads, 2, 64, 16, dtype))
    k, v = torch.randn((2, 1, heads, 64), device="cuda").to(dtype)
    slots = torch.tensor([int(tables[0, 0]) * 16 + 8], dtype=torch.int32, device="cuda")
    outs = []
    for odd in (False, True):
        pages = on_device(codes.cpu(), fields.cpu())
        bend = (lambda t, n: t.as_strided(t.shape, (n, *t.stride()[1:]))) if odd else (lambda t, n: t)
        K.kv8_store(bend(k, 131), bend(v, 77), slots, pages)
        out = torch.empty_like(q)
        table = tables.as_strided((1, 1), (1, 5)) if odd else tables
        K.kv8_attention(bend(q, 999), pages, table, cu, seq, out, 0.125, 0, 1, 9)
        outs.append((out, pages.codes, pages.exponents))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
