"""Attention over 8-bit pages whose steps lie far apart, and whose numbers are large: every row within its own bound, which
counts what the row sees and nothing else."""
import math

import pytest
import torch

from low_bit_refs import attention8
from test_kv8_gpu import attend, bound, scene

pytestmark = pytest.mark.gpu

FORMS = [("tiles", torch.bfloat16), ("whole", torch.bfloat16), ("whole", torch.float32), ("split", torch.bfloat16), ("split", torch.float32)]


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


def choose(K, monkeypatch, form):
    monkeypatch.setattr(K, "kv8_split_rows", (0, 0) if form == "tiles" else (1 << 20, 0))
    monkeypatch.setattr(K, "kv8_whole_rows", 0 if form == "whole" else 1 << 20)


def within(K, s, dim, keys, dtype, window=0):
    ref, mag, reach = attention8(*s, dim ** -0.5, window)
    out = attend(K, *s, window)
    assert out.isfinite().all()
    assert (out.double() - ref).abs().le(bound(ref, mag, reach, dim, keys, dtype)).all()


@pytest.mark.parametrize("form,dtype", FORMS)
@pytest.mark.parametrize("spread", [12, 24, 33, 60])
@pytest.mark.parametrize("dim,group,requests", [(64, 2, 2), (128, 4, 24)])
def test_a_page_of_large_values_that_a_window_has_passed(K, monkeypatch, form, dtype, spread, dim, group, requests):
    """Rows of one tile of which the first see a page whose values are 2^spread larger than all others, and the others do not.
    Many requests leave an item of the split form in one piece, whose warps have several tiles of keys."""
    choose(K, monkeypatch, form)
    s = scene([60] * requests, [400] * requests, 1, group, dim, 16, dtype, seed=spread)
    s[2][s[3][:, 12].long(), 1] = 130 + spread                         # keys 192 .. 207; the window leaves them at row 357
    within(K, s, dim, 400, dtype, window=150)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("spread", [24, 60])
def test_a_page_of_large_values_without_weight(K, dtype, spread):
    """A decoded token gives a page of large values, another one in each request, 2^-65 of the weight: the other keys' part is what it
    has to be.  More requests than CTAs run at a time, so that a warp has several pages."""
    n, dim = 600, 64
    s = scene([1] * n, [300 - r % 7 for r in range(n)], 1, 4, dim, 16, dtype, seed=spread)
    q, codes, fields, tables = s[:4]
    q.copy_((2.1 + torch.rand(q.shape, generator=torch.Generator().manual_seed(1))).to(dtype))
    fields[:, 0] = 127
    page = tables[torch.arange(n), torch.arange(n) % 18].long()
    codes[page, 0] = -128                                              # q . k = -2 sum(q): some 42 below the others
    fields[page, 1] = 130 + spread
    within(K, s, dim, 300, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_len", [1, 30])
@pytest.mark.parametrize("up", [False, True])
def test_steps_that_rise_while_weights_fall(K, dtype, q_len, up):
    """Page by page the values' step grows by 2^3 and the weight shrinks as much, so that all pages count alike; and the other way."""
    n, dim, requests = 29 * 16, 64, 600 if q_len == 1 else 40
    s = scene([q_len] * requests, [n] * requests, 1, 2, dim, 16, dtype, seed=3)
    q, codes, fields, tables = s[:4]
    q.zero_()
    q[:, :, 0] = 8 * 3 * math.log(2.0)                                 # a code of keys of step 1 is 3 in log2 of the weight
    fields[:, 0] = 133
    for i in range(29):
        p = tables[:, i].long()
        codes[p, 0, :, :, 0] = 14 - i if up else i - 14
        fields[p, 1] = 85 + 3 * (i if up else 28 - i)
    within(K, s, dim, n, dtype)


@pytest.mark.parametrize("form,dtype", [f for f in FORMS if f[0] != "tiles"])
@pytest.mark.parametrize("q_len", [1, 30])
@pytest.mark.parametrize("field,rise", [(254, 0.0), (254, 0.5), (235, 0.5), (200, 2.0), (195, 3.0)])
def test_sums_of_large_values(K, monkeypatch, form, dtype, q_len, field, rise):
    """Values up to the largest float, and scores that rise from page to page (by ``rise`` in log2): what is finite stays finite."""
    choose(K, monkeypatch, form)
    n, dim, requests = 20 * 16, 64, 600 if q_len == 1 else 40
    s = scene([q_len] * requests, [n] * requests, 1, 2, dim, 16, dtype, seed=5)
    q, codes, fields, tables = s[:4]
    q.zero_()
    q[:, :, 0] = 8 * rise * math.log(2.0)
    fields[:, 0], fields[:, 1] = 133, field
    for i in range(20):
        codes[tables[:, i].long(), 0, :, :, 0] = i - 10
    codes[:, 1].clamp_(-126, 125)                                      # (a weighted mean's rounding stays below the largest float)
    within(K, s, dim, n, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("field", [20, 90, 127, 150, 190, 220])
@pytest.mark.parametrize("keys", [1, 2, 9, 40])
def test_few_keys_with_values_of_any_size(K, dtype, field, keys):
    """Where few keys leave little to the bound but the weights' own rounding: a weight's unit is the same in the products and beside them."""
    n = 40
    s = scene([1] * n, [keys] * n, 2, 4, 64, 16, dtype, seed=field + keys)
    s[2][:, 1] = field + torch.randint(0, 20, s[2][:, 1].shape, generator=torch.Generator().manual_seed(keys)).to(torch.uint8)
    within(K, s, 64, keys, dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q_len", [1, 20])
def test_small_weights_beside_zeros(K, dtype, q_len):
    """The keys of all the weight have values of zero; of the others, 2^-150 and 2^-92 of it, in this order, the larger make the output."""
    n, dim, requests = 9 * 16, 64, 600 if q_len == 1 else 40
    s = scene([q_len] * requests, [n] * requests, 1, 2, dim, 16, dtype, seed=7)
    q, codes, fields, tables = s[:4]
    q.zero_()
    q[:, :, 0] = 8 * math.log(2.0)
    fields[:, 0], fields[:, 1] = 133, 125
    codes[:, 0, :, :, 0] = -128
    for page, code in ((0, 100), (1, -50), (8, 8)):
        codes[tables[:, page].long(), 0, :, :, 0] = code
    fields[tables[:, 0].long(), 1] = 0
    within(K, s, dim, n, dtype)
