"""4-bit matrices on the device against their plain statement in 64 bits (tests/low_bit_refs.py): rounding bit for bit, products
within the bound of a float32 sum and the output's rounding."""
import math

import pytest
import torch

from low_bit_refs import round4

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


def rows_of(rows, k, seed, dtype):
    """Rows with features of very different size, zeros, whole blocks of zeros and exact ties."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, k), generator=g) * torch.exp(2 * torch.randn((1, k), generator=g))
    x[torch.rand((rows, k), generator=g) < 0.05] = 0.0
    x[0, :32] = 0.0
    x[-1, -32:] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -4.5, -0.25, -5.0, 7.0, -7.75, 6.0, 0.5, 1.0] * 2) * 0.125
    return x.to(dtype)


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (128, 128), (131, 4096), (257, 1120)])
def test_rounding_is_the_definitions_bit_for_bit(K, dtype, rows, k):
    from infurnace_b200.kernels import Mx4Matrix
    x = rows_of(rows, k, rows * k, dtype)
    code, scale, value = round4(x)
    m = K.mx4_quantize(x.cuda(), Mx4Matrix.empty(rows, k))
    codes, scales = (t.cpu() for t in m.parts())
    assert torch.equal(scales.long(), scale)
    assert torch.equal(codes & 15, code[:, 0::2].to(torch.uint8)) and torch.equal(codes >> 4, code[:, 1::2].to(torch.uint8))
    for out_dtype in DTYPES:
        out = torch.empty((rows, k), dtype=out_dtype, device="cuda")
        assert torch.equal(K.mx4_values(m, out).cpu().double(), value)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_nan_and_the_ends_of_the_range(K, dtype):
    """A block with an infinity or a NaN is NaN and its neighbours are not; the largest and the smallest numbers round like others."""
    from infurnace_b200.kernels import Mx4Matrix
    x = torch.ones((4, 160))
    x[0, 3], x[1, 70], x[2, 159] = math.inf, -math.inf, math.nan
    x[3, :32] *= 3.0e38
    x[3, 32:64] *= 2.0 ** -126
    x[3, 64:96] *= 2.0 ** -124
    x[3, 96:100] = torch.tensor([3.3e38, 1e-38, -1e-38, 2.0 ** 125])
    x = x.to(dtype)
    _, scale, value = round4(x)
    m = K.mx4_quantize(x.cuda(), Mx4Matrix.empty(4, 160))
    assert torch.equal(m.parts()[1].cpu().long(), scale) and (scale == 255).sum() == 3
    out = torch.empty((4, 160), dtype=torch.float32, device="cuda")
    assert same(K.mx4_values(m, out).cpu().double(), value)


@pytest.mark.parametrize("rows,k", [(70001, 64), (262147, 32), (20001, 2080)])
def test_more_rows_than_a_grid_has(K, rows, k):
    """Rows in several launches, and rows four to a thread."""
    from infurnace_b200.kernels import Mx4Matrix
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((rows, k), generator=g, device="cuda").to(torch.bfloat16)
    m = K.mx4_quantize(x, Mx4Matrix.empty(rows, k))
    out = torch.empty_like(x)
    K.mx4_values(m, out)
    for at in (0, 65270, 130540, rows - 300):
        if at < rows:
            part = x[at:at + 300]
            assert torch.equal(out[at:at + 300].double().cpu(), round4(part.cpu())[2])


def test_no_rows(K):
    assert K.mx4_linear(torch.empty((0, 64), device="cuda"), K.mx4_matrix(torch.ones((5, 64), device="cuda")), torch.empty((0, 5), device="cuda")).shape == (0, 5)


def test_a_matrix_is_written_before_the_next_call_reads_it(K):
    """A product may ask for its matrix before the kernel ahead of it ends: not one that writes the matrix, be it with bits or as numbers."""
    from infurnace_b200.kernels import Mx4Matrix
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn((4, 2048), generator=g, device="cuda").to(torch.bfloat16)
    ws = [torch.randn((20000, 2048), generator=g, device="cuda").to(torch.bfloat16) * 2 ** i for i in range(3)]
    shared, numbers = Mx4Matrix.empty(20000, 2048), torch.empty((20000, 2048), dtype=torch.bfloat16, device="cuda")
    want = []
    for w in ws:
        m = K.mx4_matrix(w)
        K.mx4_values(m, numbers)
        torch.cuda.synchronize()
        want.append((torch.empty((4, 20000), device="cuda"), torch.empty((4, 20000), dtype=torch.bfloat16, device="cuda")))
        K.mx4_linear(x, m, want[-1][0])
        K.linear(x, numbers, want[-1][1])
    torch.cuda.synchronize()
    for i in range(12):
        K.mx4_quantize(ws[i % 3], shared)
        a, b = torch.empty((4, 20000), device="cuda"), torch.empty((4, 20000), dtype=torch.bfloat16, device="cuda")
        K.mx4_linear(x, shared, a)
        K.mx4_values(shared, numbers)
        K.linear(x, numbers, b)
        assert torch.equal(a, want[i % 3][0]) and torch.equal(b, want[i % 3][1])


def test_rows_that_lie_apart_and_gated_rows(K):
    from infurnace_b200.kernels import Mx4Matrix
    wide = rows_of(10, 256, 1, torch.bfloat16).cuda()
    x = wide[:, 64:192]
    m = K.mx4_quantize(x, Mx4Matrix.empty(10, 128))
    assert torch.equal(m.codes, K.mx4_quantize(x.contiguous(), Mx4Matrix.empty(10, 128)).codes)
    g = K.mx4_matrix(x.contiguous(), gated=True)
    plain, gated = m.parts(), g.parts()
    assert torch.equal(plain[0], gated[0]) and torch.equal(plain[1], gated[1])
    a, b = torch.empty((10, 128), device="cuda"), torch.empty((10, 128), device="cuda")
    assert torch.equal(K.mx4_values(m, a), K.mx4_values(g, b))


def product(xv, wv, epilogue):
    """The product of values in 64 bits, and the sum of magnitudes that bounds a float32 sum's error."""
    y, mag = xv @ wv.T, xv.abs() @ wv.abs().T
    if epilogue == "silu_gate":
        o = y.shape[1] // 2
        g, u = y[:, :o], y[:, o:]
        act = g * torch.sigmoid(g)
        # |d silu| <= 1.1: errors of the gate reach the product through the up half, and the other way round
        return act * u, 1.1 * mag[:, :o] * u.abs() + act.abs() * mag[:, o:]
    if epilogue == "relu2":
        return y.clamp(min=0) ** 2, 2 * y.abs() * mag
    return y, mag


def check(y, ref, mag, k, dtype):
    # a sum of k float32 terms in any order is off by at most k 2^-24 of the magnitudes' sum (2^-23: a sum that truncates);
    # the gate's exponential adds a few 2^-24 of the result; the output's own rounding is half a unit in its last place
    bound = (k * 2.0 ** -23 + 2.0 ** -20) * mag + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -20) * ref.abs() + 1e-30
    assert (y.double().cpu() - ref).abs().le(bound).all()


SIZES = [(1, 32, 1), (1, 1024, 4096), (2, 64, 127), (8, 12288, 130), (15, 96, 129), (16, 2048, 128), (17, 288, 300), (33, 4096, 514),
         (64, 512, 1000), (65, 1120, 258), (128, 768, 128), (129, 1024, 260), (193, 2048, 1024), (256, 256, 256), (257, 4096, 385),
         (700, 160, 130), (1025, 544, 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,features", SIZES)
@pytest.mark.parametrize("epilogue", ["none", "silu_gate"])
def test_product(K, dtype, rows, k, features, epilogue):
    gated = epilogue == "silu_gate"
    x, w = rows_of(rows, k, 1, dtype), rows_of(features * (2 if gated else 1), k, 2, torch.bfloat16) * 0.1
    ref, mag = product(round4(x)[2], round4(w)[2], epilogue)
    m = K.mx4_matrix(w.cuda(), gated=gated)
    out = torch.full((rows, features), math.nan, dtype=dtype, device="cuda")
    K.mx4_linear(x.cuda(), m, out, epilogue=epilogue)
    K.check_device_errors()
    check(out, ref, mag, k, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,features", [(129, 32, 8), (256, 256, 256), (300, 1120, 258), (257, 4096, 385), (513, 160, 130), (700, 96, 1001),
                                             (1030, 544, 1000), (2048, 512, 304)])
@pytest.mark.parametrize("epilogue", ["none", "silu_gate"])
def test_product_over_pairs_of_sms(K, dtype, rows, k, features, epilogue):
    """The kernel for many rows at sizes that the rule gives to others: rows of the output on 16 bytes (stored by TMA) and not."""
    gated = epilogue == "silu_gate"
    x, w = rows_of(rows, k, 11, dtype), rows_of(features * (2 if gated else 1), k, 12, torch.bfloat16) * 0.1
    ref, mag = product(round4(x)[2], round4(w)[2], epilogue)
    room = torch.full((rows + 2, features), 7.0, dtype=dtype, device="cuda")
    out = room[:rows]
    K.mx4_linear(x.cuda(), K.mx4_matrix(w.cuda(), gated=gated), out, epilogue=epilogue, nt=256)
    K.check_device_errors()
    check(out, ref, mag, k, dtype)
    assert (room[rows:] == 7.0).all()                                  # nothing is written behind the last row


@pytest.mark.parametrize("epilogue,dtype", [("none", torch.bfloat16), ("silu_gate", torch.bfloat16), ("none", torch.float32), ("relu2", torch.bfloat16)])
def test_product_that_the_rule_gives_to_pairs(K, epilogue, dtype):
    """Several rounds of tiles per pair."""
    gated = epilogue == "silu_gate"
    rows, k, features = 1100, 288, 6500 if not gated else 3300
    x, w = rows_of(rows, k, 13, dtype), rows_of(features * (2 if gated else 1), k, 14, torch.bfloat16) * 0.1
    ref, mag = product(round4(x)[2], round4(w)[2], epilogue)
    out = torch.full((rows, features), math.nan, dtype=dtype, device="cuda")
    K.mx4_linear(x.cuda(), K.mx4_matrix(w.cuda(), gated=gated), out, epilogue=epilogue)
    K.check_device_errors()
    check(out, ref, mag, k, dtype)


@pytest.mark.parametrize("rows,nt,splits", [(5, 16, 1), (5, 32, 3), (40, 64, 8), (40, 128, 5), (200, 128, 7), (16, 64, 2)])
def test_tiles_and_shares_that_the_rule_does_not_choose(K, rows, nt, splits):
    from infurnace_b200.kernels import Mx4Matrix
    x, w = rows_of(rows, 2208, 15, torch.bfloat16), rows_of(300, 2208, 16, torch.bfloat16) * 0.1
    q = K.mx4_quantize(x.cuda(), Mx4Matrix.empty(rows, 2208))
    out = torch.full((rows, 300), math.nan, device="cuda")
    K.mx4_linear(q, K.mx4_matrix(w.cuda()), out, nt=nt, splits=splits)
    K.check_device_errors()
    check(out, *product(round4(x)[2], round4(w)[2], "none"), 2208, torch.float32)


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_rounded_rows_unary_epilogues_and_mixed_types(K, rows):
    """Rows that are rounded once serve several products; the output's type is free of the input's; a unary epilogue."""
    from infurnace_b200.kernels import Mx4Matrix
    x, w = rows_of(rows, 352, 3, torch.bfloat16), rows_of(200, 352, 4, torch.bfloat16) * 0.1
    xv, wv = round4(x)[2], round4(w)[2]
    m, q = K.mx4_matrix(w.cuda()), K.mx4_quantize(x.cuda(), Mx4Matrix.empty(rows, 352))
    for epilogue, dtype in (("none", torch.float32), ("relu2", torch.bfloat16), ("relu2", torch.float32)):
        out = torch.empty((rows, 200), dtype=dtype, device="cuda")
        again = torch.empty_like(out)
        K.mx4_linear(q, m, out, epilogue=epilogue)
        K.mx4_linear(x.cuda(), m, again, epilogue=epilogue)
        assert torch.equal(out, again)
        check(out, *product(xv, wv, epilogue), 352, dtype)


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_a_blocks_nan_stays_in_its_row(K, rows):
    """A NaN or infinity in one row of x makes that row of the product NaN and leaves the others alone."""
    x, w = rows_of(rows, 256, 5, torch.bfloat16), rows_of(140, 256, 6, torch.bfloat16)
    bad = rows // 2
    clean = torch.empty((rows, 140), device="cuda")
    K.mx4_linear(x.cuda(), K.mx4_matrix(w.cuda()), clean)
    for v in (math.nan, math.inf):
        x[bad, 77] = v
        out = torch.empty((rows, 140), device="cuda")
        K.mx4_linear(x.cuda(), K.mx4_matrix(w.cuda()), out)
        assert out[bad].isnan().all()
        keep = torch.arange(rows) != bad
        assert torch.equal(out[keep], clean[keep])


def test_another_stream_and_a_graph(K):
    """The call runs on torch's current stream, a recorded one included, and gives the same bits there."""
    x, w = rows_of(40, 512, 7, torch.bfloat16).cuda(), rows_of(300, 512, 8, torch.bfloat16).cuda()
    m = K.mx4_matrix(w)
    a, b, c = (torch.zeros((40, 300), device="cuda") for _ in range(3))
    K.mx4_linear(x, m, a)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        K.mx4_linear(x, m, b)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.mx4_linear(x, m, c)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(a, b) and torch.equal(a, c)


def test_refusals(K):
    from infurnace_b200.errors import KernelError
    from infurnace_b200.kernels import Mx4Matrix
    x, w = torch.zeros((4, 64), device="cuda"), torch.zeros((6, 64), device="cuda")
    m, g = K.mx4_matrix(w), K.mx4_matrix(w, gated=True)
    out = torch.empty((4, 6), device="cuda")
    for call in (lambda: K.mx4_quantize(x.half(), Mx4Matrix.empty(4, 64)), lambda: K.mx4_quantize(x, Mx4Matrix.empty(5, 64)),
                 lambda: K.mx4_quantize(x.cpu(), Mx4Matrix.empty(4, 64)), lambda: K.mx4_quantize(x.t(), Mx4Matrix.empty(64, 4)),
                 lambda: K.mx4_quantize(torch.zeros((4, 65), device="cuda")[:, 1:], Mx4Matrix.empty(4, 64)),
                 lambda: K.mx4_values(m, out), lambda: K.mx4_matrix(w[:5], gated=True), lambda: K.mx4_matrix(w[:, :40]),
                 lambda: K.mx4_linear(x, m, out, epilogue="swish"), lambda: K.mx4_linear(x, m, out, epilogue="silu_gate"),
                 lambda: K.mx4_linear(x, g, out), lambda: K.mx4_linear(x[:, :32], m, out), lambda: K.mx4_linear(x, m, out[:3]),
                 lambda: K.mx4_linear(x, m, out.half()), lambda: K.mx4_linear(x, m, out.cpu()), lambda: K.mx4_linear(g, m, out),
                 lambda: K.mx4_linear(x[0], m, out), lambda: K.mx4_quantize(x[0], m)):
        with pytest.raises(KernelError):
            call()
