"""Matrices in 4 bits that torch's kernels wrote, and products that follow at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


@pytest.mark.parametrize("rows", [4, 40, 700])
def test_a_product_waits_for_parts_and_copies(K, rows):
    from infurnace_b200.kernels import Mx4Matrix
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn((rows, 2048), generator=g, device="cuda").to(torch.bfloat16)
    made = [K.mx4_matrix(torch.randn((12000, 2048), generator=g, device="cuda") * 2 ** i) for i in range(3)]
    parts, want = [m.parts() for m in made], []
    for m in made:
        torch.cuda.synchronize()
        want.append(K.mx4_linear(x, m, torch.empty((rows, 12000), dtype=torch.bfloat16, device="cuda")))
    shared = Mx4Matrix.empty(12000, 2048)
    for i in range(9):
        a, b = (torch.empty((rows, 12000), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        K.mx4_linear(x, Mx4Matrix.from_parts(*parts[i % 3]), a)
        shared.codes.copy_(made[i % 3].codes)
        shared.scales.copy_(made[i % 3].scales)
        K.mx4_linear(x, shared.written(), b)
        assert torch.equal(a, want[i % 3]) and torch.equal(b, want[i % 3])
    K.check_device_errors()
