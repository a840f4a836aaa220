"""The data of 4-bit matrices without a GPU: layout of the scales, order of gated rows, refusals, and the plain rounding rule."""
import pytest
import torch

from infurnace_b200.errors import KernelError
from infurnace_b200.kernels.low_bits import Kv8Pages, Mx4Matrix
from low_bit_refs import round4


@pytest.mark.parametrize("rows,k", [(1, 32), (33, 96), (128, 128), (130, 160), (300, 1024)])
@pytest.mark.parametrize("gated", [False, True])
def test_parts_come_back(rows, k, gated):
    rows += rows % 2 if gated else 0
    g = torch.Generator().manual_seed(rows + k)
    codes = torch.randint(0, 256, (rows, k // 2), dtype=torch.uint8, generator=g)
    scales = torch.randint(0, 255, (rows, k // 32), dtype=torch.uint8, generator=g)
    m = Mx4Matrix.from_parts(codes, scales, gated=gated)
    back = m.parts()
    assert torch.equal(back[0], codes) and torch.equal(back[1], scales)
    assert m.shape == (rows, k) and m.numel() == rows * k and m.nbytes == codes.numel() + Mx4Matrix.scale_bytes(rows, k)


def test_a_scale_lies_where_the_layout_says():
    """Byte (row % 32) * 16 + (row % 128 / 32) * 4 + block % 4 of the tile (row / 128, block / 4)."""
    rows, k = 200, 300 * 32
    scales = torch.zeros((rows, k // 32), dtype=torch.uint8)
    scales[171, 45] = 9
    m = Mx4Matrix.from_parts(torch.zeros((rows, k // 2), dtype=torch.uint8), scales)
    at = (1 * (-(-k // 128)) + 45 // 4) * 512 + (171 % 32) * 16 + (171 % 128 // 32) * 4 + 45 % 4
    assert m.scales.nonzero().flatten().tolist() == [at]


def test_gated_rows_are_pairs():
    codes = torch.arange(6, dtype=torch.uint8)[:, None].expand(6, 16).contiguous()
    m = Mx4Matrix.from_parts(codes, torch.zeros((6, 1), dtype=torch.uint8), gated=True)
    assert m.codes[:, 0].tolist() == [0, 3, 1, 4, 2, 5]


@pytest.mark.parametrize("rows,k", [(0, 32), (4, 0), (4, 16), (4, 48)])
def test_sizes_that_have_no_matrix(rows, k):
    with pytest.raises(KernelError):
        Mx4Matrix.scale_bytes(rows, k)


def test_refusals_of_the_data():
    codes, scales = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8)
    with pytest.raises(KernelError):
        Mx4Matrix.from_parts(codes, scales[:, :1])
    with pytest.raises(KernelError):
        Mx4Matrix.from_parts(codes[:3], scales[:3], gated=True)
    with pytest.raises(KernelError):
        Mx4Matrix(codes, torch.zeros(100, dtype=torch.uint8), 4, 64)
    with pytest.raises(KernelError):
        Kv8Pages(torch.zeros((3, 2, 2, 16, 64), dtype=torch.int8), torch.zeros((3, 2, 1), dtype=torch.uint8))
    with pytest.raises(KernelError):
        Kv8Pages(torch.zeros((3, 2, 2, 16, 64)), torch.zeros((3, 2, 2), dtype=torch.uint8))


def test_the_plain_rule():
    """Ties to the even code, saturation at 6 units, the largest of a block in [4, 8) units, zeros and infinities."""
    x = torch.zeros((1, 64))
    x[0, :10] = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -7.9, -0.3])
    x[0, 32] = float("inf")
    code, scale, value = round4(x)
    assert scale.tolist() == [[127, 255]]
    assert value[0, :10].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, -6, -0.5] and value[0, 32:].isnan().all()
    assert code[0, :2].tolist() == [6, 0] and int(code[0, 8]) == 15
