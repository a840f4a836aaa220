"""Calls of attention over shared pages whose tensors lie where the kernels' wide accesses cannot reach them."""
import pytest
import torch

from infurnace_b200.errors import KernelError
from test_answers_cpu import BF16, K, Tensor, shared_args      # noqa: F401 (K: a fixture)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("offset", [2, 4, 8, 14])
def test_an_output_off_a_boundary_of_16_bytes_is_refused(K, dtype, offset):      # noqa: F811
    """A contiguous one may begin anywhere in a larger tensor; results of whole items are written 8 and 16 bytes at a time."""
    args = dict(q=Tensor((5, 8, 64), dtype), kv_pages=Tensor((20, 2, 2, 16, 64), dtype))
    with pytest.raises(KernelError, match="16 bytes"):
        K.shared_prefix_attention(**shared_args(**args, out=Tensor((5, 8, 64), dtype, at=4096 + offset)))
    assert K.launches == 0
    K.shared_prefix_attention(**shared_args(**args, out=Tensor((5, 8, 64), dtype, at=4096 + 16)))
    assert K.launches > 0
