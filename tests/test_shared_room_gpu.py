"""The room of attention over shared pages: what a call writes lies within it, and it is no larger than the kernels that the call takes can use."""
import pytest
import torch

from test_shared_prefix_gpu import SCENES, K, Scene      # noqa: F401 (K: a fixture)

pytestmark = pytest.mark.gpu

SHAPES = [(64, 16, 2, 2), (128, 16, 1, 4), (128, 24, 2, 5), (96, 32, 1, 16), (64, 16, 1, 17), (128, 8, 1, 33), (144, 16, 2, 2), (256, 16, 1, 8), (256, 24, 1, 24)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,page,kv_heads,group", SHAPES)
@pytest.mark.parametrize("name", ["uneven", "questions", "full-tiles", "many", "nothing-shared", "empty-requests"])
def test_nothing_is_written_behind_the_room(K, name, dim, page, kv_heads, group, dtype):      # noqa: F811
    scene = {**SCENES[name], "page": page, "kv_heads": kv_heads, "group": group, "dim": dim}
    s = Scene(**scene, dtype=dtype, seed=71)
    size = K.shared_prefix_room(s.rows, len(s.lens), len(s.shared), kv_heads * group, kv_heads, dim, dtype)
    whole = torch.full((size + (1 << 20),), 255, dtype=torch.uint8, device="cuda")      # NaN wherever it is read as numbers
    out = s.run(K, room=whole[:size])
    assert (whole[size:] == 255).all()
    assert torch.equal(out, s.run(K))
    s.check(out)
    K.check_device_errors()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim,page,kv_heads,group", SHAPES)
@pytest.mark.parametrize("tokens,requests,groups", [(8192, 1, 0), (8192, 1, 1), (4001, 7, 3), (64, 64, 1), (1, 1, 0)])
def test_a_room_is_for_one_kernels_rows(K, tokens, requests, groups, dim, page, kv_heads, group, dtype):      # noqa: F811
    """A row's sums over shared keys and over its own: twice the output's numbers in 32 bits, in tiles of up to `rows` score rows.  Beside them tiles that are not full
    (an owner's last, and what a tile of whole tokens leaves empty), and a tile for each worker."""
    size = K.shared_prefix_room(tokens, requests, groups, kv_heads * group, kv_heads, dim, dtype)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    # (rows of a tile, workers of an SM)
    every = [(64, 2)] if dtype is torch.float32 else [(16, 8)] if group <= 16 else [(64, 1)]
    forms = every if dtype is torch.float32 or dim > 128 else [*every, (128, 1)]
    if dtype is torch.bfloat16 and dim <= 128 and group <= 16:
        # large tiles for the wide owners, and beside them one tile of sixteen rows for each that is not
        beside = ((requests + groups) * kv_heads + 8 * sms) * 16
    else:
        beside = 0
    most = 0
    for rows, workers in forms:
        tiles = 2 * (tokens // (rows // group) + 1) + requests + groups
        most = max(most, (tiles * kv_heads + workers * sms) * rows)
    bound = (most + beside) * (dim + 4) * 4 + tokens * 16 + 4096
    assert size <= bound, (size, bound)
