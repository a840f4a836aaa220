"""Calls over few bits from several host threads on one stream give the bits that they give alone."""
import threading

import pytest
import torch

from test_kv8_gpu import on_device, scene

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from infurnace_b200.kernels import load_cuda_kernels
    return load_cuda_kernels()


def together(works, times):
    """Every work's results in turn, with all works under way at once."""
    results, errors = [[] for _ in works], []

    def go(i):
        try:
            for _ in range(times):
                results[i].append(works[i]())
        except Exception as e:      # noqa: BLE001 (a thread's failure is the test's)
            errors.append(e)
    threads = [threading.Thread(target=go, args=(i,)) for i in range(len(works))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    torch.cuda.synchronize()
    return results


@pytest.mark.parametrize("rows", [40, 300])
def test_products(K, rows):
    g = torch.Generator(device="cuda").manual_seed(rows)
    m = K.mx4_matrix(torch.randn((256, 1024), generator=g, device="cuda").to(torch.bfloat16))

    def work(n):
        x = torch.randn((n, 1024), generator=g, device="cuda").to(torch.bfloat16)

        def call():
            out = torch.empty((n, 256), dtype=torch.bfloat16, device="cuda")
            return K.mx4_linear(x, m, out)
        return call
    works = [work(rows + 7 * i) for i in range(3)]
    alone = [w().clone() for w in works]
    for want, got in zip(alone, together(works, 300)):
        assert all(torch.equal(want, x) for x in got)
    K.check_device_errors()


@pytest.mark.parametrize("q_len,dtype", [(1, torch.bfloat16), (90, torch.bfloat16), (9, torch.float32)])
def test_attention(K, monkeypatch, q_len, dtype):
    monkeypatch.setattr(K, "kv8_split_rows", (0, 0))

    def work(i):
        q, codes, fields, tables, cu, seq = scene([q_len] * (i + 1), [700 + i] * (i + 1), 2, 4, 128, 16, dtype, seed=i)
        pages, q, tables, cu, seq = on_device(codes, fields), q.cuda(), tables.cuda(), cu.cuda(), seq.cuda()

        def call():
            out = torch.empty_like(q)
            return K.kv8_attention(q, pages, tables, cu, seq, out, 128 ** -0.5, 0, q_len, 702, min_q_len=q_len)
        return call
    works = [work(i) for i in range(3)]
    alone = [w().clone() for w in works]
    for want, got in zip(alone, together(works, 200)):
        assert all(torch.equal(want, x) for x in got)
    K.check_device_errors()
