"""attn_weights and kv_evict on pages gigabytes apart, K and V rows and weights of a page side by side in one buffer."""
import numpy as np
import pytest

from test_kv_evict_gpu import added64, check, entries, run_weights, same_after
from test_pages_gpu import Cache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    import torch

    import openasr_b200 as ob

    b = ob.Backend(0)
    b.set_stream(torch.cuda.current_stream())
    yield b
    b.close()


def blobs(c, w, stride):
    """views of one buffer in which a page's K rows, V rows and weights follow each other, pages `stride` bytes apart"""
    import torch

    rows = c.HKV * c.page * c.D
    buf = torch.empty(stride * (c.L * c.P - 1) + 4 * rows + 4 * c.HKV * c.page, dtype=torch.uint8, device="cuda")
    half, single = buf.view(torch.float16), buf.view(torch.float32)
    shape, at = (c.L * c.P, c.HKV, c.page, c.D), (stride // 2, c.page * c.D, c.D, 1)
    k, v = (torch.as_strided(half, shape, at, o) for o in (0, rows))
    weights = torch.as_strided(single, shape[:3], (stride // 4, c.page, 1), rows)
    for view, a in ((k, c.k), (v, c.v), (weights, w)):
        view.copy_(torch.from_numpy(a))
    return k, v, weights


@pytest.mark.parametrize("H,HKV,D,N", [(4, 2, 64, 3), (4, 1, 128, 30)])
@pytest.mark.parametrize("stride", [1 << 16, 1_300_000_256])
def test_attn_weights_over_far_pages(be, H, HKV, D, N, stride):
    rng = np.random.default_rng(D)
    c = Cache(rng, 1, N, HKV, D, 24, [60], spare=1)
    q, old = rng.standard_normal((1, H, N, D)).astype(np.float32), entries(rng, c)
    k, _, w = blobs(c, old, stride)
    want, tol = added64(c, q, [N], 0.1, 0.5, old)
    check(run_weights(be, c, q, None, 0.1, 0.5, old, k=k, w_view=w), want, tol)


@pytest.mark.parametrize("D,L", [(64, 1), (128, 2)])
@pytest.mark.parametrize("stride", [1 << 16, 900_000_256])
def test_kv_evict_over_far_pages(be, D, L, stride):
    rng = np.random.default_rng(D)
    c = Cache(rng, 1, 0, 2, D, 24, [61], L=L, spare=1, fill=None)
    w = rng.random((L * c.P, 2, 24)).astype(np.float32)
    same_after(be, c, w, [29], 2, 5, blobs(c, w, stride))
