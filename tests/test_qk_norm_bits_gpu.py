"""qk_norm_rope rounds as the decoders' own norm does (squares in 32 bits, their sum in 64, every product
rounded), so a verification pass writes the K rows that a decode step writes, to the bit.

The sum's order is not part of that: two orders in 64 bits differ by 2^-53 of the sum, and the mean is
rounded to 24 bits, so they would part in one head of 2^26 or so."""
import numpy as np
import pytest

from openasr_b200 import models as om
from test_pages_gpu import Cache, be, cuda  # noqa: F401

pytestmark = pytest.mark.gpu


def norm_rope32(x, w, eps, cos, sin):
    """x [..., D] f32 -> f32, each step rounded once"""
    f32 = np.float32
    mean = ((x * x).astype(np.float64).sum(-1) / x.shape[-1]).astype(f32)
    scale = f32(1) / np.sqrt(mean + f32(eps))
    y = (x * scale[..., None]) * w
    a, b = np.split(y, 2, -1)
    return np.concatenate([a * cos - b * sin, a * sin + b * cos], -1)


@pytest.mark.parametrize("S,N,H,HKV,D", [(4, 512, 16, 8, 128), (3, 700, 20, 20, 64), (8, 3, 16, 8, 128), (8, 3, 20, 20, 64)])
def test_rounded_as_the_decoders_norm(be, S, N, H, HKV, D):  # noqa: F811
    import torch

    rng = np.random.default_rng(D + N)
    c = Cache(rng, S, N, HKV, D, 16, rng.integers(0, 40, S), fill=None)
    x = (rng.standard_normal((S, N, H + 2 * HKV, D)) * 1.7).astype(np.float32)
    wq, wk = (rng.normal(1, 0.1, D).astype(np.float32) for _ in range(2))
    at = c.past[:, None] + np.arange(N)
    ang = np.arange(at.max() + 1)[:, None] * 1e6 ** (-np.arange(D // 2) * 2.0 / D)
    tab = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
    cos, sin = tab[at][:, :, None, :, 0], tab[at][:, :, None, :, 1]
    k, v = c.device()
    q = torch.zeros(S, N, H, D, device="cuda")
    be.qk_norm_rope(cuda(x), cuda(wq), cuda(wk), 1e-6, cuda(tab), None, cuda(c.table), cuda(c.past), None, q, k, v)
    be.synchronize()
    want_q = norm_rope32(x[:, :, :H], wq, 1e-6, cos, sin)
    want_k = norm_rope32(x[:, :, H:H + HKV], wk, 1e-6, cos, sin).astype(np.float16)
    assert np.array_equal(q.cpu().numpy().view(np.int32), want_q.view(np.int32))
    rows = k.cpu().numpy()
    for s in range(S):
        assert np.array_equal(rows[c.table[s, at[s] // 16], :, at[s] % 16].view(np.int16), want_k[s].view(np.int16))


@pytest.fixture(scope="module")
def model(gpu_backend):
    cfg = om.QWEN3_ASR_0_6B.replace(n_layers=1, n_vocab=4096, max_pos=128, max_prefill=32, max_batch=4)
    m = om.QwenModel(gpu_backend, cfg, om.qwen_synthetic_pack(cfg, seed=0x0A5A0003))
    yield m
    m.close()


@pytest.mark.parametrize("seed", range(6))
def test_a_verification_pass_writes_a_decode_steps_rows(model, seed):
    """layer 0 has no attention before its K and V: the same bits, whatever the prompt"""
    n, T, steps = 4, 12, 30
    emb = om.qwen_synthetic_prefix(0x0A5A4000 + seed, n, T, model.cfg.d_model)
    serial = model.generate(emb, n_new=steps)
    want = [model.read_kv(0, s, T + steps - 1) for s in range(n)]
    model.prefill(emb)
    chain = np.tile(np.arange(-1, steps - 2, dtype=np.int32), (n, 1))
    _, acc, _ = model.verify_tree(serial[:, :steps - 1], chain, [T] * n)
    assert (acc >= 1).all()
    for s in range(n):
        for got, w in zip(model.read_kv(0, s, T + acc[s]), want[s]):
            assert np.array_equal(got.view(np.uint16), w[:, :T + acc[s]].view(np.uint16))
