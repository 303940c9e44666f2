"""attn_weights of a whole prompt, or of its last part: hundreds of nodes of a sequence.  Tolerances as in
test_kv_evict_gpu."""
import numpy as np
import pytest

from test_kv_evict_gpu import added64, check, entries, run_weights
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


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,N,H,HKV,D,page,past", [
    (1, 512, 16, 8, 128, 64, [0]),             # a prompt from its first token on
    (3, 301, 4, 4, 64, 24, [100, 0, 37]),
    (1, 1500, 2, 1, 64, 16, [0]),              # 3000 rows of one head
    (2, 257, 20, 4, 128, 40, [700, 1290]),     # its last part: 1285 rows of a head
    (9, 129, 32, 4, 128, 8, [5 * s for s in range(9)]),
])
def test_prompts(be, S, N, H, HKV, D, page, past, f16):
    rng = np.random.default_rng(N)
    c = Cache(rng, S, N, HKV, D, page, past)
    q = rng.standard_normal((S, H, N, D)).astype(np.float16 if f16 else np.float32)
    live = np.array([N if s % 2 == 0 else N - 1 - N // 3 for s in range(S)], np.int32)
    for s in range(S):
        for p in range(c.past[s] + live[s], c.past[s] + N):
            c.k[c.table[s, p // page], :, p % page] = np.nan
    old = entries(rng, c)
    want, tol = added64(c, q, live, D**-0.5, 0.9, old)
    got = run_weights(be, c, q, live, D**-0.5, 0.9, old, f16=f16)
    check(got, want, tol)
    np.testing.assert_array_equal(got, run_weights(be, c, q, live, D**-0.5, 0.9, old, f16=f16))


def test_a_prompt_at_once_or_in_parts(be):
    """what two chunks add is what one call adds (twice the bound: the entries are rounded once more in between)"""
    rng = np.random.default_rng(3)
    N, cut = 200, 73
    c = Cache(rng, 1, N, 2, 64, 16, [0])
    q = rng.standard_normal((1, 4, N, 64)).astype(np.float32)
    old = entries(rng, c)
    want, tol = added64(c, q, [N], 0.125, 0.0, old)
    first = run_weights(be, c, q[:, :, :cut].copy(), np.array([cut], np.int32), 0.125, 0.0, old).astype(np.float32)
    c.past[0] = cut
    got = run_weights(be, c, q[:, :, cut:].copy(), np.array([N - cut], np.int32), 0.125, 1.0, first)
    check(got, want, 2 * tol)
