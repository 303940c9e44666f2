"""attn_weights after a verification pass of which something was rejected: the accepted nodes, once tree_commit
has moved their rows, are a chain from the old n_past on, and the attention that they pay is what is added.
Tolerances as in test_kv_evict_gpu."""
import numpy as np
import pytest

from test_kv_evict_gpu import added64, check, entries
from test_pages_gpu import Cache, cuda, random_parents

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    import torch

    import openasr_b200 as ob

    b = ob.Backend(0)
    b.set_stream(torch.cuda.current_stream())
    yield b
    b.close()


@pytest.mark.parametrize("N,H,HKV,D", [(8, 4, 2, 64), (33, 6, 3, 128)])
@pytest.mark.parametrize("shape", ["chain", "tree"])
def test_the_accepted_nodes_of_a_draft(be, shape, N, H, HKV, D):
    import torch

    import openasr_b200 as ob

    rng = np.random.default_rng(N)
    S, page, past = 4, 16, [40, 0, 131, 77]
    c = Cache(rng, S, N, HKV, D, page, past)
    par = np.tile(np.arange(-1, N - 1, dtype=np.int32), (S, 1)) if shape == "chain" else random_parents(rng, S, N)
    tok = rng.integers(0, 50, (S, N)).astype(np.int32)
    # the target follows some path of each tree down to a node, and then chooses what was not drafted
    target, walks = np.full((S, N), 99, np.int32), []
    for s in range(S):
        at, walk = [1, N // 2, N - 1, 0][s], []
        while at >= 0:
            walk.append(at)
            at = par[s, at]
        walks.append(walk[::-1])
        for a, b in zip(walks[s], walks[s][1:]):
            tok[s, b], target[s, a] = 50 + b, 50 + b
    q = rng.standard_normal((S, H, N, D)).astype(np.float32)
    old, scale = entries(rng, c), D**-0.5
    qd, table, n_past, w = cuda(q), cuda(c.table), cuda(c.past), cuda(old)
    k, v = c.device()
    words = cuda(np.stack([ob.tree_mask(p) for p in par]))
    o = torch.zeros(S, N, H, D, device="cuda")
    be.flash_attn_tree(qd, k, v, table, n_past, None, words, scale, o)
    path, acc, nxt, out = (torch.zeros(*d, dtype=torch.int32, device="cuda") for d in ((S, N), (S,), (S,), (S,)))
    be.tree_commit(cuda(tok), cuda(par), cuda(target), None, n_past, table, k, v, 1, path, acc, nxt, out)
    rows = path.clamp(min=0).long()[:, None, :, None].expand(S, H, N, D)
    be.attn_weights(qd.gather(2, rows), k, table, n_past, acc, scale, 0.5, w)
    be.synchronize()
    assert acc.tolist() == [len(x) for x in walks]
    taken = q.copy()
    for s in range(S):
        assert path[s, : len(walks[s])].tolist() == walks[s]
        taken[s, :, : len(walks[s])] = q[s][:, walks[s]]
        at = past[s] + np.array(walks[s])
        moved = c.k[c.table[s, at // page], :, at % page].copy()
        to = past[s] + np.arange(len(walks[s]))
        c.k[c.table[s, to // page], :, to % page] = moved
    want, tol = added64(c, taken, [len(x) for x in walks], scale, 0.5, old)
    check(w.cpu().double().numpy(), want, tol)
    if shape == "chain":  # whose accepted rows are in place already: the same queries do
        w2 = cuda(old)
        be.attn_weights(qd, k, table, n_past, acc, scale, 0.5, w2)
        be.synchronize()
        np.testing.assert_array_equal(w2.cpu().numpy(), w.cpu().numpy())
