"""Tokens drawn from the target's probabilities, with and without a draft's, against 64 bits.

Tokens have to be equal: a weight is off by at most 2^-42 of itself (an exponential good to 2^-42.7, sums in
64 bits), so that running sums differ by less than 2^-40 of the whole from those here; a drawn number of 24
bits falls that near to one of V borders once in 2^40 / V draws.  logprob is a number x in 32 bits, rounded
once: 2^-24 |x|, and 2^-38 for what goes into it."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    import torch

    import openasr_b200 as ob

    b = ob.Backend(0)
    b.set_stream(torch.cuda.current_stream())
    yield b
    b.close()


def cuda(a):
    import torch

    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def probs64(x, T):
    """p of one row of logits, or None where nothing is finite; T = 0: the first maximum"""
    x = x.astype(np.float64)
    ok = np.isfinite(x)
    if not ok.any():
        return None
    m = x[ok].max()
    if T == 0:
        p = np.zeros_like(x)
        p[np.flatnonzero(ok & (x == m))[0]] = 1.0
        return p
    w = np.zeros_like(x)
    w[ok] = np.exp((x[ok] - m) / np.float64(T))
    return w / w.sum()


def node64(x, T, u, i, n, tokens=None, parents=None, q=None):
    """(token, log of its probability) of node i; u [n][2], q the draft's row of i"""
    p = probs64(x, T)
    if p is None:
        return -1, 0.0
    r, t = p, None
    for j in range(i + 1, n) if q is not None else ():
        if parents[j] != i:
            continue
        if np.float64(u[j, 0]) * np.float64(q[tokens[j]]) < r[tokens[j]]:
            t = int(tokens[j])
            break
        r = np.maximum(r - q.astype(np.float64), 0)
        r = r / r.sum() if r.sum() > 0 else p
    if t is None:
        c = np.cumsum(r)
        t = min(int(np.searchsorted(c, np.float64(u[i, 1]) * c[-1], side="right")), int(np.flatnonzero(r)[-1]))
    return t, 0.0 if T == 0 else float(np.log(p[t]))


def want64(x, temp, u, live, tokens=None, parents=None, q=None):
    S, N, _ = x.shape
    t, lp = np.full((S, N), -1, np.int32), np.zeros((S, N))
    for s in range(S):
        for i in range(live[s]):
            t[s, i], lp[s, i] = node64(x[s, i], temp[s], u[s], i, live[s], *((None,) * 3 if q is None else
                                                                            (tokens[s], parents[s], q[s, i])))
    return t, lp


def run(be, x, temp, u, live=None, tokens=None, parents=None, q=None, logprob=True):
    import torch

    S, N = x.shape[:2]
    t = torch.full((S, N), 77, dtype=torch.int32, device="cuda")
    lp = torch.full((S, N), 77.0, device="cuda") if logprob else None
    put = [a if a is None or torch.is_tensor(a) else cuda(a) for a in (x, temp, u, tokens, parents, q, live)]
    be.tree_sample(*put, t, lp)
    be.synchronize()
    return t.cpu().numpy(), lp.cpu().double().numpy() if logprob else None


def same(got, want):
    np.testing.assert_array_equal(got[0], want[0])
    assert (np.abs(got[1] - want[1]) <= 2.0**-24 * np.abs(want[1]) + 2.0**-38).all()


def softmax(x, T=1.0):
    e = np.exp((x - x.max(-1, keepdims=True)) / T)
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def logits_of(rng, *shape):
    x = rng.standard_normal(shape).astype(np.float32) * 2
    top = rng.integers(0, shape[-1], shape[:-1] + (4,))
    np.put_along_axis(x, top, 8 * rng.random(top.shape).astype(np.float32) + 4, -1)
    return x


@pytest.mark.parametrize("S,N,V", [
    (1, 1, 1), (2, 3, 2), (3, 1, 5), (2, 2, 31), (1, 4, 128), (2, 3, 129), (5, 1, 1000), (2, 3, 2047), (1, 2, 2048),
    (4, 3, 4099), (2, 2, 8191), (1, 1, 16385), (3, 2, 33001), (1, 1, 51866), (3, 5, 51866), (2, 1, 151936),
    (300, 1, 700), (40, 30, 2500), (20, 2, 40001),
])
def test_sampling_matches_64_bits(be, S, N, V):
    rng = np.random.default_rng(V + N)
    x = logits_of(rng, S, N, V)
    temp = rng.choice(np.array([0.0, 0.2, 0.7, 1.0, 1.0, 3.0], np.float32), S)
    u = rng.random((S, N, 2), np.float32)
    live = np.array([N if s % 3 else max(0, N - 1) for s in range(S)], np.int32)
    same(run(be, x, temp, u, live), want64(x, temp, u, live))


@pytest.mark.parametrize("cut,step", [(0, 0), (1, 1), (2, 2), (3, 5), (1, 3)])
def test_rows_of_any_alignment(be, cut, step):
    import torch

    rng = np.random.default_rng(cut)
    S, N, V = 3, 4, 5003
    buf = torch.full((S * N * (V + step) + 8,), 1e30, device="cuda")  # between the rows: what would win
    view = torch.as_strided(buf, (S, N, V), (N * (V + step), V + step, 1), cut)
    x = logits_of(rng, S, N, V)
    view.copy_(torch.from_numpy(x))
    u = rng.random((S, N, 2), np.float32)
    wide = torch.zeros(S, N, 5, device="cuda")  # strided uniforms
    wide[..., :2] = cuda(u)
    temp = np.array([1.0, 0.0, 0.5], np.float32)
    live = [N] * S
    same(run(be, view, temp, wide[..., :2]), want64(x, temp, u, live))
    q = softmax(x + rng.standard_normal(x.shape).astype(np.float32))
    par = np.tile(np.array([-1, 0, 0, 1], np.int32), (S, 1))
    tok = np.array([[rng.choice(V, p=q[s, max(p, 0)] / q[s, max(p, 0)].astype(np.float64).sum()) for p in par[s]] for s in range(S)], np.int32)
    same(run(be, view, temp, wide[..., :2], None, tok, par, q), want64(x, temp, u, live, tok, par, q))


def test_borders_are_exact(be):
    """equal logits: p = 1 / V each, and a number on a border belongs to the value behind it"""
    V = 4096
    k = np.arange(0, V, 7)
    x = np.full((len(k), 1, V), 3.5, np.float32)
    u = np.zeros((len(k), 1, 2), np.float32)
    u[:, 0, 1] = k / V
    t, _ = run(be, x, np.ones(len(k), np.float32), u)
    np.testing.assert_array_equal(t[:, 0], k)
    u[:, 0, 1] = np.nextafter(np.float32(1), np.float32(0))
    t, _ = run(be, x, None, u)
    assert (t == V - 1).all()


@pytest.mark.parametrize("T", [0.0, 1e-30, 1e-6, 0.01, 1.0, 1e30])
def test_what_is_not_finite_has_no_weight(be, T):
    rng = np.random.default_rng(7)
    S, V = 8, 9000
    x = logits_of(rng, S, 1, V)
    x[0, 0, ::2] = -np.inf
    x[1, 0, 5::3] = np.nan
    x[2, 0, ::7] = np.inf
    x[3] = -np.inf
    x[3, 0, 8123] = -4.0          # all but one
    x[4] = np.nan                 # nothing finite
    x[5, 0, :8000] = -np.inf      # whole runs of nothing
    x[6, 0, 4000:] = 3.0e38       # the largest numbers there are
    x[6, 0, :4000] = -3.0e38
    x[7, 0] = np.linspace(-3000, 3000, V)  # rising: the reference is left far behind
    temp, u = np.full(S, T, np.float32), rng.random((S, 1, 2), np.float32)
    same(run(be, x, temp, u), want64(x, temp, u, [1] * S))


def chains_and_trees(rng, S, N, V, shape):
    if shape == "chain":
        par = np.tile(np.arange(-1, N - 1), (S, 1)).astype(np.int32)
    elif shape == "star":
        par = np.zeros((S, N), np.int32)
        par[:, 0] = -1
    else:
        par = np.full((S, N), -1, np.int32)
        for i in range(1, N):
            par[:, i] = rng.integers(0, i, S)
        par[rng.random((S, N)) < 0.1] = -1  # nodes of no tree
    x = logits_of(rng, S, N, V)
    q = softmax(x + 0.7 * rng.standard_normal(x.shape).astype(np.float32))
    up = np.maximum(par, 0)
    tok = np.zeros((S, N), np.int32)
    for s in range(S):
        for j in range(N):
            p = q[s, up[s, j]].astype(np.float64)
            tok[s, j] = rng.choice(V, p=p / p.sum())
    return x, q, tok, par


@pytest.mark.parametrize("shape", ["chain", "tree", "star"])
@pytest.mark.parametrize("S,N,V", [(1, 2, 3), (3, 8, 40), (2, 33, 300), (2, 6, 20011), (1, 3, 70001), (30, 12, 2100)])
def test_rejection_matches_64_bits(be, shape, S, N, V):
    rng = np.random.default_rng(S * V)
    x, q, tok, par = chains_and_trees(rng, S, N, V, shape)
    temp = rng.choice(np.array([0.0, 0.8, 1.0, 1.0], np.float32), S)
    u = rng.random((S, N, 2), np.float32)
    live = np.array([N if s % 2 == 0 else N - N // 4 for s in range(S)], np.int32)
    same(run(be, x, temp, u, live, tok, par, q), want64(x, temp, u, live, tok, par, q))


def test_a_residual_without_mass_leaves_the_targets_probabilities(be):
    """a draft that claims more than the target everywhere: what is left is p itself"""
    rng = np.random.default_rng(3)
    S, N, V = 4, 3, 500
    x = logits_of(rng, S, N, V)
    q = np.ones((S, N, V), np.float32)
    par = np.tile(np.array([-1, 0, 0], np.int32), (S, 1))
    tok = rng.integers(0, V, (S, N)).astype(np.int32)
    u = np.full((S, N, 2), 0.75, np.float32)
    u[..., 1] = rng.random((S, N))
    temp = np.ones(S, np.float32)
    same(run(be, x, temp, u, None, tok, par, q), want64(x, temp, u, [N] * S, tok, par, q))


@pytest.mark.parametrize("T", [1e-30, 1e-4, 1e30, 3e35, 1e37, 3e38])
def test_rejection_at_any_temperature(be, T):
    """and with logits that are not finite, a row's end inside a tile"""
    rng = np.random.default_rng(5)
    S, N, V = 6, 7, 3001
    x, q, tok, par = chains_and_trees(rng, S, N, V, "tree")
    x[0, :, ::3] = -np.inf
    x[1, :, 1::5] = np.nan
    x[2, :, ::7] = np.inf
    x[3] *= 1e30
    q = softmax(rng.standard_normal(x.shape).astype(np.float32))
    u = rng.random((S, N, 2), np.float32)
    temp = np.full(S, T, np.float32)
    same(run(be, x, temp, u, None, tok, par, q), want64(x, temp, u, [N] * S, tok, par, q))


def test_accepted_tokens_are_distributed_as_the_targets(be):
    """65536 sequences with one drafted child: the token after the root is distributed as p, whatever the
    draft's q (five standard deviations of a count at fixed seeds)"""
    rng = np.random.default_rng(11)
    S, V = 65536, 7
    x1 = np.array([0.3, -1.0, 2.0, 0.0, 1.0, -3.0, 0.5], np.float32)
    q1 = softmax(np.array([1.0, 1.0, -1.0, 0.0, 2.0, 0.0, -2.0], np.float32))
    x, q = np.broadcast_to(x1, (S, 2, V)), np.broadcast_to(q1, (S, 2, V))
    tok = np.stack([np.zeros(S), rng.choice(V, S, p=q1.astype(np.float64) / q1.astype(np.float64).sum())], 1).astype(np.int32)
    par = np.tile(np.array([-1, 0], np.int32), (S, 1))
    t, _ = run(be, x, None, rng.random((S, 2, 2), np.float32), None, tok, par, q)
    p = probs64(x1, 1.0)
    count = np.bincount(t[:, 0], minlength=V)
    assert (np.abs(count - S * p) <= 5 * np.sqrt(S * p * (1 - p))).all()
    assert (t[:, 0] == tok[:, 1]).mean() > 0.2, "some of the drafted tokens are taken"


def test_with_tree_commit(be):
    """the drafted path that the sampled tokens follow is the one that tree_commit keeps"""
    import torch

    rng = np.random.default_rng(12)
    S, N, V, page = 6, 10, 90, 16
    x, q, tok, par = chains_and_trees(rng, S, N, V, "tree")
    par[:, 1:] = np.maximum(par[:, 1:], 0)
    u = rng.random((S, N, 2), np.float32)
    temp = np.array([0.0, 0.5, 1, 1, 1, 2], np.float32)
    target = torch.zeros(S, N, dtype=torch.int32, device="cuda")
    be.tree_sample(cuda(x), cuda(temp), cuda(u), cuda(tok), cuda(par), cuda(q), None, target, None)
    past = rng.integers(0, 20, S).astype(np.int32)
    table = rng.permutation(S * 3).reshape(S, 3).astype(np.int32)
    k, v = (torch.randn(S * 3, 2, page, 64, device="cuda").half() for _ in range(2))
    path, acc, nxt, out = (torch.zeros(*d, dtype=torch.int32, device="cuda") for d in ((S, N), (S,), (S,), (S,)))
    be.tree_commit(cuda(tok), cuda(par), target, None, cuda(past), cuda(table), k, v, 1, path, acc, nxt, out)
    be.synchronize()
    want, _ = want64(x, temp, u, [N] * S, tok, par, q)
    some = 0
    for s in range(S):
        walk = [0]
        while True:
            kids = [j for j in range(walk[-1] + 1, N) if par[s, j] == walk[-1] and tok[s, j] == want[s, walk[-1]]]
            if not kids:
                break
            walk.append(kids[0])
        some += len(walk) - 1
        assert path[s, : len(walk)].tolist() == walk and int(acc[s]) == len(walk) and int(nxt[s]) == want[s, walk[-1]]
    assert some > 0


def test_values_out_of_range_are_reported(be):
    import openasr_b200 as ob

    rng = np.random.default_rng(4)
    S, N, V = 2, 3, 600
    x, q, tok, par = chains_and_trees(rng, S, N, V, "chain")
    u = rng.random((S, N, 2), np.float32)
    temp, live = np.ones(S, np.float32), np.full(S, N, np.int32)

    def changed(a, at, value):
        b = a.copy()
        b[at] = value
        return b

    for args in ((x, changed(temp, 1, -0.5), u, live), (x, changed(temp, 1, np.nan), u, live), (x, changed(temp, 1, np.inf), u, live),
                 (x, temp, changed(u, (1, 2, 1), 1.0), live), (x, temp, changed(u, (0, 0, 1), -0.1), live),
                 (x, temp, changed(u, (0, 0, 1), np.nan), live), (x, temp, u, changed(live, 1, N + 1)), (x, temp, u, changed(live, 0, -1)),
                 (x, temp, u, live, changed(tok, (1, 1), V), par, q), (x, temp, u, live, changed(tok, (1, 1), -2), par, q),
                 (x, temp, changed(u, (1, 1, 0), 1.5), live, tok, par, q)):
        with pytest.raises(ob.GgmlBackendError, match="out-of-range"):
            run(be, *args)
    same(run(be, x, temp, u, live, tok, par, q), want64(x, temp, u, live, tok, par, q))
    # numbers that nothing is drawn with may be anything
    loose = changed(changed(u, (0, 0, 0), 9.0), (1, slice(None), 1), np.nan)
    same(run(be, x, changed(temp, 1, 0.0), loose, live, tok, par, q), want64(x, changed(temp, 1, 0.0), u, live, tok, par, q))


def test_empty_calls_and_missing_arguments(be):
    import torch

    rng = np.random.default_rng(5)
    x, u = logits_of(rng, 2, 2, 300), rng.random((2, 2, 2), np.float32)
    t, _ = run(be, x, None, u, logprob=False)
    np.testing.assert_array_equal(t, want64(x, [1.0, 1.0], u, [2, 2])[0])
    none = torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    be.tree_sample(torch.zeros(0, 2, 300, device="cuda"), None, torch.zeros(0, 2, 2, device="cuda"), None, None, None, None, none, None)
    be.synchronize()


def test_on_another_stream_and_in_a_captured_step(be):
    import torch

    rng = np.random.default_rng(6)
    S, N, V = 4, 5, 7000
    x, q, tok, par = chains_and_trees(rng, S, N, V, "chain")
    temp, u = np.array([1, 0.6, 0, 1], np.float32), rng.random((S, N, 2), np.float32)
    put = [cuda(a) for a in (x, temp, u, tok, par, q)]
    t, lp = torch.zeros(S, N, dtype=torch.int32, device="cuda"), torch.zeros(S, N, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    be.set_stream(stream)
    try:
        be.tree_sample(*put, None, t, lp)
        be.synchronize()
        same((t.cpu().numpy(), lp.cpu().double().numpy()), want64(x, temp, u, [N] * S, tok, par, q))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            be.tree_sample(*put, None, t, lp)
        for _ in range(3):
            x2, u2 = logits_of(rng, S, N, V), rng.random((S, N, 2), np.float32)
            with torch.cuda.stream(stream):
                put[0].copy_(cuda(x2))
                put[2].copy_(cuda(u2))
                graph.replay()
            be.synchronize()
            same((t.cpu().numpy(), lp.cpu().double().numpy()), want64(x2, temp, u2, [N] * S, tok, par, q))
    finally:
        be.set_stream(torch.cuda.current_stream())


def test_offsets_past_32_bits(be):
    """rows 2^31 bytes and more from the first"""
    import torch

    rng = np.random.default_rng(8)
    S, N, V = 2, 3, 5001
    big = torch.empty(S * N * 300_000_000, dtype=torch.float32, device="cuda")
    view = torch.as_strided(big, (S, N, V), (N * 300_000_000, 300_000_000, 1), 0)
    x = logits_of(rng, S, N, V)
    view.copy_(torch.from_numpy(x))
    u = rng.random((S, N, 2), np.float32)
    same(run(be, view, None, u), want64(x, [1.0] * S, u, [N] * S))


def test_refusals(be):
    import torch

    import openasr_b200 as ob

    S, N, V = 2, 3, 50

    def f(*d):
        return torch.zeros(*d, device="cuda")

    def i(*d):
        return torch.zeros(*d, dtype=torch.int32, device="cuda")

    base = dict(x=f(S, N, V), temp=f(S), u=f(S, N, 2), tok=i(S, N), par=i(S, N), q=f(S, N, V), live=i(S), t=i(S, N), lp=f(S, N))
    other = f(S * N * 4)
    for change, says in (
            (dict(x=f(S, N, V).half()), "logits must be F32"), (dict(x=f(S, V, N).transpose(1, 2)), "logits must be F32"),
            (dict(x=f(S, N, 0)), "1 to 2"), (dict(u=f(S, N, 3)), "uniforms"), (dict(u=f(S, N + 1, 2)), "uniforms"),
            (dict(temp=f(S + 1)), "temperature"), (dict(temp=i(S)), "temperature"), (dict(live=f(S)), "n_nodes"),
            (dict(tok=None), "come together"), (dict(q=None), "come together"), (dict(q=f(S, N, V + 1)), "draft_probs"),
            (dict(par=i(S, N + 1)), "tokens and parents"), (dict(t=f(S, N)), "target must be"), (dict(t=i(N, S)), "target must be"),
            (dict(lp=i(S, N)), "logprob"), (dict(t=base["tok"]), "overlap an input"), (dict(lp=base["u"].view(-1)[:S * N].view(S, N)), "overlap an input"),
            (dict(t=other.view(torch.int32)[:S * N].view(S, N), lp=other[2:2 + S * N].view(S, N)), "must not overlap"),
            (dict(t=i(S, 1).expand(S, N)), "target must be"), (dict(t=i(1, N).expand(S, N)), "must not overlap")):
        a = {**base, **change}
        with pytest.raises(ob.GgmlBackendError, match=says):
            be.tree_sample(a["x"], a["temp"], a["u"], a["tok"], a["par"], a["q"], a["live"], a["t"], a["lp"])
    with pytest.raises(ob.GgmlBackendError, match="1024"):
        be.tree_sample(f(1, 1025, 4), None, f(1, 1025, 2), i(1, 1025), i(1, 1025), f(1, 1025, 4), None, i(1, 1025), None)


def test_supports_op(be):
    import torch

    import openasr_b200 as ob
    from openasr_b200 import backend as bk

    assert be.supports_op(bk.OP_TREE_SAMPLE, ob.describe(torch.zeros(2, 2, 9)))
    assert not be.supports_op(bk.OP_TREE_SAMPLE, ob.describe(torch.zeros(2, 2, 9, dtype=torch.float16)))
