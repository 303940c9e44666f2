"""What is left of the target's probabilities after rejected children, where it is nothing, or less than the
roundings of what it was taken from.  Tokens equal to 64 bits', tolerances as in test_tree_sample_gpu."""
import numpy as np
import pytest

from test_tree_sample_gpu import run, same, want64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    import torch

    import openasr_b200 as ob

    b = ob.Backend(0)
    b.set_stream(torch.cuda.current_stream())
    yield b
    b.close()


def inside(x, gap):
    """the rows inside a larger buffer whose other values would win"""
    import torch

    S, N, V = x.shape
    buf = torch.full((S * N * (V + gap) + 8,), 1e30, device="cuda")
    view = torch.as_strided(buf, (S, N, V), (N * (V + gap), V + gap, 1), 4)
    view.copy_(torch.from_numpy(x))
    return view


def certain(rng, S, N, V, rest):
    """rows with one likely token, the others without probability or `rest` nats below it; the draft's children are others"""
    top = rng.integers(0, V, (S, N, 1))
    level = rng.uniform(-220, 220, (S, N, 1))
    level[::3] /= 20
    x = np.full((S, N, V), -np.inf) if rest is None else level - rest - rng.random((S, N, V))
    np.put_along_axis(x, top, level, -1)
    par = np.zeros((S, N), np.int32)
    par[:, 0] = -1
    tok = ((top[:, :1, 0] + rng.integers(1, V, (S, N))) % V).astype(np.int32)  # none is the root's likely one
    u = rng.random((S, N, 2), np.float32)
    u[..., 0] = 0.25 + u[..., 0] / 2
    return x.astype(np.float32), top, tok, par, u


@pytest.mark.parametrize("draft,rest", [("ones", None), ("ones", 40.0), ("ones", 600.0), ("the same token", None),
                                        ("the same token", 40.0), ("the same token", 90.0)])
@pytest.mark.parametrize("S,N,V", [(700, 2, 5), (64, 4, 300), (40, 3, 6007), (6, 2, 51866)])
def test_a_certain_token_that_the_draft_was_certain_of(be, S, N, V, draft, rest):
    """p and q are 1 on one token: nothing is left of it, however exp and sums were rounded.  Then either nothing
    is left at all and the token is drawn from p, or the others share what they had."""
    rng = np.random.default_rng(V)
    x, top, tok, par, u = certain(rng, S, N, V, rest)
    q = np.ones((S, N, V), np.float32)
    if draft != "ones":
        q[:] = 0
        np.put_along_axis(q, top, np.float32(1), -1)
    temp = np.ones(S, np.float32)
    # a number against q(t) = 0 is accepted wherever p(t) is not 0: such tokens are no children here
    if draft != "ones" and rest is not None:
        np.put_along_axis(q[:, 0], tok, np.float32(1), -1)
    got = run(be, inside(x, 3), temp, u, None, tok, par, q)
    same(got, want64(x, temp, u, [N] * S, tok, par, q))
    if draft == "ones" or rest is None:
        assert (got[0][:, 0] == top[:, 0, 0]).all()
    elif V > N:
        assert (got[0][:, 0] != top[:, 0, 0]).any()


@pytest.mark.parametrize("T", [1e-30, 1e-4, 0.02, 1e4, 1e30])
def test_a_certain_token_at_any_temperature(be, T):
    rng = np.random.default_rng(5)
    S, N, V = 200, 3, 1001
    x, top, tok, par, u = certain(rng, S, N, V, None)
    temp = np.full(S, T, np.float32)
    q = np.ones((S, N, V), np.float32)
    got = run(be, inside(x, 1), temp, u, None, tok, par, q)
    same(got, want64(x, temp, u, [N] * S, tok, par, q))
    assert (got[0] == top[..., 0]).all()


@pytest.mark.parametrize("V", [2, 64, 4096, 32768])
def test_a_flat_row_that_the_draft_knew(be, V):
    """p = q = 1 / V to the bit, and a child that is no token of the draft's: p once more, after any number of rounds"""
    rng = np.random.default_rng(V)
    S, N = 12, 5
    x = np.broadcast_to(rng.uniform(-50, 50, (S, N, 1)).astype(np.float32), (S, N, V + 1)).copy()
    x[..., -1] = -np.inf
    q = np.full((S, N, V + 1), 1 / V, np.float32)
    q[..., -1] = 0
    par = np.zeros((S, N), np.int32)
    par[:, 0] = -1
    tok = np.full((S, N), V, np.int32)
    u = rng.random((S, N, 2), np.float32)
    temp = np.ones(S, np.float32)
    got = run(be, x, temp, u, None, tok, par, q)
    same(got, want64(x, temp, u, [N] * S, tok, par, q))
    np.testing.assert_array_equal(got[0], np.floor(u[..., 1].astype(np.float64) * V).astype(np.int32))


def test_differences_above_the_roundings_are_kept(be):
    """what p and q differ by through q's 32 bits, 2^-25 of p and less, is far above 2^-40"""
    rng = np.random.default_rng(9)
    S, V = 400, 3
    l = rng.uniform(-3, 3, (S, 1, V)).astype(np.float32)
    x = np.repeat(l, 2, 1)
    e = np.exp(x.astype(np.float64))
    q = (e / e.sum(-1, keepdims=True)).astype(np.float32)
    q[:, :, 2] = 0  # all of the third is left, and 2^-25 of the others or nothing
    tok = np.zeros((S, 2), np.int32)
    par = np.tile(np.array([-1, 0], np.int32), (S, 1))
    q[:, 0, 0] = 2  # rejected
    u = rng.random((S, 2, 2), np.float32)
    u[..., 0] = 0.999
    temp = np.ones(S, np.float32)
    same(run(be, x, temp, u, None, tok, par, q), want64(x, temp, u, [2] * S, tok, par, q))


@pytest.mark.parametrize("kids", [2, 3, 5])
def test_tokens_after_several_children_are_distributed_as_the_targets(be, kids):
    """65536 roots with children drawn from q one after the other: the token after the root is distributed as p (five
    standard deviations of a count at fixed seeds), and each further child is taken now and then"""
    rng = np.random.default_rng(kids)
    S, V, N = 65536, 7, 1 + kids
    x1 = np.array([0.3, -1.0, 2.0, 0.0, 1.0, -3.0, 0.5], np.float32)
    q1 = np.exp(np.array([1.0, 1.0, -1.0, 0.0, 2.0, 0.0, -2.0]))
    q1 = (q1 / q1.sum()).astype(np.float32)
    p = np.exp(x1.astype(np.float64))
    p /= p.sum()
    x, q = np.broadcast_to(x1, (S, N, V)), np.broadcast_to(q1, (S, N, V))
    tok = rng.choice(V, (S, N), p=q1.astype(np.float64) / q1.astype(np.float64).sum()).astype(np.int32)
    par = np.zeros((S, N), np.int32)
    par[:, 0] = -1
    t, _ = run(be, x, None, rng.random((S, N, 2), np.float32), None, tok, par, q)
    count = np.bincount(t[:, 0], minlength=V)
    assert (np.abs(count - S * p) <= 5 * np.sqrt(S * p * (1 - p))).all()
    first = [(t[:, 0] == tok[:, j]) & (t[:, :1] != tok[:, 1:j]).all(-1) for j in range(1, N)]
    assert all(f.mean() > 0.01 for f in first), [f.mean() for f in first]


@pytest.mark.parametrize("q0", [0.5, 0.9, 0.99])
@pytest.mark.parametrize("N", [14, 64, 1024])
def test_one_token_is_left_after_any_number_of_children(be, N, q0):
    """what is left of p is one token's from the first rejected child on, and is 1 again after each: the next ones take
    q0 of it and no more, although together they have taken all but (1 - q0)^N"""
    rng = np.random.default_rng(N)
    S, V = 3, 37
    p = np.full((S, N, V), 0.004 / (V - 1))
    p[..., 5] = 0.996
    q = np.full((S, N, V), (1 - q0) / (V - 1), np.float32)
    q[..., 5] = q0
    x = np.log(p).astype(np.float32)
    tok = rng.integers(6, V, (S, N)).astype(np.int32)
    par = np.zeros((S, N), np.int32)
    par[:, 0] = -1
    u = rng.random((S, N, 2), np.float32)
    u[..., 0] = 0.999
    u[:, 0, 1] = 0.9999  # another one of p's
    temp = np.ones(S, np.float32)
    got = run(be, x, temp, u, None, tok, par, q)
    same(got, want64(x, temp, u, [N] * S, tok, par, q))
    assert (got[0][:, 0] == 5).all()


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, -3e38, 3e38, -1.0])
@pytest.mark.parametrize("V", [9, 5003, 60001])
def test_a_draft_that_is_no_probability_still_gives_a_token(be, bad, V):
    """the outputs are then undefined, but tokens of the vocabulary, and the other sequences' their own"""
    rng = np.random.default_rng(V)
    S, N = 12, 4
    x, top, tok, par, u = certain(rng, S, N, V, 3.0)
    q = np.exp(x.astype(np.float64) + rng.standard_normal(x.shape))
    q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
    want = want64(x, np.ones(S), u, [N] * S, tok, par, q)
    spoiled = q.copy()
    spoiled[::2, :, rng.integers(0, V, 3)] = bad
    spoiled[::4] = bad
    t, lp = run(be, inside(x, 2), None, u, None, tok, par, spoiled)
    assert ((0 <= t) & (t < V)).all() and np.isfinite(lp).all()
    same((t[1::2], lp[1::2]), (want[0][1::2], want[1][1::2]))
