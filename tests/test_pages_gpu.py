"""The paged K/V cache and drafted trees against plain implementations in 64 bits.

Tolerances come from the arithmetic, before any run.  Attention: a score is a dot product of
D products in 32 bits, so it is off by at most ds = 2^-20 * scale * max sum|q||k| (D <= 128
roundings of 2^-24 and as much again for an operand kept in two 16-bit halves); a weight is off
by a factor of 1 +- (2 ds + 2^-20) (its own score, the row's sum, the exponential), and outputs
are weighted means of V, so they move by at most twice that times max|v|.  f16 outputs add half
a unit in the last place, 2^-11 |o| + 2^-25.  Norms and rotation: a handful of roundings of
2^-24 on values of magnitude m: 16 * 2^-24 * m, and 2^-11 for f16 rows."""
import math

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


def cuda(a, dtype=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if dtype is None else t.to(dtype)).cuda()


class Cache:
    """A pool of pages in scattered order; positions past a sequence's end hold NaN."""

    def __init__(self, rng, S, N, HKV, D, page, past, L=1, layout="head", spare=2, fill=np.nan):
        self.S, self.N, self.HKV, self.D, self.page, self.L = S, N, HKV, D, page, L
        self.past = np.array(past, np.int32)
        self.MP = max(1, -(-(int(self.past.max(initial=0)) + N) // page))
        self.P = S * self.MP + spare
        self.table = rng.permutation(self.P)[: S * self.MP].reshape(S, self.MP).astype(np.int32)
        shape = (L * self.P, HKV, page, D)
        self.k, self.v = (rng.standard_normal(shape).astype(np.float16) for _ in range(2))
        used = np.zeros((self.P, page), bool)
        for s in range(S):
            for p in range(self.past[s] + N):
                used[self.table[s, p // page], p % page] = True
        if fill is not None:
            for x in (self.k, self.v):
                x.reshape(L, self.P, HKV, page, D).transpose(0, 1, 3, 2, 4)[:, ~used] = fill
        self.layout = layout

    def device(self):
        """torch views [L * P, HKV, page, D]; `layout` "row": positions slower than heads in memory"""
        if self.layout == "row":
            return [cuda(x.transpose(0, 2, 1, 3)).permute(0, 2, 1, 3) for x in (self.k, self.v)]
        return [cuda(x) for x in (self.k, self.v)]

    def rows(self, x, s, n, layer=0):
        """[HKV, n, D] of positions 0..n-1 of sequence s"""
        p = np.arange(n)
        return x[layer * self.P + self.table[s, p // self.page], :, p % self.page].transpose(1, 0, 2)


def random_parents(rng, S, N):
    par = np.full((S, N), -1, np.int32)
    for i in range(1, N):
        par[:, i] = rng.integers(0, i, S)
    return par


def sees_of(par):
    n = len(par)
    see = np.zeros((n, n), bool)
    for i in range(n):
        j = i
        while j >= 0:
            see[i, j] = True
            j = par[j]
    return see


def words_of(see):
    S, N, _ = see.shape
    w = np.zeros((S, N, (N + 31) // 32), np.uint32)
    for j in range(N):
        w[:, :, j // 32] |= see[:, :, j].astype(np.uint32) << np.uint32(j % 32)
    return w.view(np.int32)


def attend64(c, q, live, sees, scale):
    """q [S, H, N, D] -> ([S, N, H, D] in 64 bits, bound on the error of 32-bit arithmetic)"""
    S, H, N, D = q.shape
    G = H // c.HKV
    out, tol = np.zeros((S, N, H, D)), np.zeros((S, N, H, 1))
    for s in range(S):
        n = int(live[s])
        T = int(c.past[s]) + n
        k, v = (c.rows(x, s, T).astype(np.float64) for x in (c.k, c.v))
        for i in range(n):
            vis = np.concatenate([np.ones(c.past[s], bool), sees[s, i, :n]])
            if not vis.any():
                continue
            for h in range(H):
                kk, vv = k[h // G][vis], v[h // G][vis]
                x = kk @ q[s, h, i].astype(np.float64) * scale
                w = np.exp(x - x.max())
                out[s, i, h] = (w / w.sum()) @ vv
                ds = 2.0**-20 * abs(scale) * (np.abs(kk) @ np.abs(q[s, h, i].astype(np.float64))).max()
                tol[s, i, h] = 2 * (2 * ds + 2.0**-20) * np.abs(vv).max()
    return out, tol


def run_attn(be, c, q, live, words, scale, f16=False, pages=None, q_view=None):
    import torch

    S, H, N, D = q.shape
    dt = torch.float16 if f16 else torch.float32
    k, v = pages or c.device()
    qd = q_view if q_view is not None else cuda(q, dt)
    out = torch.full((S, N, H, D), 7.0, dtype=dt, device="cuda")
    be.flash_attn_tree(qd, k, v, cuda(c.table), cuda(c.past), None if live is None else cuda(live),
                       None if words is None else cuda(words), scale, out)
    be.synchronize()
    return out.cpu().double().numpy()


def check(got, want, tol, f16):
    allowed = tol + (2.0**-11 * np.abs(want) + 2.0**-25 if f16 else 2.0**-22 * np.abs(want))
    # committed positions that were never written hold NaN here: what sees them is NaN on both sides
    bad = ~((np.abs(got - want) <= allowed) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want))}"


# S, N, H, HKV, D, page, past, tree
ATTN = [
    (1, 1, 16, 8, 128, 64, [390], False),
    (1, 1, 16, 8, 128, 64, [0], False),             # the first token: sees itself alone
    (2, 1, 20, 20, 64, 16, [0, 63], False),
    (3, 16, 16, 8, 128, 16, [5, 700, 63], True),
    (3, 7, 20, 20, 64, 24, [441, 0, 57], False),    # pages that end inside every tile
    (2, 61, 16, 8, 128, 40, [129, 1000], True),
    (1, 64, 16, 8, 128, 8, [127], True),
    (2, 33, 8, 1, 128, 64, [300, 31], True),        # 264 rows of one K/V head
    (1, 17, 6, 6, 64, 256, [257], True),
    (2, 5, 32, 4, 128, 64, [2500, 2049], True),
    (1, 150, 4, 2, 64, 32, [77], True),             # five mask words
    (1, 300, 4, 2, 128, 64, [45], False),           # a chain longer than a tile of rows
    (5, 3, 15, 5, 128, 8, [1, 0, 9, 120, 4096], True),
]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,N,H,HKV,D,page,past,tree", ATTN)
def test_flash_attn_tree_matches_64_bits(be, S, N, H, HKV, D, page, past, tree, f16):
    rng = np.random.default_rng(S * 1000 + N)
    c = Cache(rng, S, N, HKV, D, page, past)
    q = rng.standard_normal((S, H, N, D)).astype(np.float16 if f16 else np.float32)
    live = np.array([N if s % 2 == 0 else max(1, N - 1 - N // 3) for s in range(S)], np.int32)
    for s in range(S):  # rows of padding nodes are garbage too
        for p in range(c.past[s] + live[s], c.past[s] + N):
            for x in (c.k, c.v):
                x[c.table[s, p // page], :, p % page] = np.nan
    if tree:
        sees = np.stack([sees_of(p) for p in random_parents(rng, S, N)])
    else:
        sees = np.broadcast_to(np.tril(np.ones((N, N), bool)), (S, N, N))
    scale = 1 / math.sqrt(D)
    want, tol = attend64(c, q, live, sees, scale)
    got = run_attn(be, c, q, live, words_of(sees) if tree else None, scale, f16)
    check(got, want, tol, f16)
    for s in range(S):
        assert not got[s, live[s]:].any(), "padding nodes must be zeros"


def test_flash_attn_tree_large_scores_and_values(be):
    """scores of hundreds (one weight is all that is left) and values of thousands"""
    rng = np.random.default_rng(5)
    c = Cache(rng, 2, 9, 2, 128, 16, [200, 31])
    for x in (c.k, c.v):
        x *= np.float16(16)
    q = rng.standard_normal((2, 8, 9, 128)).astype(np.float32) * 20
    sees = np.stack([sees_of(p) for p in random_parents(rng, 2, 9)])
    live = np.array([9, 9], np.int32)
    want, tol = attend64(c, q, live, sees, 1 / math.sqrt(128))
    check(run_attn(be, c, q, None, words_of(sees), 1 / math.sqrt(128)), want, tol, False)


def test_a_row_that_sees_nothing_is_zeros(be):
    rng = np.random.default_rng(6)
    N = 40
    c = Cache(rng, 2, N, 4, 64, 16, [0, 3])
    q = rng.standard_normal((2, 8, N, 64)).astype(np.float32)
    sees = rng.random((2, N, N)) < 0.2
    sees[:, ::3] = False  # nothing among the nodes: sequence 0 has no committed positions either
    want, tol = attend64(c, q, [N, N], sees, 0.125)
    got = run_attn(be, c, q, None, words_of(sees), 0.125)
    assert not got[0, ::3].any() and got[1, ::3].all()
    check(got, want, tol, False)


def test_empty_sequences_and_empty_calls(be):
    import torch

    rng = np.random.default_rng(7)
    c = Cache(rng, 3, 4, 2, 128, 16, [9, 0, 100])
    q = rng.standard_normal((3, 4, 4, 128)).astype(np.float32)
    live = np.array([0, 0, 4], np.int32)
    sees = np.broadcast_to(np.tril(np.ones((4, 4), bool)), (3, 4, 4))
    want, tol = attend64(c, q, live, sees, 0.1)
    got = run_attn(be, c, q, live, None, 0.1)
    assert not got[:2].any()
    check(got, want, tol, False)
    k, v = c.device()
    none = torch.empty(3, 0, 4, 128, device="cuda")
    be.flash_attn_tree(none.permute(0, 2, 1, 3), k, v, cuda(c.table), cuda(c.past), None, None, 0.1, none)
    be.synchronize()


@pytest.mark.parametrize("H,HKV,D,N", [(4, 2, 128, 9), (4, 2, 128, 80), (6, 6, 64, 9)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_a_row_does_not_see_does_not_reach_it(be, H, HKV, D, N, bad):
    rng = np.random.default_rng(8)
    past = 70
    c = Cache(rng, 1, N, HKV, D, 16, [past])
    hidden, seen = 5, 3  # node 5 is hidden from every node but itself; node 3 stays finite
    par = np.arange(-1, N - 1, dtype=np.int32)[None].copy()
    par[0, 6] = 4
    pg, off = c.table[0, (past + hidden) // 16], (past + hidden) % 16
    q = rng.standard_normal((1, H, N, D)).astype(np.float32)
    sees = sees_of(par[0])[None]
    want, tol = attend64(c, q, [N], sees, 0.1)
    c.k[pg, :, off] = bad
    c.v[pg, :, off, ::3] = bad
    got = run_attn(be, c, q, None, words_of(sees), 0.1)
    rest = [i for i in range(N) if i != hidden]
    assert not sees[0, rest][:, hidden].any() and sees[0, 6, seen]
    check(got[:, rest], want[:, rest], tol[:, rest], False)


@pytest.mark.parametrize("N", [4, 80])
def test_an_infinite_value_reaches_the_rows_that_see_it(be, N):
    rng = np.random.default_rng(9)
    past = 50
    c = Cache(rng, 1, N, 2, 128, 16, [past])
    q = rng.standard_normal((1, 4, N, 128)).astype(np.float32)
    par = random_parents(rng, 1, N)
    sees = sees_of(par[0])[None]
    want, tol = attend64(c, q, [N], sees, 0.05)
    j = 2
    pg, off = c.table[0, (past + j) // 16], (past + j) % 16
    c.v[pg, :, off, 5] = np.inf
    c.v[pg, :, off, 9] = np.nan
    got = run_attn(be, c, q, None, words_of(sees), 0.05)
    for i in range(N):
        if sees[0, i, j]:
            assert np.isposinf(got[0, i, :, 5]).all() and np.isnan(got[0, i, :, 9]).all()
            got[0, i, :, [5, 9]] = want[0, i, :, [5, 9]]
    check(got, want, tol, False)


@pytest.mark.parametrize("S,N,H,HKV,D,page,past", [
    (1, 12, 4, 2, 128, 64, [20000]),      # 24, 60, 63 and 200 rows over a long cache: many parts of an item
    (2, 30, 4, 2, 64, 32, [9000, 137]),
    (1, 9, 14, 2, 128, 16, [15001]),
    (2, 50, 8, 2, 128, 64, [11000, 300]),
    (1, 100, 4, 2, 64, 256, [16383]),
])
def test_long_caches(be, S, N, H, HKV, D, page, past):
    rng = np.random.default_rng(N)
    c = Cache(rng, S, N, HKV, D, page, past)
    q = rng.standard_normal((S, H, N, D)).astype(np.float32)
    sees = np.stack([sees_of(p) for p in random_parents(rng, S, N)])
    want, tol = attend64(c, q, [N] * S, sees, 1 / math.sqrt(D))
    check(run_attn(be, c, q, None, words_of(sees), 1 / math.sqrt(D)), want, tol, False)


@pytest.mark.parametrize("S,N,H,HKV,D,page", [(33, 1, 2, 1, 128, 64), (70, 5, 4, 2, 64, 16), (40, 40, 4, 2, 128, 32)])
def test_more_sequences_than_lanes(be, S, N, H, HKV, D, page):
    """ragged batches, empty sequences among them"""
    rng = np.random.default_rng(S)
    past = [int(x) for x in rng.integers(0, 700, S)]
    past[0], past[S - 1] = 0, 900
    c = Cache(rng, S, N, HKV, D, page, past)
    live = rng.integers(0, N + 1, S).astype(np.int32)
    live[S - 1] = N
    q = rng.standard_normal((S, H, N, D)).astype(np.float32)
    sees = np.broadcast_to(np.tril(np.ones((N, N), bool)), (S, N, N))
    want, tol = attend64(c, q, live, sees, 0.1)
    check(run_attn(be, c, q, live, None, 0.1), want, tol, False)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("N", [3, 14, 30, 80])
@pytest.mark.parametrize("scale", [-0.11, 0.0])
def test_scales_that_are_not_positive(be, N, scale, f16):
    rng = np.random.default_rng(20)
    c = Cache(rng, 2, N, 2, 128, 16, [150, 0])
    q = rng.standard_normal((2, 4, N, 128)).astype(np.float16 if f16 else np.float32)
    sees = np.stack([sees_of(p) for p in random_parents(rng, 2, N)])
    want, tol = attend64(c, q, [N, N], sees, scale)
    check(run_attn(be, c, q, None, words_of(sees), scale, f16), want, tol, f16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("N", [7, 14, 30, 80])
def test_rows_of_very_different_queries(be, N, D):
    """a row's accuracy goes by its own size, whatever lies beside it in a tile"""
    rng = np.random.default_rng(21)
    c = Cache(rng, 1, N, 2, D, 16, [300])
    size = 2.0 ** rng.integers(-40, 4, (1, 4, N, 1))
    size[0, 1, 2] = 2.0**90      # scores past 2^90: one weight is all that is left
    q = (rng.standard_normal((1, 4, N, D)) * size).astype(np.float32)
    q[0, 2, 3] = 0
    sees = np.tril(np.ones((1, N, N), bool))
    want, tol = attend64(c, q, [N], sees, 0.1)
    check(run_attn(be, c, q, None, None, 0.1), want, tol, False)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("N", [7, 14, 30, 80])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_query_that_is_not_finite_spoils_its_own_row_alone(be, N, bad, f16):
    rng = np.random.default_rng(22)
    c = Cache(rng, 1, N, 2, 128, 16, [200])
    q = rng.standard_normal((1, 4, N, 128)).astype(np.float16 if f16 else np.float32)
    sees = np.tril(np.ones((1, N, N), bool))
    want, tol = attend64(c, q, [N], sees, 0.1)
    q[0, 1, 4, 17] = bad   # times positive and negative keys: the softmax has no value
    got = run_attn(be, c, q, None, None, 0.1, f16)
    assert np.isnan(got[0, 4, 1]).all()
    got[0, 4, 1] = want[0, 4, 1]
    check(got, want, tol, f16)


@pytest.mark.parametrize("layout", ["head", "row"])
@pytest.mark.parametrize("N,H,HKV", [(1, 16, 8), (12, 16, 8), (70, 4, 2)])
def test_strides(be, layout, N, H, HKV):
    """pages with positions slower than heads, q and out inside wider rows, a longer page table"""
    import torch

    rng = np.random.default_rng(10)
    c = Cache(rng, 2, N, HKV, 128, 16, [100, 37], layout=layout)
    q = rng.standard_normal((2, H, N, 128)).astype(np.float32)
    sees = np.broadcast_to(np.tril(np.ones((N, N), bool)), (2, N, N))
    want, tol = attend64(c, q, [N, N], sees, 0.09)
    wide = torch.full((2, N, H + 3, 160), 3.0, device="cuda")
    wide[:, :, 2:H + 2, 16:144] = cuda(q).permute(0, 2, 1, 3)
    out = torch.full((2, N, H + 1, 256), 5.0, device="cuda")
    table = torch.full((2, c.MP + 5), -1, dtype=torch.int32, device="cuda")
    table[:, :c.MP] = cuda(c.table)
    k, v = c.device()
    be.flash_attn_tree(wide[:, :, 2:H + 2, 16:144].permute(0, 2, 1, 3), k, v, table, cuda(c.past), None, None, 0.09,
                       out[:, :, 1:, 64:192])
    be.synchronize()
    check(out[:, :, 1:, 64:192].cpu().double().numpy(), want, tol, False)
    out[:, :, 1:, 64:192] = 5.0
    assert bool((out == 5.0).all()), "nothing outside the view is written"


def test_offsets_past_32_bits(be):
    import torch

    rng = np.random.default_rng(11)
    page, HKV, D = 256, 8, 128
    P = (5 << 30) // (HKV * page * D * 2)
    k, v = (torch.zeros(P, HKV, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    table = np.array([[P - 1, 3, P - 2]], np.int32)
    N, past = 6, 2 * page + 11
    kk, vv = (rng.standard_normal((3, HKV, page, D)).astype(np.float16) for _ in range(2))
    k[torch.from_numpy(table[0]).long().cuda()] = cuda(kk)
    v[torch.from_numpy(table[0]).long().cuda()] = cuda(vv)
    c = Cache(rng, 1, N, HKV, D, page, [past])
    c.k, c.v, c.table, c.P = kk, vv, np.array([[0, 1, 2]], np.int32), 3
    q = rng.standard_normal((1, 16, N, D)).astype(np.float32)
    sees = np.tril(np.ones((1, N, N), bool))
    want, tol = attend64(c, q, [N], sees, 0.1)
    c.table = table
    check(run_attn(be, c, q, None, None, 0.1, pages=(k, v)), want, tol, False)


@pytest.mark.parametrize("S,N,past", [(1, 1, [9000]), (3, 16, [4000, 100, 2500]), (2, 61, [3000, 5000])])
def test_the_same_call_gives_the_same_bits(be, S, N, past):
    rng = np.random.default_rng(12)
    c = Cache(rng, S, N, 8, 128, 64, past)
    q = rng.standard_normal((S, 16, N, 128)).astype(np.float32)
    pages = c.device()
    first = run_attn(be, c, q, None, None, 0.09, pages=pages)
    for _ in range(20):
        assert np.array_equal(first, run_attn(be, c, q, None, None, 0.09, pages=pages))


def test_on_another_stream_and_in_a_captured_step(be):
    """a step captured once is replayed while n_past grows in device memory"""
    import torch

    rng = np.random.default_rng(13)
    N = 5
    c = Cache(rng, 2, N, 4, 128, 16, [300, 200])
    q = rng.standard_normal((2, 8, N, 128)).astype(np.float32)
    sees = np.broadcast_to(np.tril(np.ones((N, N), bool)), (2, N, N))
    k, v = c.device()
    qd, table, past = cuda(q), cuda(c.table), cuda(c.past)
    out = torch.zeros(2, N, 8, 128, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    be.set_stream(side)
    try:
        be.flash_attn_tree(qd, k, v, table, past, None, None, 0.1, out)
        be.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            be.flash_attn_tree(qd, k, v, table, past, None, None, 0.1, out)
        for step in ([300, 200], [17, 64], [0, 299]):
            past.copy_(torch.tensor(step, dtype=torch.int32))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            c.past = np.array(step, np.int32)
            want, tol = attend64(c, q, [N, N], sees, 0.1)
            check(out.cpu().double().numpy(), want, tol, False)
        del g
    finally:
        be.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("N", [30, 70])
def test_a_captured_call_with_a_join(be, N):
    """items shared by many CTAs, replayed with other lengths: long, within a unit, long again"""
    import torch

    rng = np.random.default_rng(23)
    c = Cache(rng, 2, N, 2, 128, 64, [4000, 2500])
    q = rng.standard_normal((2, 4, N, 128)).astype(np.float32)
    sees = np.broadcast_to(np.tril(np.ones((N, N), bool)), (2, N, N))
    k, v = c.device()
    k.nan_to_num_(0.0), v.nan_to_num_(0.0)
    c.k, c.v = np.nan_to_num(c.k), np.nan_to_num(c.v)
    qd, table, past = cuda(q), cuda(c.table), cuda(c.past)
    out = torch.zeros(2, N, 4, 128, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    be.set_stream(side)
    try:
        be.flash_attn_tree(qd, k, v, table, past, None, None, 0.1, out)
        be.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            be.flash_attn_tree(qd, k, v, table, past, None, None, 0.1, out)
            be.flash_attn_tree(qd, k, v, table, past, None, None, 0.1, out)
        for step in ([4000, 2500], [0, 5], [3999, 100]):
            past.copy_(torch.tensor(step, dtype=torch.int32))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            c.past = np.array(step, np.int32)
            want, tol = attend64(c, q, [N, N], sees, 0.1)
            check(out.cpu().double().numpy(), want, tol, False)
        del g
    finally:
        be.set_stream(torch.cuda.current_stream())


@pytest.mark.parametrize("N", [1, 70])
def test_lengths_and_pages_out_of_range_are_reported(be, N):
    import torch

    import openasr_b200 as ob

    rng = np.random.default_rng(14)
    c = Cache(rng, 2, N, 2, 128, 16, [40, 20], fill=None)
    q = rng.standard_normal((2, 4, N, 128)).astype(np.float32)
    sees = np.broadcast_to(np.tril(np.ones((N, N), bool)), (2, N, N))
    want, tol = attend64(c, q, [N, N], sees, 0.1)
    k, v = c.device()

    def call(table, past, live):
        out = torch.zeros(2, N, 4, 128, device="cuda")
        be.flash_attn_tree(cuda(q), k, v, cuda(table), cuda(past), cuda(live), None, 0.1, out)
        be.synchronize()
        return out.cpu().double().numpy()

    full = np.array([N, N], np.int32)
    for page_id in (-1, c.P, 2**31 - 1):
        table = c.table.copy()
        table[1, 0] = page_id
        with pytest.raises(ob.backend.ExecutionFailed):
            call(table, c.past, full)
    for past, live in (([-1, 20], full), ([40, c.MP * 16], full), (c.past, [N, N + 1]), (c.past, [-1, N]),
                       ([2**31 - 1, 20], full)):
        with pytest.raises(ob.backend.ExecutionFailed):
            call(c.table, np.array(past, np.int32), np.array(live, np.int32))
    check(call(c.table, c.past, full), want, tol, False)


# ---- norms, rotation, cache write -----------------------------------------------------------
def norm64(x, w, eps):
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return y if w is None else y * w


def turn64(y, rope, pos):
    h = y.shape[-1] // 2
    c, s = rope[pos][..., 0].astype(np.float64), rope[pos][..., 1].astype(np.float64)
    c, s = c[..., None, :], s[..., None, :]
    a, b = y[..., :h], y[..., h:]
    return np.concatenate([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("layout", ["head", "row"])
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,N,H,HKV,D,page,past,norm,rope,pos", [
    (1, 1, 16, 8, 128, 64, [390], True, True, False),
    (3, 7, 20, 20, 64, 24, [0, 57, 100], False, False, False),
    (2, 61, 16, 8, 128, 16, [129, 3], True, True, True),
    (2, 5, 15, 5, 128, 8, [0, 20], True, True, False),
    (1, 300, 12, 2, 64, 40, [11], False, True, True),
    (4, 33, 6, 6, 64, 16, [0, 1, 2, 3], True, False, False),
])
def test_qk_norm_rope_matches_64_bits(be, S, N, H, HKV, D, page, past, norm, rope, pos, f16, layout):
    import torch

    rng = np.random.default_rng(N)
    c = Cache(rng, S, N, HKV, D, page, past, layout=layout, fill=None)
    x = (rng.standard_normal((S, N, H + 2 * HKV, D)) * 2).astype(np.float32)
    wq, wk = (rng.normal(1, 0.2, D).astype(np.float32) for _ in range(2))
    n_pos = max(past) + N
    ang = np.arange(n_pos)[:, None] * 10000.0 ** (-np.arange(D // 2) * 2.0 / D)
    tab = np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)
    live = np.array([N if s % 2 == 0 else max(1, N - 2) for s in range(S)], np.int32)
    at = c.past[:, None] + np.arange(N)
    turn = rng.integers(0, n_pos, (S, N)).astype(np.int32) if pos else at
    q64 = norm64(x[:, :, :H], wq, 1e-6) if norm else x[:, :, :H].astype(np.float64)
    k64 = norm64(x[:, :, H:H + HKV], wk, 1e-6) if norm else x[:, :, H:H + HKV].astype(np.float64)
    if rope:
        q64, k64 = turn64(q64, tab, turn), turn64(k64, tab, turn)
    wide = torch.zeros(S, N, H + 2 * HKV, D + 16, device="cuda")
    wide[..., 8:D + 8] = cuda(x)
    k, v = c.device()
    q = torch.full((S, N, H, D), 9.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    be.qk_norm_rope(wide[..., 8:D + 8], cuda(wq) if norm else None, cuda(wk) if norm else None, 1e-6,
                    cuda(tab) if rope else None, cuda(turn) if pos else None, cuda(c.table), cuda(c.past), cuda(live), q, k, v)
    be.synchronize()
    got = q.cpu().double().numpy()
    m = max(np.abs(q64).max(), np.abs(k64).max())
    unit = 16 * 2.0**-24 * m
    for s in range(S):
        n = live[s]
        assert (np.abs(got[s, :n] - q64[s, :n]) <= unit + (2.0**-11 * np.abs(q64[s, :n]) if f16 else 0)).all()
        assert not got[s, n:].any()
    ek, ev = c.k.astype(np.float64), c.v.astype(np.float64)
    for s in range(S):
        for i in range(live[s]):
            pg, off = c.table[s, at[s, i] // page], at[s, i] % page
            ek[pg, :, off], ev[pg, :, off] = k64[s, i], x[s, i, H + HKV:]
    gk, gv = k.cpu().double().numpy(), v.cpu().double().numpy()
    assert (np.abs(gk - ek) <= unit + 2.0**-11 * np.abs(ek)).all()
    assert (np.abs(gv - ev) <= 2.0**-11 * np.abs(ev) + 2.0**-25).all()


def test_qk_norm_rope_reports_positions_out_of_range(be):
    import torch

    import openasr_b200 as ob

    rng = np.random.default_rng(3)
    c = Cache(rng, 1, 4, 2, 64, 8, [5], fill=None)
    x = cuda(rng.standard_normal((1, 4, 8, 64)).astype(np.float32))
    tab = cuda(np.ones((9, 32, 2), np.float32))
    q = torch.zeros(1, 4, 4, 64, device="cuda")
    k, v = c.device()
    be.qk_norm_rope(x, None, None, 0.0, tab, None, cuda(c.table), cuda(c.past), None, q, k, v)
    be.synchronize()
    for pos in ([[0, 1, 9, 2]], [[-1, 1, 2, 3]]):
        with pytest.raises(ob.backend.ExecutionFailed):
            be.qk_norm_rope(x, None, None, 0.0, tab, cuda(np.array(pos, np.int32)), cuda(c.table), cuda(c.past), None, q, k, v)
            be.synchronize()
    before = k.clone()
    with pytest.raises(ob.backend.ExecutionFailed):
        be.qk_norm_rope(x * 2, None, None, 0.0, None, None, cuda(np.array([[c.P, -3]], np.int32)), cuda(c.past), None, q, k, v)
        be.synchronize()
    assert torch.equal(before, k)


# ---- acceptance, copies -------------------------------------------------------------------
def commit_plain(c, tok, par, tgt, live):
    S, N = tok.shape
    path, count, nxt = np.full((S, N), -1, np.int32), np.zeros(S, np.int32), np.full(S, -1, np.int32)
    k, v = c.k.copy(), c.v.copy()
    for s in range(S):
        if live[s] == 0:
            continue
        walk = [0]
        while True:
            kids = [j for j in range(walk[-1] + 1, live[s]) if par[s, j] == walk[-1] and tok[s, j] == tgt[s, walk[-1]]]
            if not kids:
                break
            walk.append(kids[0])
        path[s, :len(walk)], count[s], nxt[s] = walk, len(walk), tgt[s, walk[-1]]
        for x in (k, v):
            for layer in range(c.L):
                for to, frm in enumerate(walk):
                    a, b = c.past[s] + frm, c.past[s] + to
                    x[layer * c.P + c.table[s, b // c.page], :, b % c.page] = \
                        x[layer * c.P + c.table[s, a // c.page], :, a % c.page]
    return path, count, nxt, k, v


def settled(c, x, count, N):
    """x with the rows that a commit leaves undefined set to zero"""
    x = x.copy()
    for s in range(c.S):
        for p in range(c.past[s] + count[s], c.past[s] + N):
            x.reshape(c.L, c.P, c.HKV, c.page, c.D)[:, c.table[s, p // c.page], :, p % c.page] = 0
    return x


@pytest.mark.parametrize("layout", ["head", "row"])
@pytest.mark.parametrize("S,N,HKV,D,L,page,past,vocab", [
    (1, 1, 8, 128, 3, 16, [390], 5),
    (3, 16, 8, 128, 4, 16, [5, 700, 63], 3),
    (4, 61, 5, 64, 3, 24, [0, 1, 2, 100], 2),
    (2, 300, 2, 64, 2, 8, [7, 64], 1),        # every child agrees: the first of them
    (3, 40, 1, 128, 1, 64, [0, 63, 64], 2),
])
def test_tree_commit_matches_the_walk(be, S, N, HKV, D, L, page, past, vocab, layout):
    import torch

    rng = np.random.default_rng(N + S)
    c = Cache(rng, S, N, HKV, D, page, past, L=L, layout=layout, fill=None)
    tok, tgt = (rng.integers(0, vocab, (S, N)).astype(np.int32) for _ in range(2))
    par = random_parents(rng, S, N)
    par[:, 1:][rng.random((S, N - 1)) < 0.1] = -1   # not part of the tree
    if N > 20:
        par[0, 11], par[0, 12] = 15, 12             # a later node, itself: never accepted
    live = np.array([N if s % 2 == 0 else max(1, N - 3) for s in range(S)], np.int32)
    if S > 3:
        live[3] = 0
    path, count, nxt, ek, ev = commit_plain(c, tok, par, tgt, live)
    k, v = c.device()
    gp = torch.full((S, N), 77, dtype=torch.int32, device="cuda")
    gc, gn, gq = (torch.full((S,), 77, dtype=torch.int32, device="cuda") for _ in range(3))
    be.tree_commit(cuda(tok), cuda(par), cuda(tgt), cuda(live), cuda(c.past), cuda(c.table), k, v, L, gp, gc, gn, gq)
    be.synchronize()
    assert np.array_equal(gp.cpu().numpy(), path) and np.array_equal(gc.cpu().numpy(), count)
    assert np.array_equal(gn.cpu().numpy(), nxt) and np.array_equal(gq.cpu().numpy(), c.past + count)
    for got, want in ((k, ek), (v, ev)):
        assert np.array_equal(settled(c, got.cpu().numpy(), count, N), settled(c, want, count, N))
    assert N < 16 or count.max() > 2


def test_tree_commit_reports_bad_pages(be):
    import torch

    import openasr_b200 as ob

    rng = np.random.default_rng(2)
    c = Cache(rng, 1, 6, 2, 64, 8, [6], fill=None)
    z = np.zeros((1, 6), np.int32)
    par = np.array([[-1, 0, 0, 2, 3, 4]], np.int32)
    tok = np.array([[0, 5, 0, 0, 0, 0]], np.int32)
    k, v = c.device()
    outs = [torch.zeros(1, 6, dtype=torch.int32, device="cuda")] + [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(3)]
    before = k.clone()
    with pytest.raises(ob.backend.ExecutionFailed):
        be.tree_commit(cuda(tok), cuda(par), cuda(z), None, cuda(c.past), cuda(np.array([[0, c.P]], np.int32)), k, v, 1, *outs)
        be.synchronize()
    with pytest.raises(ob.backend.ExecutionFailed):
        be.tree_commit(cuda(tok), cuda(par), cuda(z), None, cuda(np.array([99], np.int32)), cuda(c.table), k, v, 1, *outs)
        be.synchronize()
    assert torch.equal(before, k)


@pytest.mark.parametrize("layout", ["head", "row"])
@pytest.mark.parametrize("n,HKV,D,L,page", [(1, 1, 64, 1, 8), (5, 8, 128, 3, 16), (7, 5, 64, 2, 24), (3, 2, 128, 4, 256)])
def test_kv_pages_copy(be, n, HKV, D, L, page, layout):
    rng = np.random.default_rng(n)
    c = Cache(rng, 1, 1, HKV, D, page, [0], L=L, layout=layout, spare=2 * n + 2)
    c.k, c.v = (rng.integers(0, 2**16, x.shape, dtype=np.uint16).view(np.float16) for x in (c.k, c.v))  # any bits
    order = rng.permutation(c.P)
    pairs = np.stack([order[:n][rng.integers(0, n, n)], order[n:2 * n]], 1).astype(np.int32)
    pairs = np.concatenate([pairs, [[-1, order[-1]], [order[0], -1]]]).astype(np.int32)
    k, v = c.device()
    be.kv_pages_copy(k, v, L, cuda(pairs))
    be.synchronize()
    for got, x in ((k, c.k), (v, c.v)):
        w = x.copy().reshape(L, c.P, HKV, page, D)
        for a, b in pairs[:n]:
            w[:, b] = w[:, a]
        assert np.array_equal(got.cpu().numpy().view(np.uint16), w.reshape(x.shape).view(np.uint16))


def test_kv_pages_copy_reports_bad_pages(be):
    import torch

    import openasr_b200 as ob

    c = Cache(np.random.default_rng(1), 1, 1, 2, 64, 8, [0], fill=None)
    k, v = c.device()
    before = k.clone()
    for pair in ([0, c.P], [c.P, 0]):
        with pytest.raises(ob.backend.ExecutionFailed):
            be.kv_pages_copy(k, v, 1, cuda(np.array([pair], np.int32)))
            be.synchronize()
    assert torch.equal(before, k)
    be.kv_pages_copy(k, v, 1, torch.empty(0, 2, dtype=torch.int32, device="cuda"))


# ---- refusals --------------------------------------------------------------------------------
def test_refusals(be):
    import torch

    import openasr_b200 as ob

    def z(*shape, dtype=torch.float32):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    i32, f16 = torch.int32, torch.float16
    S, N, H, HKV, D, page, P = 2, 3, 4, 2, 64, 16, 5
    ok = dict(q=z(S, H, N, D), k=z(P, HKV, page, D, dtype=f16), v=z(P, HKV, page, D, dtype=f16), table=z(S, 2, dtype=i32),
              past=z(S, dtype=i32), nodes=None, tree=z(S, N, 1, dtype=i32), scale=0.1, out=z(S, N, H, D))

    def attn(**kw):
        a = {**ok, **kw}
        be.flash_attn_tree(a["q"], a["k"], a["v"], a["table"], a["past"], a["nodes"], a["tree"], a["scale"], a["out"])
        be.synchronize()

    attn()
    pages = lambda *s, dtype=f16: dict(k=z(*s, dtype=dtype), v=z(*s, dtype=dtype))  # noqa: E731
    for kw in (
        pages(P, HKV, page, D, dtype=torch.float32), pages(P, HKV, 12, D), pages(P, HKV, page, 96), pages(P, 3, page, D),
        dict(v=z(P, HKV, page + 8, D, dtype=f16)), dict(k=z(P, HKV, page, 2 * D, dtype=f16)[..., ::2]),
        dict(k=z(P, HKV, page, D + 4, dtype=f16)[..., :D], v=z(P, HKV, page, D + 4, dtype=f16)[..., :D]),
        dict(q=z(S, H, N, 128)), dict(q=z(S, H, N, D, dtype=i32)), dict(q=z(S, H, N, D + 1)[..., :D]),
        dict(out=z(S, N, H, D, dtype=i32)), dict(out=z(S, H, N, D)), dict(out=z(S, N, H, D + 2)[..., :D]),
        dict(table=z(S + 1, 2, dtype=i32)), dict(table=z(S, 2, dtype=torch.int64)), dict(past=z(S + 1, dtype=i32)),
        dict(past=z(S)), dict(nodes=z(S - 1, dtype=i32)), dict(tree=z(S, N, 2, dtype=i32)), dict(tree=z(S, N + 1, 1, dtype=i32)),
        dict(tree=z(S, N, 1)), dict(scale=float("nan")),
        dict(q=z(S, H, 1025, D), out=z(S, 1025, H, D), tree=z(S, 1025, 33, dtype=i32), table=z(S, 70, dtype=i32)),
    ):
        with pytest.raises(ob.backend.UnsupportedInputs):
            attn(**kw)

    nr = dict(x=z(S, N, H + 2 * HKV, D), wq=z(D), wk=z(D), eps=1e-6, rope=z(40, D // 2, 2), pos=z(S, N, dtype=i32),
              table=ok["table"], past=ok["past"], nodes=None, q=z(S, N, H, D), k=ok["k"], v=ok["v"])

    def norm(**kw):
        be.qk_norm_rope(*{**nr, **kw}.values())
        be.synchronize()

    norm()
    for kw in (dict(x=z(S, N, H + 2 * HKV, D, dtype=f16)), dict(x=z(S, N, 2 * HKV, D)), dict(x=z(S, N, H + 2 * HKV + 1, D)),
               dict(wq=z(D + 1)), dict(wk=z(D, dtype=f16)), dict(eps=-1.0), dict(eps=float("nan")), dict(rope=z(40, D, 2)),
               dict(rope=z(40, D // 2, 2, dtype=f16)), dict(pos=z(S, N + 1, dtype=i32)), dict(q=z(S, N, H + 1, D)),
               dict(q=z(S, H, N, D)), dict(x=z(S, N, H + 2 * HKV, D + 1)[..., :D]), dict(table=z(S, 2))):
        with pytest.raises(ob.backend.UnsupportedInputs):
            norm(**kw)

    n2 = z(S, N, dtype=i32)
    n1 = [z(S, dtype=i32) for _ in range(3)]
    cm = dict(tok=n2, par=n2.clone(), tgt=n2.clone(), nodes=None, past=ok["past"], table=ok["table"], k=ok["k"], v=ok["v"], L=1,
              path=n2.clone(), count=n1[0], nxt=n1[1], past_out=n1[2])

    def commit(**kw):
        be.tree_commit(*{**cm, **kw}.values())
        be.synchronize()

    commit()
    for kw in (dict(L=0), dict(L=2), dict(tok=z(S, N)), dict(par=z(S, N + 1, dtype=i32)), dict(path=z(S, N - 1, dtype=i32)),
               dict(count=z(S + 1, dtype=i32)), dict(past_out=ok["past"]), dict(nxt=z(S)),
               dict(tok=z(S, 0, dtype=i32), par=z(S, 0, dtype=i32), tgt=z(S, 0, dtype=i32), path=z(S, 0, dtype=i32))):
        with pytest.raises(ob.backend.UnsupportedInputs):
            commit(**kw)

    for L, pairs in ((2, z(1, 2, dtype=i32)), (0, z(1, 2, dtype=i32)), (1, z(1, 3, dtype=i32)), (1, z(1, 2))):
        with pytest.raises(ob.backend.UnsupportedInputs):
            be.kv_pages_copy(ok["k"], ok["v"], L, pairs)


def test_supports_op(be):
    import torch

    import openasr_b200 as ob
    from openasr_b200 import backend as bk

    d = ob.describe
    k = d(torch.zeros(4, 2, 16, 64, dtype=torch.float16, device="cuda"))
    k12 = d(torch.zeros(4, 2, 12, 64, dtype=torch.float16, device="cuda"))
    q = d(torch.zeros(1, 4, 3, 64, device="cuda"))
    assert be.supports_op(bk.OP_FLASH_ATTN_TREE, q, k) and not be.supports_op(bk.OP_FLASH_ATTN_TREE, q, k12)
    assert be.supports_op(bk.OP_QK_NORM_ROPE, d(torch.zeros(1, 3, 8, 64, device="cuda")), k)
    assert not be.supports_op(bk.OP_QK_NORM_ROPE, d(torch.zeros(1, 3, 7, 64, device="cuda")), k)
    assert be.supports_op(bk.OP_TREE_COMMIT, d(torch.zeros(1, 3, dtype=torch.int32, device="cuda")), k)
    assert be.supports_op(bk.OP_KV_PAGES_COPY, k) and not be.supports_op(bk.OP_KV_PAGES_COPY, k12)
