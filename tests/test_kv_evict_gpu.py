"""Attention added up per cached position, and eviction by it, against plain implementations in 64 bits.

Tolerances come from the arithmetic.  A score is off by at most ds = 2^-20 * |scale| * max sum|q||k| (D <= 128
roundings of 2^-24 and as much again for an operand kept in two 16-bit halves, its scaling included), a weight
by a factor of 1 +- (2 ds + 2^-20) (its own score, the row's sum, two exponentials of 2^-22); sums over R rows
add R 2^-24, the old value times decay two roundings of 2^-24.  Eviction moves values: bit for bit."""
import math

import numpy as np
import pytest

from test_pages_gpu import Cache, cuda

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    import torch

    import openasr_b200 as ob

    b = ob.Backend(0)
    b.set_stream(torch.cuda.current_stream())
    yield b
    b.close()


# ---- attention added up ------------------------------------------------------------------------
def added64(c, q, live, scale, decay, old):
    """new entries [P, HKV, page] in 64 bits, and what they may be off by"""
    S, H, N, D = q.shape
    G = H // c.HKV
    out, tol = old.astype(np.float64), np.zeros(old.shape)
    for s in range(S):
        n = int(live[s])
        T = int(c.past[s]) + n
        if n == 0:
            continue
        k = c.rows(c.k, s, T).astype(np.float64)
        p = np.arange(T)
        pg, off = c.table[s, p // c.page], p % c.page
        hide = p[None] > c.past[s] + np.arange(n)[:, None]
        for h in range(c.HKV):
            got, err = np.zeros(T), np.zeros(T)
            for a in range(h * G, (h + 1) * G):
                x = q[s, a, :n].astype(np.float64) @ k[h].T * scale
                x[hide] = -np.inf
                w = np.exp(x - x.max(-1, keepdims=True))
                w /= w.sum(-1, keepdims=True)
                size = np.where(hide, 0, np.abs(q[s, a, :n].astype(np.float64)) @ np.abs(k[h]).T).max(-1, keepdims=True)
                got += w.sum(0)
                err += (w * (2 * 2.0**-20 * abs(scale) * size + 2.0**-20)).sum(0)
            kept = np.where(p < c.past[s], out[pg, h, off] * decay if decay else 0.0, 0.0)
            out[pg, h, off] = kept + got
            tol[pg, h, off] = err + (n * G + 8) * 2.0**-24 * got + 2.0**-22 * np.abs(kept)
    return out, tol


def run_weights(be, c, q, live, scale, decay, old, k=None, f16=False, q_view=None, w_view=None):
    import torch

    w = w_view if w_view is not None else cuda(old)
    be.attn_weights(q_view if q_view is not None else cuda(q, torch.float16 if f16 else torch.float32), k if k is not None else c.device()[0],
                    cuda(c.table), cuda(c.past), None if live is None else cuda(live), scale, decay, w)
    be.synchronize()
    return w.cpu().double().numpy()


def entries(rng, c):
    """old entries: NaN where nothing has been scored yet (new positions, and past the end)"""
    w = np.full((c.P, c.HKV, c.page), np.nan, np.float32)
    for s in range(c.S):
        for p in range(int(c.past[s])):
            w[c.table[s, p // c.page], :, p % c.page] = rng.random(c.HKV) * 3
    return w


def check(got, want, tol):
    bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)))
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.nanmax(np.abs(got - want) / np.maximum(tol, 1e-30))} times the bound"


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("decay", [1.0, 0.0, 0.75])
@pytest.mark.parametrize("S,N,H,HKV,D,page,past", [
    (1, 1, 16, 8, 128, 64, [390]),
    (1, 1, 16, 8, 128, 64, [0]),                # the first token gets all of its own attention
    (3, 1, 20, 20, 64, 16, [0, 63, 441]),
    (2, 4, 16, 8, 128, 16, [5, 700]),           # 8 rows
    (2, 5, 16, 8, 128, 24, [129, 1]),           # 10 rows
    (2, 32, 20, 20, 64, 24, [57, 300]),
    (1, 61, 8, 1, 128, 40, [333]),              # 488 rows of one head
    (1, 3, 6, 6, 64, 8, [1021]),
    (1, 17, 15, 5, 64, 256, [257]),
    (2, 2, 32, 4, 128, 64, [2500, 2049]),
    (40, 1, 8, 8, 64, 8, list(range(40))),      # more heads than SMs
])
def test_attn_weights_matches_64_bits(be, S, N, H, HKV, D, page, past, decay, f16):
    rng = np.random.default_rng(S * 100 + N)
    c = Cache(rng, S, N, HKV, D, page, past)
    q = rng.standard_normal((S, H, N, D)).astype(np.float16 if f16 else np.float32)
    live = np.array([N if s % 2 == 0 else N - 1 - N // 3 if N > 1 else 1 for s in range(S)], np.int32)
    for s in range(S):  # rows of padding nodes are garbage too
        for p in range(c.past[s] + live[s], c.past[s] + N):
            c.k[c.table[s, p // page], :, p % page] = np.nan
    old = entries(rng, c)
    scale = 1 / math.sqrt(D)
    want, tol = added64(c, q, live, scale, decay, old)
    check(run_weights(be, c, q, live, scale, decay, old, f16=f16), want, tol)


@pytest.mark.parametrize("S,N,H,HKV,D,page,past", [(1, 1, 8, 4, 128, 64, [30011]), (2, 9, 2, 1, 64, 16, [20003, 9]), (1, 3, 4, 1, 128, 128, [60001])])
def test_long_caches(be, S, N, H, HKV, D, page, past):
    """more positions than a CTA keeps the scores of"""
    rng = np.random.default_rng(N)
    c = Cache(rng, S, N, HKV, D, page, past, spare=0)
    q = rng.standard_normal((S, H, N, D)).astype(np.float32)
    old = entries(rng, c)
    live = np.full(S, N, np.int32)
    want, tol = added64(c, q, live, 0.1, 1.0, old)
    check(run_weights(be, c, q, None, 0.1, 1.0, old), want, tol)


@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales_and_sizes_of_rows(be, scale):
    """rows of very different queries keep their own accuracy; scores of hundreds"""
    rng = np.random.default_rng(9)
    c = Cache(rng, 2, 5, 4, 128, 16, [100, 31])
    q = rng.standard_normal((2, 8, 5, 128)).astype(np.float32)
    q *= 10.0 ** rng.integers(-8, 2, (2, 8, 5, 1))
    old = entries(rng, c)
    want, tol = added64(c, q, [5, 5], scale, 1.0, old)
    check(run_weights(be, c, q, None, scale, 1.0, old), want, tol)


def test_the_weights_of_a_row_add_up_to_one(be):
    rng = np.random.default_rng(10)
    c = Cache(rng, 3, 2, 4, 64, 16, [50, 0, 333])
    q = rng.standard_normal((3, 12, 2, 64)).astype(np.float32)
    got = run_weights(be, c, q, None, 0.125, 0.0, entries(rng, c))
    for s in range(3):
        p = np.arange(c.past[s] + 2)
        total = got[c.table[s, p // 16], :, p % 16].sum(0)
        assert (np.abs(total - 2 * 3) <= 6 * 2.0**-18).all()


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_what_is_not_finite_stays_with_its_row(be, bad, f16):
    """a spoiled query reaches what it sees, a spoiled key the rows that see it; nothing else"""
    import torch

    rng = np.random.default_rng(12)
    c = Cache(rng, 2, 4, 2, 64, 16, [40, 20])
    q = rng.standard_normal((2, 2, 4, 64)).astype(np.float16 if f16 else np.float32)
    q[0, 1, 1, 7] = bad                                           # head 1, node 1 of sequence 0: sees positions 0..41
    c.k[c.table[1, 22 // 16], 0, 22 % 16, 3] = bad                # head 0, node 2 of sequence 1
    got = run_weights(be, c, q, None, 0.125, 0.0, entries(rng, c), f16=f16)
    at = lambda s, h, n: got[c.table[s, np.arange(n) // 16], h, np.arange(n) % 16]  # noqa: E731
    assert np.isnan(at(0, 1, 44)[:42]).all() and np.isfinite(at(0, 1, 44)[42:]).all()
    assert np.isfinite(at(0, 0, 44)).all() and np.isfinite(at(1, 1, 24)).all()
    # a key whose score is -inf gets nothing and spoils nobody; otherwise the rows that see it are NaN
    row = at(1, 0, 24)
    if np.isnan(bad):
        assert np.isnan(row[:24]).all()
    assert torch.isfinite(torch.tensor(got[c.table[0, 0], 0])).all()


def test_positions_past_the_last_node_stay(be):
    rng = np.random.default_rng(13)
    c = Cache(rng, 2, 6, 2, 64, 16, [10, 29], fill=0)
    old = rng.random((c.P, 2, 16)).astype(np.float32)
    live = np.array([3, 0], np.int32)
    got = run_weights(be, c, rng.standard_normal((2, 2, 6, 64)).astype(np.float32), live, 0.125, 1.0, old)
    for s, T in ((0, 13), (1, 0)):
        for p in range(T, c.MP * 16):
            np.testing.assert_array_equal(got[c.table[s, p // 16], :, p % 16], old[c.table[s, p // 16], :, p % 16])


@pytest.mark.parametrize("layout", ["head", "row"])
def test_strides(be, layout):
    import torch

    rng = np.random.default_rng(14)
    S, N, H, HKV, D, page = 2, 3, 8, 4, 128, 24
    c = Cache(rng, S, N, HKV, D, page, [100, 51], layout=layout)
    q = rng.standard_normal((S, H, N, D)).astype(np.float32)
    wide = torch.zeros(S, N, H + 2, D + 4, device="cuda")
    view = wide.permute(0, 2, 1, 3)[:, 1:-1, :, :D]
    view.copy_(torch.from_numpy(q))
    old = entries(rng, c)
    w = torch.zeros(HKV, c.P, page + 3, device="cuda").permute(1, 0, 2)[:, :, 1:page + 1]
    w.copy_(torch.from_numpy(old))
    want, tol = added64(c, q, [N] * S, 0.09, 0.5, old)
    check(run_weights(be, c, q, None, 0.09, 0.5, old, q_view=view, w_view=w), want, tol)


def test_the_same_call_gives_the_same_bits_and_in_a_captured_step(be):
    import torch

    rng = np.random.default_rng(15)
    S, N, H, HKV, D, page = 3, 4, 16, 8, 128, 16
    c = Cache(rng, S, N, HKV, D, page, [700, 33, 250])
    c.past[:] -= 3  # the captured step replays while the sequences grow
    q, old = rng.standard_normal((S, H, N, D)).astype(np.float32), entries(rng, c)
    first = run_weights(be, c, q, None, 0.1, 1.0, old)
    np.testing.assert_array_equal(first, run_weights(be, c, q, None, 0.1, 1.0, old))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    be.set_stream(stream)
    try:
        qd, k, table, past, w = cuda(q), c.device()[0], cuda(c.table), cuda(c.past), cuda(old)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            be.attn_weights(qd, k, table, past, None, 0.1, 1.0, w)
        for step in range(3):
            want, tol = added64(c, q, [N] * S, 0.1, 1.0, w.cpu().numpy())
            with torch.cuda.stream(stream):
                graph.replay()
            be.synchronize()
            check(w.cpu().double().numpy(), want, tol)
            c.past += 1
            past.copy_(torch.from_numpy(c.past))
            torch.cuda.synchronize()
    finally:
        be.set_stream(torch.cuda.current_stream())


def test_lengths_and_pages_out_of_range_are_reported(be):
    import openasr_b200 as ob

    rng = np.random.default_rng(16)
    for spoil in ("page", "low", "past", "nodes", "more"):
        c = Cache(rng, 2, 2, 2, 64, 16, [40, 20])
        old, live = entries(rng, c), np.array([2, 2], np.int32)
        want = run_weights(be, c, np.ones((2, 2, 2, 64), np.float32), live, 0.1, 1.0, old)
        other = c.table[1, :2].copy()
        if spoil == "page":
            c.table[0, 1] = c.P
        elif spoil == "low":
            c.table[0, 0] = -1
        elif spoil == "past":
            c.past[0] = -1
        elif spoil == "nodes":
            live[0] = 3
        else:
            c.past[0] = c.MP * 16
        with pytest.raises(ob.GgmlBackendError, match="out-of-range"):
            w = cuda(old)
            be.attn_weights(cuda(np.ones((2, 2, 2, 64), np.float32)), c.device()[0], cuda(c.table), cuda(c.past), cuda(live), 0.1, 1.0, w)
            be.synchronize()
        np.testing.assert_array_equal(w.cpu().numpy()[other].astype(np.float64), want[other]), "the other sequence is not touched"


# ---- eviction ------------------------------------------------------------------------------------
def evict_host(c, w, keep, sink, recent):
    """in place: c.k, c.v, w [L * P, HKV, page]; -> n_past_out"""
    out = c.past.copy()
    for s in range(c.S):
        T, K = int(c.past[s]), int(keep[s])
        if T <= K:
            continue
        out[s] = K
        to = np.arange(K)
        for layer in range(c.L):
            rows = c.table[s] + layer * c.P
            for h in range(c.HKV):
                mid = np.arange(sink, T - recent)
                x = w[rows[mid // c.page], h, mid % c.page].astype(np.float64)
                rank = np.lexsort((mid, np.where(np.isnan(x), 0, -x), np.isnan(x)))  # NaN last, then by weight, then by position
                best = np.sort(mid[rank[:K - sink - recent]])
                pick = np.concatenate([np.arange(sink), best, np.arange(T - recent, T)])
                for a in (c.k, c.v, w):
                    a[rows[to // c.page], h, to % c.page] = a[rows[pick // c.page], h, pick % c.page]
    return out


def run_evict(be, c, w, keep, sink, recent, views=None):
    import torch

    k, v, wd = views or (*c.device(), cuda(w))
    out = torch.full((c.S,), -5, dtype=torch.int32, device="cuda")
    be.kv_evict(wd, cuda(c.table), cuda(c.past), cuda(np.asarray(keep, np.int32)), sink, recent, k, v, c.L, out)
    be.synchronize()
    return k.cpu().numpy(), v.cpu().numpy(), wd.cpu().numpy(), out.cpu().numpy()


def same_after(be, c, w, keep, sink, recent, views=None):
    got = run_evict(be, c, w, keep, sink, recent, views)
    out = evict_host(c, w, keep, sink, recent)
    for a, b in zip(got, (c.k, c.v, w, out)):
        np.testing.assert_array_equal(a.view(np.uint8) if a.flags.c_contiguous else np.ascontiguousarray(a).view(np.uint8),
                                      np.ascontiguousarray(b).view(np.uint8))


@pytest.mark.parametrize("kind", ["random", "ties", "odd"])
@pytest.mark.parametrize("S,HKV,D,L,page,past,keep,sink,recent", [
    (1, 8, 128, 1, 64, [512], [448], 4, 64),
    (3, 2, 64, 3, 16, [300, 20, 700], [100, 50, 700], 4, 16),   # one below its budget, one at it
    (2, 4, 128, 2, 24, [257, 1000], [256, 1], 0, 0),            # one position left
    (2, 1, 64, 1, 8, [9, 64], [8, 63], 8, 0),                   # nothing competes
    (1, 3, 128, 2, 40, [333], [100], 0, 100),                   # the last ones alone
    (1, 1, 64, 1, 16, [5000], [2500], 1, 7),
    (2, 2, 64, 1, 256, [100, 255], [0, 10], 0, 0),              # everything
    (1, 20, 64, 4, 16, [1025], [513], 16, 32),
    (5, 2, 128, 1, 8, [0, 1, 2, 3, 40], [1, 1, 1, 1, 17], 1, 0),
])
def test_kv_evict_matches_the_host(be, S, HKV, D, L, page, past, keep, sink, recent, kind):
    rng = np.random.default_rng(len(kind) + past[0])
    c = Cache(rng, S, 0, HKV, D, page, past, L=L, fill=None)
    w = rng.random((L * c.P, HKV, page)).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 3, w.shape).astype(np.float32) / 2
    elif kind == "odd":  # signs, both zeros, infinities, NaN of both signs, numbers next to one another
        pick = np.array([0.0, -0.0, 1.0, np.nextafter(np.float32(1), np.float32(2)), -1.0, np.inf, -np.inf, np.nan, -np.nan, 1e-45, -3e38], np.float32)
        w = pick[rng.integers(0, len(pick), w.shape)]
    same_after(be, c, w, keep, sink, recent)


@pytest.mark.parametrize("past,keep", [([32003, 30011], [8000, 29000]), ([70001, 5], [35000, 5])])
def test_long_sequences(be, past, keep):
    rng = np.random.default_rng(past[0])
    c = Cache(rng, 2, 0, 1, 64, 64, past, L=2, fill=None)
    w = np.exp(rng.standard_normal((2 * c.P, 1, 64)) * 2).astype(np.float32)
    same_after(be, c, w, keep, 4, 2)


def test_evict_strides(be):
    import torch

    rng = np.random.default_rng(21)
    c = Cache(rng, 2, 0, 4, 64, 24, [200, 131], L=2, layout="row", fill=None)
    w = rng.random((2 * c.P, 4, 24)).astype(np.float32)
    wd = torch.zeros(4, 2 * c.P, 27, device="cuda").permute(1, 0, 2)[:, :, 2:26]
    wd.copy_(torch.from_numpy(w))
    same_after(be, c, w, [150, 64], 2, 20, (*c.device(), wd))


def test_evict_is_captured_and_repeated(be):
    import torch

    rng = np.random.default_rng(22)
    c = Cache(rng, 2, 0, 2, 64, 16, [90, 40], L=2, fill=None)
    w = rng.random((2 * c.P, 2, 16)).astype(np.float32)
    stream = torch.cuda.Stream()
    be.set_stream(stream)
    try:
        k, v = c.device()
        wd, table, past, keep = cuda(w), cuda(c.table), cuda(c.past), cuda(np.array([60, 60], np.int32))
        out = torch.zeros(2, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            be.kv_evict(wd, table, past, keep, 2, 8, k, v, 2, out)
        for lengths in ([90, 40], [61, 96], [10, 60]):
            c.past[:] = lengths
            past.copy_(torch.from_numpy(c.past))
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                graph.replay()
            be.synchronize()
            want = evict_host(c, w, [60, 60], 2, 8)
            for a, b in ((k, c.k), (v, c.v), (wd, w), (out, want)):
                np.testing.assert_array_equal(a.cpu().numpy(), b)
    finally:
        be.set_stream(torch.cuda.current_stream())


def test_evict_reports_what_does_not_fit(be):
    import openasr_b200 as ob

    for spoil in ("page", "low", "past", "more", "keep", "negative"):
        rng = np.random.default_rng(23)
        c = Cache(rng, 2, 0, 2, 64, 16, [60, 33], fill=None)
        w = rng.random((c.P, 2, 16)).astype(np.float32)
        keep = np.array([40, 20], np.int32)
        k, v, wd = (*c.device(), cuda(w))
        table, past = c.table.copy(), c.past.copy()
        if spoil == "page":
            table[0, 3] = c.P
        elif spoil == "low":
            table[0, 0] = -1
        elif spoil == "past":
            past[0] = -1
        elif spoil == "more":
            past[0] = 16 * c.MP + 1
        elif spoil == "keep":
            keep[0] = 11
        else:
            keep[0] = -1
        import torch

        out = torch.zeros(2, dtype=torch.int32, device="cuda")
        be.kv_evict(wd, cuda(table), cuda(past), cuda(keep), 4, 8, k, v, 1, out)
        with pytest.raises(ob.GgmlBackendError, match="out-of-range"):
            be.synchronize()
        before = c.k.copy()
        c.past[0] = 0
        evict_host(c, w, [40, 20], 4, 8)
        mine, other = c.table[1], c.table[0]
        np.testing.assert_array_equal(k.cpu().numpy()[mine], c.k[mine])
        np.testing.assert_array_equal(k.cpu().numpy()[other], before[other])
        assert int(out[1]) == 20


def test_a_cache_kept_at_its_budget(be):
    """Steps of a decoder over a bounded cache, pages from the pool: rows written, attended to, scored,
    evicted.  The cache holds what a host that keeps lists of rows holds, bit for bit."""
    import torch

    import openasr_b200 as ob

    rng = np.random.default_rng(24)
    S, N, H, HKV, D, page, L, keep, sink, recent = 2, 5, 4, 2, 64, 8, 2, 24, 2, 6
    pool = ob.KvPool(40, page, 8, S)
    seqs = [pool.open() for _ in range(S)]
    P = 40
    k, v = (torch.zeros(L * P, HKV, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    w = torch.full((L * P, HKV, page), np.nan, device="cuda")
    rope = torch.randn(200, D // 2, 2, device="cuda")
    past = np.zeros(S, np.int32)
    seen = np.zeros(S, np.int32)  # positions counted on through evictions
    rows = {}                     # (layer, s, h) -> list of (k, v, weight)
    evictions = 0
    for step in range(12):
        n = np.array([N, 1 + step % N], np.int32)
        for s in range(S):
            assert len(pool.extend(seqs[s], int(past[s]), int(past[s] + n[s]))) == 0
        table = np.where((t := pool.table(seqs)) < 0, 0, t).astype(np.int32)
        dev = [cuda(a) for a in (table, past, n)]
        pos = cuda((seen[:, None] + np.arange(N)).astype(np.int32))
        for layer in range(L):
            part = slice(layer * P, (layer + 1) * P)
            qkv = torch.randn(S, N, H + 2 * HKV, D, device="cuda")
            q, o = torch.zeros(S, N, H, D, device="cuda"), torch.zeros(S, N, H, D, device="cuda")
            be.qk_norm_rope(qkv, None, None, 0.0, rope, pos, *dev, q, k[part], v[part])
            be.flash_attn_tree(q.permute(0, 2, 1, 3), k[part], v[part], *dev, None, 0.125, o)
            be.attn_weights(q.permute(0, 2, 1, 3), k[part], *dev, 0.125, 0.9, w[part])
            be.synchronize()
            kk, vv, ww = (x[part].cpu().numpy() for x in (k, v, w))
            for s in range(S):
                p = np.arange(past[s] + n[s])
                pg, off = table[s, p // page], p % page
                for h in range(HKV):
                    have = rows.setdefault((layer, s, h), [])
                    for j, (a, b, _) in enumerate(have):  # what was there is still there
                        np.testing.assert_array_equal(kk[pg[j], h, off[j]], a)
                        np.testing.assert_array_equal(vv[pg[j], h, off[j]], b)
                    rows[layer, s, h] = [(kk[pg[j], h, off[j]].copy(), vv[pg[j], h, off[j]].copy(), ww[pg[j], h, off[j]]) for j in p]
                    assert np.isfinite([x[2] for x in rows[layer, s, h]]).all()
        past += n
        seen += n
        out = torch.zeros(S, dtype=torch.int32, device="cuda")
        be.kv_evict(w, dev[0], cuda(past), cuda(np.full(S, keep, np.int32)), sink, recent, k, v, L, out)
        be.synchronize()
        for key, have in rows.items():
            T = len(have)
            if T > keep:
                mid = sorted(range(sink, T - recent), key=lambda j: (-have[j][2], j))[:keep - sink - recent]
                rows[key] = [have[j] for j in list(range(sink)) + sorted(mid) + list(range(T - recent, T))]
        evictions += int((past > keep).sum())
        past = out.cpu().numpy()
        assert (past == np.minimum(past, keep)).all()
        for s in range(S):
            pool.truncate(seqs[s], int(past[s]))
    assert evictions > S * 3
    pool.close_pool()


def test_refusals(be):
    import torch

    import openasr_b200 as ob

    S, N, H, HKV, D, page, P = 2, 3, 4, 2, 64, 16, 6

    def f(*d):
        return torch.zeros(*d, device="cuda")

    def i(*d):
        return torch.zeros(*d, dtype=torch.int32, device="cuda")

    base = dict(q=f(S, H, N, D), k=f(P, HKV, page, D).half(), v=f(P, HKV, page, D).half(), table=i(S, 3), past=i(S), live=i(S), scale=0.1,
                decay=1.0, w=f(P, HKV, page), keep=i(S), sink=0, recent=0, L=1, out=i(S))
    for change, says in (
            (dict(q=f(S, 3, N, D)), "q must be"), (dict(q=f(S, H, N, 128)), "q must be"), (dict(q=i(S, H, N, D)), "q must be"),
            (dict(q=f(S, H, N, D + 1)[..., :D]), "16-byte"), (dict(q=f(S, H, D, N).transpose(2, 3)), "contiguous"),
            (dict(k=f(P, HKV, page, D)), "must be F16"), (dict(k=f(P, HKV, 12, D).half()), "multiple of 8"),
            (dict(w=f(P, HKV, page + 1)), "weights must be"), (dict(w=f(P, page, HKV)), "weights must be"), (dict(w=f(P, HKV, page).half()), "weights must be"),
            (dict(scale=math.nan), "scale"), (dict(decay=-0.5), "decay"), (dict(decay=math.inf), "decay"), (dict(decay=math.nan), "decay"),
            (dict(table=i(3, S)), "page_table"), (dict(past=f(S)), "n_past"), (dict(live=i(S + 1)), "n_nodes")):
        a = {**base, **change}
        with pytest.raises(ob.GgmlBackendError, match=says):
            be.attn_weights(a["q"], a["k"], a["table"], a["past"], a["live"], a["scale"], a["decay"], a["w"])
    both = i(2 * S)
    for change, says in (
            (dict(v=f(P, HKV, page, 128).half()), "one shape"), (dict(k=f(P, HKV, page, D), v=f(P, HKV, page, D)), "must be F16"),
            (dict(w=f(P, HKV, page + 1)), "weights must be"), (dict(L=4), "n_layers"), (dict(L=0), "n_layers"), (dict(sink=-1), "negative"),
            (dict(recent=-1), "negative"), (dict(keep=f(S)), "n_keep"), (dict(keep=i(S + 1)), "n_keep"), (dict(out=i(S, 1)), "n_past_out"),
            (dict(out=base["past"]), "overlap"), (dict(out=base["keep"]), "overlap"), (dict(keep=both[:S], out=both[1:S + 1]), "overlap"),
            (dict(table=i(S + 1, 3)), "page_table")):
        a = {**base, **change}
        with pytest.raises(ob.GgmlBackendError, match=says):
            be.kv_evict(a["w"], a["table"], a["past"], a["keep"], a["sink"], a["recent"], a["k"], a["v"], a["L"], a["out"])
    # nothing to do
    be.attn_weights(f(0, H, N, D), base["k"], i(0, 3), i(0), None, 0.1, 1.0, base["w"])
    be.attn_weights(f(S, H, 0, D), base["k"], base["table"], base["past"], None, 0.1, 1.0, base["w"])
    be.kv_evict(base["w"], i(0, 3), i(0), i(0), 0, 0, base["k"], base["v"], 1, i(0))
    be.synchronize()


def test_supports_op(be):
    import torch

    import openasr_b200 as ob
    from openasr_b200 import backend as bk

    k = ob.describe(torch.zeros(6, 2, 16, 64, dtype=torch.float16))
    for op, yes, no in ((bk.OP_ATTN_WEIGHTS, torch.zeros(2, 4, 3, 64), torch.zeros(2, 3, 3, 64)),
                        (bk.OP_KV_EVICT, torch.zeros(6, 2, 16), torch.zeros(6, 2, 24))):
        assert be.supports_op(op, ob.describe(yes), k)
        assert not be.supports_op(op, ob.describe(no), k)
        assert not be.supports_op(op, ob.describe(yes))


def test_lengths_past_the_limits_are_reported(be):
    """2^30 positions for attn_weights, 2^18 for kv_evict: a table of one page over and over, which stays as it was"""
    import torch

    import openasr_b200 as ob

    page, MP = 1 << 20, 1 << 11
    k = torch.zeros(1, 1, page, 64, dtype=torch.float16, device="cuda")
    v, w = torch.zeros_like(k), torch.full((1, 1, page), 5.0, device="cuda")
    table = torch.zeros(1, MP, dtype=torch.int32, device="cuda")
    out = torch.zeros(1, dtype=torch.int32, device="cuda")
    for past, n in (((1 << 30), 1), ((1 << 30) - 1, 2), ((1 << 31) - 130, 1)):
        be.attn_weights(torch.zeros(1, 1, n, 64, device="cuda"), k, table, cuda(np.array([past], np.int32)), None, 0.1, 0.0, w)
        with pytest.raises(ob.GgmlBackendError, match="out-of-range"):
            be.synchronize()
    for past in ((1 << 18) + 1, (1 << 31) - 129):
        be.kv_evict(w, table, cuda(np.array([past], np.int32)), cuda(np.array([7], np.int32)), 0, 0, k, v, 1, out)
        with pytest.raises(ob.GgmlBackendError, match="out-of-range"):
            be.synchronize()
        assert int(out[0]) == past
    assert (w == 5).all()


def test_the_longest_sequence_that_may_be_evicted(be):
    rng = np.random.default_rng(31)
    c = Cache(rng, 1, 0, 1, 64, 4096, [1 << 18], fill=None, spare=0)
    w = rng.integers(0, 1 << 16, (c.P, 1, 4096)).astype(np.float32)
    same_after(be, c, w, [100001], 3, 1000)


@pytest.mark.parametrize("S", [32, 33, 70])
def test_many_sequences_of_all_lengths(be, S):
    """their order by length is worked out by one warp up to 32 of them"""
    rng = np.random.default_rng(S)
    c = Cache(rng, S, 2, 2, 64, 16, rng.integers(0, 300, S))
    c.past[3] = c.past[4]
    q = rng.standard_normal((S, 4, 2, 64)).astype(np.float32)
    old = entries(rng, c)
    for s in range(S):
        for p in range(c.past[s], c.past[s] + 2):
            c.k[c.table[s, p // 16], :, p % 16] = rng.standard_normal((2, 64)).astype(np.float16)
    want, tol = added64(c, q, [2] * S, 0.125, 1.0, old)
    check(run_weights(be, c, q, None, 0.125, 1.0, old), want, tol)


# ---- more rows than fit into registers: groups of rows, scores kept or not ------------------------
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,N,H,HKV,D,page,past", [
    (1, 17, 2, 2, 128, 8, [3]),                 # one row more than the registers hold
    (2, 12, 6, 3, 64, 24, [200, 0]),            # 24 and fewer of 64 values
    (2, 25, 4, 4, 64, 16, [100, 300]),          # 25
    (1, 11, 8, 4, 128, 16, [611]),              # 22
    (3, 13, 16, 2, 128, 16, [901, 17, 333]),    # 104: two groups of 52
    (2, 61, 8, 1, 64, 16, [1700, 400]),         # 488: eight groups over the CTAs of a cluster
    (50, 10, 32, 4, 128, 64, [7 * s for s in range(50)]),  # 80, a CTA per head
    (7, 33, 15, 5, 128, 40, [257] * 7),         # 99
])
def test_many_rows(be, S, N, H, HKV, D, page, past, f16):
    rng = np.random.default_rng(S * 100 + N)
    c = Cache(rng, S, N, HKV, D, page, past)
    q = rng.standard_normal((S, H, N, D)).astype(np.float16 if f16 else np.float32)
    live = np.array([N if s % 3 == 0 else rng.integers(0, N + 1) for s in range(S)], np.int32)
    for s in range(S):
        for p in range(c.past[s] + live[s], c.past[s] + N):
            c.k[c.table[s, p // page], :, p % page] = np.nan
    old = entries(rng, c)
    want, tol = added64(c, q, live, 0.1, 0.75, old)
    got = run_weights(be, c, q, live, 0.1, 0.75, old, f16=f16)
    check(got, want, tol)
    np.testing.assert_array_equal(got, run_weights(be, c, q, live, 0.1, 0.75, old, f16=f16))


@pytest.mark.parametrize("N,H,D,past,decay", [(20, 4, 128, 30011, 1.0), (20, 4, 128, 83009, 0.5), (7, 4, 64, 83009, 0.0)])
def test_many_rows_of_a_long_cache(be, N, H, D, past, decay):
    """scores of a part of the positions kept; sums too many to keep"""
    rng = np.random.default_rng(past)
    c = Cache(rng, 1, N, 1, D, 128, [past], spare=0)
    q = rng.standard_normal((1, H, N, D)).astype(np.float32)
    old = entries(rng, c)
    want, tol = added64(c, q, [N], 0.1, decay, old)
    check(run_weights(be, c, q, None, 0.1, decay, old), want, tol)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("D,N,HKV", [(128, 20, 1), (64, 45, 1), (128, 36, 2)])
def test_what_is_not_finite_stays_with_its_row_of_many(be, bad, f16, D, N, HKV):
    rng = np.random.default_rng(D + N)
    c = Cache(rng, 2, N, HKV, D, 16, [300, 20])
    q = rng.standard_normal((2, 2, N, D)).astype(np.float16 if f16 else np.float32)
    row = N - 3
    q[0, 0, row, 7] = bad                                        # sees positions 0 .. 300 + row
    c.k[c.table[1, 5 // 16], :, 5 % 16, 3] = bad                 # with finite queries a score of +-inf, or NaN
    got = run_weights(be, c, q, None, 0.125, 0.0, entries(rng, c), f16=f16)
    at = lambda s, h, n: got[c.table[s, np.arange(n) // 16], h, np.arange(n) % 16]  # noqa: E731
    assert np.isnan(at(0, 0, 300 + N)[: 301 + row]).all() and np.isfinite(at(0, 0, 300 + N)[301 + row:]).all()
    if HKV == 2:
        assert np.isfinite(at(0, 1, 300 + N)).all()
    if math.isnan(bad):
        assert np.isnan(at(1, 0, 20 + N)).all()


def test_a_key_of_minus_inf_gets_nothing_from_many_rows(be):
    """nor do rows of padding, whose products with it are NaN, spoil it"""
    rng = np.random.default_rng(21)
    N, at = 18, 77
    c = Cache(rng, 1, N, 1, 128, 16, [500])
    q = rng.standard_normal((1, 1, N, 128)).astype(np.float16)
    q[..., 9] = np.abs(q[..., 9]) + 1
    key = c.k[c.table[0, at // 16], 0, at % 16]
    key[:] = 0
    old = entries(rng, c)
    _, tol = added64(c, q, [N], 0.1, 0.0, old)  # of the others, which gain less than 1 part in 2 without it
    key[9] = -65504                             # times 1 or more: e^-6550 of the row
    want, _ = added64(c, q, [N], 0.1, 0.0, old)
    key[9] = -np.inf
    got = run_weights(be, c, q, None, 0.1, 0.0, old, f16=True)
    assert got[c.table[0, at // 16], 0, at % 16] == 0
    p = np.delete(np.arange(500 + N), at)
    pg, off = c.table[0, p // 16], p % 16
    assert (np.abs(got[pg, 0, off] - want[pg, 0, off]) <= 2 * tol[pg, 0, off]).all()


def test_pages_out_of_range_are_reported_with_many_rows(be):
    import openasr_b200 as ob

    rng = np.random.default_rng(22)
    c = Cache(rng, 2, 20, 2, 128, 16, [140, 20])
    q, old = rng.standard_normal((2, 4, 20, 128)).astype(np.float32), entries(rng, c)
    want = run_weights(be, c, q, None, 0.1, 1.0, old)
    other = c.table[1, :2].copy()
    c.table[0, 3], c.table[0, 8] = c.P, -1
    with pytest.raises(ob.GgmlBackendError, match="out-of-range"):
        w = cuda(old)
        be.attn_weights(cuda(q), c.device()[0], cuda(c.table), cuda(c.past), None, 0.1, 1.0, w)
        be.synchronize()
    np.testing.assert_array_equal(w.cpu().numpy()[other].astype(np.float64), want[other])


@pytest.mark.parametrize("spoil", ["page", "low", "past", "more", "keep", "negative"])
def test_a_sequence_that_is_not_shortened_keeps_its_length(be, spoil):
    """n_past_out goes into the next captured call: a sequence whose rows stay has the length that it had"""
    import torch

    import openasr_b200 as ob

    rng = np.random.default_rng(25)
    c = Cache(rng, 3, 0, 2, 64, 16, [60, 33, 47], fill=None)
    w = rng.random((c.P, 2, 16)).astype(np.float32)
    table, past, keep = c.table.copy(), c.past.copy(), np.array([40, 20, 47], np.int32)
    if spoil == "page":
        table[0, 3] = c.P
    elif spoil == "low":
        table[0, 0] = -1
    elif spoil == "past":
        past[0] = -1
    elif spoil == "more":
        past[0] = 16 * c.MP + 1
    else:
        keep[0] = 11 if spoil == "keep" else -1
    k, v, wd = (*c.device(), cuda(w))
    out = torch.full((3,), -5, dtype=torch.int32, device="cuda")
    be.kv_evict(wd, cuda(table), cuda(past), cuda(keep), 4, 8, k, v, 1, out)
    with pytest.raises(ob.GgmlBackendError, match="out-of-range"):
        be.synchronize()
    assert out.tolist() == [int(past[0]), 20, 47]
    np.testing.assert_array_equal(k.cpu().numpy()[c.table[0]], c.k[c.table[0]])
    np.testing.assert_array_equal(wd.cpu().numpy()[c.table[0]], w[c.table[0]])
