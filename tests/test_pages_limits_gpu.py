"""The paged cache's operators at the ends of their ranges: calls of very many steps, long chains, mixed
types, lengths near 2^31.  Tolerances as in test_pages_gpu.py; where a sum has very many terms, n
additions in 32 bits add 8 sqrt(n) 2^-24 of it (roundings are as often up as down)."""
import math

import numpy as np
import pytest

from test_pages_gpu import Cache, attend64, be, check, cuda, run_attn, words_of  # noqa: F401

pytestmark = pytest.mark.gpu


def attend_pool(pool_k, pool_v, q, counts, scale):
    """Rows q [N, H, D] over one K/V head's pool rows [R, D], row r seen counts[N, R] times -> [N, H, D]
    in 64 bits, and the largest sum |q| |k| of a visible position."""
    import torch

    k, v, q = pool_k.double(), pool_v.double(), q.double()
    x = torch.einsum("nhd,rd->nhr", q, k) * scale
    seen = (counts > 0)[:, None]
    w = torch.exp(x - x.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)) * counts[:, None]
    o = torch.einsum("nhr,rd->nhd", w, v) / w.sum(-1, keepdim=True)
    return o, torch.einsum("nhd,rd->nhr", q.abs(), k.abs()).max()


def repeated_pages(seed, page, pages, D, past, N):
    """One sequence over a pool of few pages (reads may share them) -> K, V, its table row, and how
    often node i sees each of the pool's rows"""
    import torch

    g = torch.Generator("cuda")
    g.manual_seed(seed)
    k, v = (torch.randn(pages, 1, page, D, generator=g, device="cuda").half() for _ in range(2))
    MP = -(-(past + N) // page)
    order = torch.arange(MP, device="cuda") * 7 % pages
    p = torch.arange(past + N, device="cuda")
    row = order[p // page] * page + p % page
    base = torch.bincount(row[:past], minlength=pages * page)
    own = torch.nn.functional.one_hot(row[past:], pages * page).cumsum(0)
    return k, v, order.int()[None], (base[None] + own).double()


@pytest.mark.parametrize("past,N,H,D,page,f16", [
    (1000000, 4968, 32, 64, 64, True),   # 1242 tiles of 128 rows, 7822 steps each: 66000 steps to a CTA
    (0, 1500, 3, 128, 16, False),        # a chain longer than a tree may be
    (70, 1100, 1, 64, 40, False),
])
def test_long_chains(be, past, N, H, D, page, f16):  # noqa: F811
    import torch

    k, v, table, counts = repeated_pages(N, page, 15, D, past, N)
    g = torch.Generator("cuda")
    g.manual_seed(N + 1)
    dt = torch.float16 if f16 else torch.float32
    q = torch.randn(1, N, H, D, generator=g, device="cuda").to(dt)
    out = torch.full((1, N, H, D), 7.0, dtype=dt, device="cuda")
    scale = 1 / math.sqrt(D)
    be.flash_attn_tree(q.permute(0, 2, 1, 3), k, v, table, cuda(np.array([past], np.int32)), None, None, scale, out)
    be.synchronize()
    units = -(-(past + N) // 128)
    for n0 in range(0, N, 512):
        want, big = attend_pool(k[:, 0].reshape(-1, D), v[:, 0].reshape(-1, D), q[0, n0:n0 + 512], counts[n0:n0 + 512], scale)
        ds = 2.0**-20 * scale * float(big)
        tol = (2 * (2 * ds + 2.0**-20) + 8 * math.sqrt(128 * units) * 2.0**-24) * float(v.abs().max())
        check(out[0, n0:n0 + 512].double().cpu().numpy(), want.cpu().numpy(), tol, f16)


# ---- what tree_commit writes must not be what it reads ------------------------------------------
def commit_args(S=3, N=5):
    import torch

    i32 = dict(dtype=torch.int32, device="cuda")
    pages = [torch.zeros(4 * S, 2, 8, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    table = torch.arange(2 * S, **i32).view(S, 2)
    parents = torch.arange(-1, N - 1, **i32).repeat(S, 1)
    return dict(tokens=torch.zeros(S, N, **i32), parents=parents, target=torch.zeros(S, N, **i32), n_nodes=torch.full((S,), N, **i32),
                n_past=torch.arange(S, **i32), table=table, k=pages[0], v=pages[1], layers=1, path=torch.zeros(S, N, **i32),
                n_accept=torch.zeros(S, **i32), next=torch.zeros(S, **i32), past_out=torch.zeros(S, **i32))


def test_tree_commit_refuses_results_over_its_inputs(be):  # noqa: F811
    import torch

    import openasr_b200 as ob

    ok = commit_args()
    be.tree_commit(*ok.values())
    be.synchronize()
    wide = torch.zeros(3, 12, dtype=torch.int32, device="cuda")
    for kw in (*(dict(path=ok[x]) for x in ("tokens", "parents", "target")), dict(n_accept=ok["n_nodes"]), dict(n_accept=ok["n_past"]),
               dict(next=ok["n_past"]), dict(next=ok["n_nodes"]), dict(past_out=ok["n_past"]), dict(past_out=ok["n_nodes"]),
               dict(n_accept=ok["parents"].view(-1)[6:9]), dict(next=ok["table"].view(-1)[3:6]),       # a part of one
               dict(tokens=wide[:, 1:6], path=wide[:, 5:10]), dict(next=ok["n_accept"]), dict(past_out=ok["next"]),
               dict(n_accept=ok["path"].view(-1)[12:15]), dict(path=torch.zeros(1, 5, dtype=torch.int32, device="cuda").expand(3, 5))):
        with pytest.raises(ob.backend.UnsupportedInputs, match="overlap"):
            be.tree_commit(*{**ok, **kw}.values())
            be.synchronize()


def test_tree_commit_takes_rows_side_by_side_in_one_buffer(be):  # noqa: F811
    """inputs may be one tensor, and results may lie between them, as long as no value is both"""
    import torch

    a = commit_args()
    want = {**a, **{x: a[x].clone() for x in ("path", "n_accept", "next", "past_out")}}
    be.tree_commit(*want.values())
    all_ = torch.zeros(3, 10, dtype=torch.int32, device="cuda")
    vec = torch.zeros(12, dtype=torch.int32, device="cuda")
    vec[:3] = a["n_past"]
    got = {**a, "tokens": all_[:, :5], "target": all_[:, :5], "path": all_[:, 5:], "n_past": vec[:3], "n_accept": vec[3:6],
           "next": vec[6:9], "past_out": vec[9:]}
    be.tree_commit(*got.values())
    be.synchronize()
    for x in ("path", "n_accept", "next", "past_out"):
        assert torch.equal(got[x], want[x])
    assert want["n_accept"].tolist() == [5] * 3


def test_an_allocation_that_failed_is_reported_once():
    """the call after it is not refused for the same error"""
    import torch

    import openasr_b200 as ob
    from openasr_b200 import backend as bk

    b = ob.Backend(0)
    try:
        b.set_stream(torch.cuda.current_stream())
        with pytest.raises(bk.AllocFailed):
            b.reserve_scratch(1 << 50)
        c = Cache(np.random.default_rng(1), 1, 2, 1, 64, 8, [20])
        q = np.random.default_rng(2).standard_normal((1, 2, 2, 64)).astype(np.float32)
        sees = np.tril(np.ones((1, 2, 2), bool))
        want, tol = attend64(c, q, [2], sees, 0.1)
        check(run_attn(b, c, q, None, None, 0.1), want, tol, False)
    finally:
        b.close()


def test_positions_up_to_2_31(be):  # noqa: F811
    """Two pages of 2^20 positions, repeated 4096 times: the longest cache that 32-bit positions allow is
    read whole, one position more is reported by every operator."""
    import torch

    import openasr_b200 as ob

    D, page, MP, T = 64, 1 << 20, 4096, (1 << 31) - 129
    g = torch.Generator("cuda")
    g.manual_seed(7)
    k = torch.randn(2, 1, page, D, generator=g, device="cuda").half()
    # the first half of the cache has values about 1, the second about 3
    v = (torch.randn(2, 1, page, D, generator=g, device="cuda") / 4 + torch.tensor([1.0, 3.0], device="cuda").view(2, 1, 1, 1)).half()
    table = (torch.arange(MP, device="cuda") >= MP // 4).int()[None]
    q = torch.randn(1, 1, 2, D, generator=g, device="cuda")
    out = torch.full((1, 1, 2, D), 7.0, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    be.flash_attn_tree(q.permute(0, 2, 1, 3), k, v, table, torch.tensor([T - 1], **i32), None, None, 0.125, out)
    be.synchronize()
    p = page * torch.tensor([MP // 4, MP // 4], dtype=torch.int64)  # positions 0 .. T - 1: the last page lacks 129
    counts = torch.full((1, 2 * page), MP // 4, dtype=torch.float64, device="cuda")
    counts[0, -129:] -= 1
    assert int(counts.sum()) == T and int(p.sum()) == T + 129
    want, big = attend_pool(k[:, 0].reshape(-1, D), v[:, 0].reshape(-1, D), q[0], counts, 0.125)
    # per sum: 2^24 units in 296 CTAs one after the other, then the 296 parts
    ds = 2.0**-20 * 0.125 * float(big)
    tol = (2 * (2 * ds + 2.0**-20) + 8 * math.sqrt(2.0**24 / 296 + 296) * 2.0**-24) * float(v.abs().max())
    check(out[0].double().cpu().numpy(), want.cpu().numpy(), tol, False)

    x = torch.randn(1, 2, 4, D, generator=g, device="cuda")
    z2, z1 = torch.zeros(1, 2, **i32), [torch.zeros(1, **i32) for _ in range(4)]
    before = k.clone()
    for past, n in ((T - 1, 2), (2**31 - 1, 1), (2**31 - 2, 2)):
        lens = torch.tensor([past], **i32), torch.tensor([n], **i32)
        o2 = torch.zeros(1, 2, 2, D, device="cuda")
        for call in (lambda: be.flash_attn_tree(x[:, :, :2].permute(0, 2, 1, 3), k, v, table, *lens, None, 0.125, o2),
                     lambda: be.qk_norm_rope(x, None, None, 0.0, None, None, table, *lens, o2, k, v),
                     lambda: be.tree_commit(z2, z2 - 1, z2, lens[1], lens[0], table, k, v, 1, z2.clone(), z1[0], z1[1], z1[2])):
            with pytest.raises(ob.backend.ExecutionFailed):
                call()
                be.synchronize()
    assert torch.equal(before, k)


@pytest.mark.parametrize("N,H,HKV,D", [(1, 4, 2, 128), (7, 6, 6, 64), (20, 8, 2, 128), (61, 4, 2, 128), (150, 2, 1, 64)])
@pytest.mark.parametrize("q16,o16", [(False, True), (True, False)])
def test_queries_and_outputs_of_different_types(be, N, H, HKV, D, q16, o16):  # noqa: F811
    import torch

    rng = np.random.default_rng(N + D)
    c = Cache(rng, 2, N, HKV, D, 16, [130, 9])
    q = rng.standard_normal((2, H, N, D)).astype(np.float16 if q16 else np.float32)
    sees = np.broadcast_to(np.tril(np.ones((N, N), bool)), (2, N, N))
    live = np.array([N, max(1, N // 2)], np.int32)
    want, tol = attend64(c, q, live, sees, 0.09)
    k, v = c.device()
    out = torch.full((2, N, H, D), 7.0, dtype=torch.float16 if o16 else torch.float32, device="cuda")
    be.flash_attn_tree(cuda(q), k, v, cuda(c.table), cuda(c.past), cuda(live), None, 0.09, out)
    be.synchronize()
    check(out.cpu().double().numpy(), want, tol, o16)


@pytest.mark.parametrize("N", [3, 14, 30, 80])
@pytest.mark.parametrize("f16", [False, True])
def test_a_key_whose_score_is_minus_infinity(be, N, f16):  # noqa: F811
    """f16 queries: the position has no weight; f32 ones: that, or the row is NaN"""
    rng = np.random.default_rng(N)
    c = Cache(rng, 1, N, 2, 128, 16, [150])
    q = rng.standard_normal((1, 4, N, 128)).astype(np.float16 if f16 else np.float32)
    q[..., 5] = -np.abs(q[..., 5]) - np.float16(0.5)
    c.k[c.table[0, 1], :, 4, 5] = np.inf  # position 20
    sees = np.tril(np.ones((1, N, N), bool))
    without = Cache(rng, 1, N, 2, 128, 16, [149])
    for name in ("k", "v"):
        rows = np.delete(c.rows(getattr(c, name), 0, 150 + N), 20, axis=1)
        at = np.arange(149 + N)
        getattr(without, name)[without.table[0, at // 16], :, at % 16] = rows.transpose(1, 0, 2)
    want, tol = attend64(without, q, [N], sees, 0.1)
    got = run_attn(be, c, q, None, None, 0.1, f16)
    if not f16:
        assert np.isnan(got).all(-1)[np.isnan(got).any(-1)].all()
        got = np.where(np.isnan(got), want, got)
    check(got, want, tol, f16)


def test_calls_of_too_many_steps_are_refused(be):  # noqa: F811
    """rows and positions that 31 bits do not count (views of little memory: nothing is read)"""
    import torch

    import openasr_b200 as ob

    k, v = (torch.zeros(1, 1, 4096, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    past = torch.zeros(1, dtype=torch.int32, device="cuda")
    row = torch.zeros(1, 1, 1, 64, device="cuda")
    table = torch.zeros(1, 1 << 22, dtype=torch.int32, device="cuda")
    for S, N, H, MP in ((1, 1 << 24, 128, 1), (1, 1 << 24, 1, 1 << 18), (1, 1 << 17, 1, 1 << 22), (128, (1 << 24) - 1, 1, 1)):
        with pytest.raises(ob.backend.UnsupportedInputs, match="too many"):
            be.flash_attn_tree(row.expand(S, H, N, 64), k, v, table[:, :MP].expand(S, MP), past.repeat(S), None, None, 0.1,
                               row.expand(S, N, H, 64))


def test_addresses_that_are_not_aligned_are_refused(be):  # noqa: F811
    """descriptors whose 4-byte values lie two bytes off (a tensor of torch cannot); nothing is launched"""
    import torch

    import openasr_b200 as ob

    def off(t):
        d = ob.describe(t)
        d.data += 2
        return d

    a = commit_args()
    S, N, H, D = 3, 5, 4, 64
    f32 = dict(device="cuda")
    x, q = torch.zeros(S, N, H + 4, D, **f32), torch.zeros(S, N, H, D, **f32)
    gain, tree = torch.ones(D, **f32), torch.zeros(S, N, 1, dtype=torch.int32, device="cuda")
    pairs = torch.full((2, 2), -1, dtype=torch.int32, device="cuda")
    norm = dict(x=x, wq=gain, wk=gain, eps=1e-6, rope=None, pos=a["tokens"], table=a["table"], past=a["n_past"], nodes=a["n_nodes"],
                q=q, k=a["k"], v=a["v"])
    attn = dict(q=q.permute(0, 2, 1, 3), k=a["k"], v=a["v"], table=a["table"], past=a["n_past"], nodes=a["n_nodes"], tree=tree,
                scale=0.1, out=q.clone())
    for call, args, names in ((be.tree_commit, a, ("tokens", "parents", "target", "n_nodes", "n_past", "table", "path", "n_accept",
                                                   "next", "past_out")),
                              (be.qk_norm_rope, norm, ("wq", "wk", "pos", "table", "past", "nodes")),
                              (be.flash_attn_tree, attn, ("table", "past", "nodes", "tree"))):
        call(*args.values())
        for name in names:
            with pytest.raises(ob.backend.UnsupportedInputs):
                call(*{**args, name: off(args[name])}.values())
    with pytest.raises(ob.backend.UnsupportedInputs):
        be.kv_pages_copy(a["k"], a["v"], 1, off(pairs))
    be.synchronize()
