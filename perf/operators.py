"""The operators of speculative decoding over a paged K/V cache: what is measured of them.

One decoding step of a drafted tree runs, in every layer, `qk_norm_rope` (norms and
rotation of the projected heads, K/V rows into the sequence's pages) and
`flash_attn_tree` (the drafted nodes attend to the committed positions and to their own
ancestors); then `tree_commit` accepts the longest path that the model agrees with and
compacts its rows in every layer.  `kv_pages_copy` copies the pages that a forked
sequence is about to write.

Layouts (torch shapes; S sequences, N nodes at most, L layers, P pages of `page` positions):
  pages       f16 (P, HKV, page, D), or (L * P, HKV, page, D) for all layers
  page_table  i32 (S, MP): page of positions [j * page, (j + 1) * page)
  n_past      i32 (S,): committed positions; node i of sequence s is at position n_past[s] + i
  n_nodes     i32 (S,): live nodes (the others are padding: zeros come out)
  tree        i32 (S, N, W): bit j of node i's words: node i sees node j
"""
import math

import numpy as np
import torch

own = False

VOCAB = 151936
EPS = 1e-6
THETA = 1e6


# ---- cases ------------------------------------------------------------------------------
def listed():
    """Head layouts: 16 / 8 heads of 128 (28 layers) and 20 heads of 64 are the two decoders
    of this repository, 32 / 4 of 128 a generic wider grouping."""
    return [
        # one token of one sequence after a 390-frame prompt: the latency of a single call
        dict(name="attn 1 token", op="attn", S=1, N=1, H=16, HKV=8, D=128, page=64, lo=390, hi=390, chain=True, half=False),
        # a batch of eight ragged sequences, 16-node trees, small pages: the usual step
        dict(name="attn 8 trees of 16", op="attn", S=8, N=16, H=16, HKV=8, D=128, page=16, lo=390, hi=1990, chain=False, half=False),
        # the other decoder's heads (no grouping, width 64), short caches, a drafted chain of 7
        dict(name="attn 8 chains of 7, D 64", op="attn", S=8, N=7, H=20, HKV=20, D=64, page=24, lo=4, hi=441, chain=True, half=False),
        # two long recordings, eight query heads to a K/V head, small trees, f16 in and out
        dict(name="attn 2 long", op="attn", S=2, N=5, H=32, HKV=4, D=128, page=64, lo=30011, hi=32003, chain=False, half=True),
        # a full server: long ragged caches, wide trees, f16 in and out
        dict(name="attn 16 wide trees", op="attn", S=16, N=61, H=16, HKV=8, D=128, page=128, lo=4001, hi=8190, chain=False, half=True),
        # one token for each of eight sequences: the plain decoding step
        dict(name="norm 8 tokens", op="norm", S=8, N=1, H=16, HKV=8, D=128, page=64, lo=390, hi=1990, chain=True, half=False),
        # eight 61-node trees, the other head width
        dict(name="norm 8 trees of 61, D 64", op="norm", S=8, N=61, H=20, HKV=20, D=64, page=16, lo=4, hi=380, chain=False, half=False),
        # a prompt chunk of 512 rows for each of eight sequences
        dict(name="norm 8 prompts of 512", op="norm", S=8, N=512, H=16, HKV=8, D=128, page=64, lo=0, hi=1000, chain=True, half=True),
        # acceptance of the usual step, 28 layers
        dict(name="commit 8 trees of 16", op="commit", S=8, N=16, HKV=8, D=128, L=28, page=16, lo=390, hi=1990, accept=4),
        # acceptance of the full server's step
        dict(name="commit 32 trees of 61", op="commit", S=32, N=61, HKV=8, D=128, L=28, page=64, lo=40, hi=300, accept=13),
        # eight sequences forked: the part-filled last page of each, small pages
        dict(name="copy 8 pages of 16", op="copy", n=8, HKV=8, D=128, L=28, page=16),
        # a beam's worth of forks with large pages
        dict(name="copy 64 pages of 64", op="copy", n=64, HKV=8, D=128, L=28, page=64),
    ]


def draw(rng):
    def span(lo, hi):  # spread over the logarithm, ends included
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)) - 0.001)))))

    op = rng.choice(["attn", "attn", "attn", "norm", "commit", "copy"])
    H, HKV, D = rng.choice([(16, 8, 128), (16, 8, 128), (20, 20, 64), (32, 4, 128), (6, 6, 64), (12, 2, 64), (8, 1, 128), (15, 5, 128)])
    page = rng.choice([8, 16, 16, 24, 32, 40, 64, 64, 128, 256])
    if op == "attn":
        S, N = span(1, 32), span(1, 64)
        most = min(32003, 16 * 6000 * 8 * 128 // (S * HKV * D))  # no more cache than the largest listed case
        most = min(most, 16 * 6000 * 61 * 16 * 128 // (S * N * H * D))
        hi = span(1, max(1, most))
        return dict(op=op, S=S, N=N, H=H, HKV=HKV, D=D, page=page, lo=rng.choice([hi, hi // 2, hi // 7, 0]), hi=hi,
                    chain=rng.random() < 0.4, half=rng.random() < 0.5)
    if op == "norm":
        S = span(1, 16)
        N = span(1, 4096 // S)
        hi = span(1, 2000)
        return dict(op=op, S=S, N=N, H=H, HKV=HKV, D=D, page=page, lo=rng.choice([hi, hi // 3, 0]), hi=hi,
                    chain=N > 256 or rng.random() < 0.5, half=rng.random() < 0.5)
    if op == "commit":
        S, N, L = span(1, 32), span(1, 61), rng.choice([4, 12, 28, 32])
        while S * L * HKV * D > 32 * 28 * 8 * 128:
            S -= 1
        hi = span(1, 300)
        return dict(op=op, S=S, N=N, HKV=HKV, D=D, L=L, page=page, lo=rng.choice([hi, hi // 3, 0]), hi=hi, accept=span(1, min(N, 13)))
    L = rng.choice([4, 12, 28, 32])
    n = span(1, max(1, 64 * 28 * 8 * 128 * 64 // (L * HKV * D * page)))
    return dict(op=op, n=n, HKV=HKV, D=D, L=L, page=page)


# ---- what a case fixes: lengths (the seed makes values, trees and page orders) ----------
def pasts(c):
    """Committed positions per sequence: spread evenly over [lo, hi], shuffled by a stride."""
    S = c["S"]
    return [c["hi"] - (c["hi"] - c["lo"]) * ((s * 5) % S) // max(1, S - 1) if S > 1 else c["hi"] for s in range(S)]


def nodes(c):
    """Live nodes per sequence: every third sequence drafts about three quarters of the width."""
    return [c["N"] if s % 3 != 2 or c["op"] == "commit" else max(1, c["N"] * 3 // 4) for s in range(c["S"])]


def pages_per_seq(c):
    return -(-(c["hi"] + c["N"]) // c["page"])


def work(case):
    c = case
    if c["op"] == "copy":
        return {"bytes": 2 * c["n"] * c["L"] * 2 * c["HKV"] * c["page"] * c["D"] * 2, "flops": 0}
    S, N = c["S"], c["N"]
    if c["op"] == "commit":
        # accepted rows but the root, which is in place, read and written in each layer, K and V
        rows = S * (c["accept"] - 1)
        return {"bytes": 2 * rows * c["L"] * 2 * c["HKV"] * c["D"] * 2 + S * (N * 16 + 16), "flops": 0}
    n = nodes(c)
    if c["op"] == "norm":
        row = (c["H"] + 2 * c["HKV"]) * c["D"]
        out = c["H"] * c["D"] * (2 if c["half"] else 4)
        return {"bytes": sum(n) * (row * 4 + 2 * c["HKV"] * c["D"] * 2 + c["D"] * 4) + S * N * out, "flops": sum(n) * row * 8}
    keys = [p + m for p, m in zip(pasts(c), n)]
    el = 2 if c["half"] else 4
    b = sum(keys) * c["HKV"] * c["D"] * 4 + 2 * S * N * c["H"] * c["D"] * el + (0 if c["chain"] else S * N * ((N + 31) // 32) * 4)
    return {"bytes": b, "flops": 4 * c["H"] * c["D"] * sum(k * m for k, m in zip(keys, n))}


# ---- inputs -------------------------------------------------------------------------------
def random_trees(r, S, N):
    """Parents of random draft trees: node 0 is the root, a node's parent comes before it."""
    par = np.full((S, N), -1, np.int32)
    for i in range(1, N):
        par[:, i] = np.where(r.rand(S) < 0.6, i - 1, (r.rand(S) * i).astype(np.int32))
    return par


def ancestors(par):
    """bool (S, N, N): node i sees itself and its ancestors."""
    S, N = par.shape
    see = np.zeros((S, N, N), bool)
    for i in range(N):
        up = par[:, i]
        see[:, i] = np.where((up >= 0)[:, None], see[np.arange(S), np.maximum(up, 0)], False)
        see[:, i, i] = True
    return see


def as_words(see):
    S, N, _ = see.shape
    W = (N + 31) // 32
    bits = np.zeros((S, N, W * 32), np.uint64)
    bits[:, :, :N] = see
    w = (bits.reshape(S, N, W, 32) << np.arange(32, dtype=np.uint64)).sum(-1)
    return w.astype(np.uint32).view(np.int32)


def rope_table(n_pos, D):
    """(cos, sin) of position p times theta^(-2 i / D), in f32."""
    f = THETA ** (-2.0 * np.arange(D // 2) / D)
    a = np.arange(n_pos)[:, None] * f[None]
    return torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).cuda()


def prepare(case, seed):
    c = case
    r = np.random.RandomState(seed % (1 << 32))
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()

    HKV, D, page = c["HKV"], c["D"], c["page"]
    st = dict(c)
    if c["op"] == "copy":
        n, L = c["n"], c["L"]
        P = 2 * n + 3
        st["P"] = P
        st["k"], st["v"] = (normal(L * P, HKV, page, D, dtype=torch.float16) for _ in range(2))
        order = r.permutation(P)
        # a page may be forked more than once; every copy goes to a page of its own
        st["pairs"] = ints(np.stack([order[:n][r.randint(0, n, n)], order[n:2 * n]], 1))
        return st
    S, N = c["S"], c["N"]
    MP = pages_per_seq(c)
    P = S * MP + 2
    L = c.get("L", 1)
    st["P"] = P
    st["k"], st["v"] = (normal(L * P, HKV, page, D, dtype=torch.float16) for _ in range(2))
    st["page_table"] = ints(r.permutation(P)[: S * MP].reshape(S, MP))
    past, live = np.array(pasts(c)), np.array(nodes(c))
    st["n_past"], st["n_nodes"] = ints(past), ints(live)
    if c["op"] == "commit":
        A = c["accept"]
        par = random_trees(r, S, N)
        tok = np.stack([r.choice(VOCAB, N, replace=False) for _ in range(S)]).astype(np.int32)
        tgt = r.randint(0, VOCAB, (S, N)).astype(np.int32)
        for s in range(S):
            path = [0] + sorted(r.choice(np.arange(1, N), A - 1, replace=False).tolist()) if A > 1 else [0]
            for a, b in zip(path, path[1:]):
                par[s, b] = a
                tgt[s, a] = tok[s, b]
                for j in range(b + 1, N):  # a sibling drafted twice: the first of the two counts
                    if j not in path and r.rand() < 0.05:
                        par[s, j], tok[s, j] = a, tok[s, b]
            end = path[-1]
            while np.any((par[s] == end) & (tok[s] == tgt[s, end])):
                tgt[s, end] = r.randint(0, VOCAB)
        st["tokens"], st["parents"], st["target"] = ints(tok), ints(par), ints(tgt)
        st["sees"] = torch.from_numpy(ancestors(par)).cuda()
        st["path"], st["n_accept"] = ints(np.zeros((S, N))), ints(np.zeros(S))
        st["next"], st["n_past_out"] = ints(np.zeros(S)), ints(np.zeros(S))
        return st
    H = c["H"]
    dt = torch.float16 if c["half"] else torch.float32
    par = random_trees(r, S, N)
    if c["chain"]:
        par = np.broadcast_to(np.arange(-1, N - 1, dtype=np.int32), (S, N)).copy()
    st["out"] = torch.empty(S, N, H, D, device="cuda", dtype=dt)
    if c["op"] == "norm":
        depth = np.zeros((S, N), np.int64)
        for i in range(1, N):
            depth[:, i] = depth[np.arange(S), par[:, i]] + 1
        st["pos"] = None if c["chain"] else ints(past[:, None] + depth)
        st["rope"] = rope_table(c["hi"] + N, D)
        st["qkv"] = normal(S, N, H + 2 * HKV, D) * 1.7
        st["q_norm"], st["k_norm"] = (1 + 0.1 * normal(D) for _ in range(2))
        return st
    # normed queries and keys: entries about 1, scores of a few units
    st["q"] = normal(S, N, H, D).to(dt).permute(0, 2, 1, 3)
    st["tree"] = None if c["chain"] else ints(as_words(ancestors(par)))
    st["scale"] = 1.0 / math.sqrt(D)
    return st


# ---- one pass --------------------------------------------------------------------------------
_be = None


def backend():
    """The backend handle that a program makes once."""
    global _be
    if _be is None:
        import openasr_b200 as ob

        _be = ob.Backend(0)
        _be.set_stream(torch.cuda.current_stream())
    return _be


def run(st):
    if not own:
        return {"attn": plain_attn, "norm": plain_norm, "commit": plain_commit, "copy": plain_copy}[st["op"]](st)
    be = backend()
    if st["op"] == "attn":
        be.flash_attn_tree(st["q"], st["k"], st["v"], st["page_table"], st["n_past"], st["n_nodes"], st["tree"], st["scale"], st["out"])
        return st["out"]
    if st["op"] == "norm":
        be.qk_norm_rope(st["qkv"], st["q_norm"], st["k_norm"], EPS, st["rope"], st["pos"], st["page_table"], st["n_past"], st["n_nodes"],
                        st["out"], st["k"], st["v"])
        return [st["out"], st["k"], st["v"]]
    if st["op"] == "commit":
        be.tree_commit(st["tokens"], st["parents"], st["target"], st["n_nodes"], st["n_past"], st["page_table"], st["k"], st["v"], st["L"],
                       st["path"], st["n_accept"], st["next"], st["n_past_out"])
        return [st["path"], st["n_accept"], st["next"], st["n_past_out"], st["k"], st["v"]]
    be.kv_pages_copy(st["k"], st["v"], st["L"], st["pairs"])
    return [st["k"], st["v"]]


def plain_attn(st):
    S, N, H, HKV, D, page = (st[x] for x in ("S", "N", "H", "HKV", "D", "page"))
    dev = st["q"].device
    pt = st["page_table"].long()
    k, v = (st[x][pt].permute(0, 2, 1, 3, 4).reshape(S, HKV, -1, D).float() for x in ("k", "v"))
    T = k.shape[2]
    node = torch.arange(T, device=dev)[None] - st["n_past"][:, None]  # (S, T): which node the position holds, < 0: committed
    live = node < st["n_nodes"][:, None]
    i = torch.arange(N, device=dev)
    if st["tree"] is None:
        sees = node[:, None] <= i[None, :, None]
    else:
        bits = ((st["tree"][..., None] >> torch.arange(32, device=dev)) & 1).bool().reshape(S, N, -1)
        at = node.clamp(0, N - 1)[:, None].expand(S, N, T)
        sees = (node < 0)[:, None] | bits.gather(2, at)
    sees = sees & live[:, None] & (i[None] < st["n_nodes"][:, None])[..., None]  # (S, N, T)
    q = st["q"].float().reshape(S, HKV, H // HKV, N, D).reshape(S, HKV, -1, D)
    s = torch.matmul(q, k.transpose(2, 3)) * st["scale"]  # (S, HKV, G * N, T)
    s = s.reshape(S, H, N, T).masked_fill(~sees[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / l, torch.zeros_like(p))
    v = torch.where(live[:, None, :, None], v, torch.zeros_like(v))
    o = torch.matmul(p.reshape(S, HKV, -1, T), v).reshape(S, H, N, D)
    return o.permute(0, 2, 1, 3).contiguous().to(st["out"].dtype)


def plain_norm(st):
    S, N, H, HKV, D, page = (st[x] for x in ("S", "N", "H", "HKV", "D", "page"))
    x = st["qkv"]
    i = torch.arange(N, device=x.device)
    live = i[None] < st["n_nodes"][:, None]
    at = (st["n_past"][:, None] + i[None]).long()
    rot = st["rope"][at if st["pos"] is None else st["pos"].long()]  # (S, N, D / 2, 2)
    cos, sin = rot[:, :, None, :, 0], rot[:, :, None, :, 1]

    def turn(y, w):
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS) * w
        a, b = y[..., : D // 2], y[..., D // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    q = turn(x[:, :, :H], st["q_norm"])
    k = turn(x[:, :, H:H + HKV], st["k_norm"])
    q = torch.where(live[:, :, None, None], q, torch.zeros_like(q)).to(st["out"].dtype)
    pg, off = st["page_table"].long().gather(1, at // page), at % page
    for pages, rows in ((st["k"], k), (st["v"], x[:, :, H + HKV:])):
        pages[pg, :, off] = torch.where(live[:, :, None, None], rows.half(), pages[pg, :, off])
    return [q, st["k"], st["v"]]


def plain_commit(st):
    S, N, L, P, HKV, D, page = (st[x] for x in ("S", "N", "L", "P", "HKV", "D", "page"))
    tok, par, tgt = st["tokens"], st["parents"].long(), st["target"]
    i = torch.arange(N, device=tok.device)
    live = i[None] < st["n_nodes"][:, None]
    up = par.clamp(min=0)
    agrees = live & (par >= 0) & (par < i) & (tok == tgt.gather(1, up))
    # the first child that agrees, by parent
    first = torch.full((S, N), N, device=tok.device).scatter_reduce(1, up, torch.where(agrees, i.expand(S, N), N), "amin")
    chosen = agrees & (first.gather(1, up) == i)
    chosen[:, 0] = live[:, 0]
    on = live & ~(st["sees"] & ~chosen[:, None]).any(-1)  # itself and all ancestors chosen
    count = on.sum(1)
    path = torch.where(on, i, N).sort(1).values
    keep = i[None] < count[:, None]
    last = path.gather(1, (count - 1).clamp(min=0)[:, None])
    nxt = torch.where(count > 0, tgt.gather(1, last.clamp(max=N - 1))[:, 0], torch.full_like(tgt[:, 0], -1))
    path = torch.where(keep, path, torch.full_like(path, -1))
    pt, past = st["page_table"].long(), st["n_past"].long()[:, None]
    src, dst = past + path.clamp(min=0), past + i[None]
    for pages in (st["k"], st["v"]):
        x = pages.view(L, P, HKV, page, D)
        moved = x[:, pt.gather(1, src // page), :, src % page]  # (S, N, L, HKV, D)
        to = (slice(None), pt.gather(1, dst // page), slice(None), dst % page)
        x[to] = torch.where(keep[:, :, None, None, None], moved, x[to])
    out = [path.int(), count.int(), nxt.int(), (st["n_past"] + count).int()]
    return out + [st["k"], st["v"]]


def plain_copy(st):
    L, P = st["L"], st["P"]
    src, dst = st["pairs"][:, 0].long(), st["pairs"][:, 1].long()
    for pages in (st["k"], st["v"]):
        x = pages.view(L, P, *pages.shape[1:])
        x[:, dst] = x[:, src]
    return [st["k"], st["v"]]


# ---- 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    st = prepare(c, seed)
    if c["op"] == "copy":
        pairs = st["pairs"].cpu().numpy()
        out = []
        for pages in (st["k"], st["v"]):
            x = pages.double().view(c["L"], st["P"], -1)
            for a, b in pairs:
                x[:, b].copy_(x[:, a])
            out.append(x.view(pages.shape))
        return out
    S, N, HKV, D, page = (c[x] for x in ("S", "N", "HKV", "D", "page"))
    past, live = pasts(c), nodes(c)
    table = st["page_table"].cpu().numpy()

    def row(s, p):  # (page, offset) of position p
        return int(table[s, p // page]), p % page

    if c["op"] == "commit":
        L, P = c["L"], st["P"]
        tok, par, tgt = (st[x].cpu().numpy() for x in ("tokens", "parents", "target"))
        path = np.full((S, N), -1, np.int32)
        count, nxt = np.zeros(S, np.int32), np.zeros(S, np.int32)
        k, v = (st[x].double().view(L, P, HKV, page, D) for x in ("k", "v"))
        for s in range(S):
            walk = [0]
            while True:
                kids = [j for j in range(walk[-1] + 1, N) if par[s, j] == walk[-1] and tok[s, j] == tgt[s, walk[-1]]]
                if not kids:
                    break
                walk.append(kids[0])
            path[s, : len(walk)], count[s], nxt[s] = walk, len(walk), tgt[s, walk[-1]]
            for j, node in enumerate(walk):
                (pa, a), (pb, b) = row(s, past[s] + node), row(s, past[s] + j)
                for x in (k, v):
                    x[:, pb, :, b] = x[:, pa, :, a]
        ints = [torch.from_numpy(x).cuda() for x in (path, count, nxt, np.array(past, np.int32) + count)]
        return ints + [x.view(L * P, HKV, page, D) for x in (k, v)]
    H = c["H"]
    G = H // HKV
    if c["op"] == "norm":
        x = st["qkv"].double()
        q = torch.zeros(S, N, H, D, device="cuda", dtype=torch.float64)
        k, v = st["k"].double(), st["v"].double()
        half = D // 2
        for s in range(S):
            n = live[s]
            p = torch.arange(past[s], past[s] + n, device="cuda")
            ang = st["rope"].double()[p if st["pos"] is None else st["pos"][s, :n].long()]
            z = torch.complex(ang[..., 0], ang[..., 1])[:, None]  # (n, 1, D / 2)

            def normed(y, w):
                y = y / ((y * y).sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
                t = torch.complex(y[..., :half], y[..., half:]) * z
                return torch.cat([t.real, t.imag], -1)

            q[s, :n] = normed(x[s, :n, :H], st["q_norm"])
            pg, off = torch.from_numpy(table[s]).cuda().long()[p // page], p % page
            k[pg, :, off] = normed(x[s, :n, H:H + HKV], st["k_norm"])
            v[pg, :, off] = x[s, :n, H + HKV:]
        return [q, k, v]
    out = torch.zeros(S, N, H, D, device="cuda", dtype=torch.float64)
    tree = None if st["tree"] is None else st["tree"].cpu().numpy().view(np.uint32)
    for s in range(S):
        n, T = live[s], past[s] + live[s]
        see = np.ones((n, T), bool)
        for i in range(n):
            see[i, past[s]:] = [j <= i if tree is None else bool(tree[s, i, j // 32] >> np.uint32(j % 32) & np.uint32(1)) for j in range(n)]
        hide = ~torch.from_numpy(see).cuda()
        pg = torch.from_numpy(table[s]).cuda().long()
        for h in range(HKV):
            k, v = (st[x][pg, h].reshape(-1, D)[:T].double() for x in ("k", "v"))
            q = st["q"][s, h * G:(h + 1) * G, :n].double()  # (G, n, D)
            w = (q @ k.T * st["scale"]).masked_fill(hide, -math.inf)
            out[s, :n, h * G:(h + 1) * G] = (torch.softmax(w, -1) @ v).transpose(0, 1)
    return out
