"""Operators next to speculative decoding over a paged K/V cache: what is measured of them.

`tree_sample` draws the token after each node of a drafted tree from the target's
probabilities (at a temperature, from given uniform numbers), or, where the draft gives the
probabilities that it drew from, accepts drafted children by rejection; `tree_commit` then
follows the result.  `attn_weights` adds up the attention that the cached positions of a
sequence get; `kv_evict` keeps the positions with the most of it and moves their rows to the
front of the pages.

Layouts (torch shapes; S sequences, N nodes at most, V tokens, L layers, P pages of `page` positions):
  logits      f32 (S, N, V); draft_probs f32 (S, N, V): what the children of node i were drawn from
  uniforms    f32 (S, N, 2): a child's for its acceptance, a node's for the token after it
  target      i32 (S, N): the token after each node; logprob f32 (S, N): the log of its probability
  pages       f16 (P, HKV, page, D), or (L * P, HKV, page, D) for all layers
  weights     f32 (P, HKV, page), or (L * P, HKV, page)
  page_table  i32 (S, MP): page of positions [j * page, (j + 1) * page)
  n_past      i32 (S,): committed positions; node i of sequence s is at position n_past[s] + i
  n_nodes     i32 (S,): live nodes
"""
import math

import numpy as np
import torch

own = False


# ---- cases ------------------------------------------------------------------------------
def listed():
    """Vocabularies of 51866 and 151936 and the heads 16 / 8 of 128 (28 layers) and 20 of 64 are
    those of the two decoders of this repository, 32 / 4 of 128 a generic wider grouping."""
    return [
        # one utterance of the smaller vocabulary at a temperature: the latency of a call
        dict(name="sample 1 token", op="sample", S=1, N=1, V=51866, kids=0, greedy=False),
        # the plain step of eight sequences, one of them still greedy
        dict(name="sample 8 tokens", op="sample", S=8, N=1, V=151936, kids=0, greedy=True),
        # eight drafted chains with the draft model's probabilities: speculative sampling
        dict(name="verify 8 chains of 8", op="sample", S=8, N=8, V=151936, kids=1, greedy=False),
        # trees with siblings from the draft's distribution; rows of odd alignment
        dict(name="verify 4 trees of 31", op="sample", S=4, N=31, V=51866, kids=3, greedy=True),
        # a full server's trees from a draft without probabilities (an n-gram table)
        dict(name="sample 32 trees of 61", op="sample", S=32, N=61, V=151936, kids=0, greedy=True),
        # one token of one sequence after a 390-frame prompt: the latency of a call
        dict(name="weights 1 token", op="weights", S=1, N=1, H=16, HKV=8, D=128, page=64, lo=390, hi=390, half=False, decay=1.0),
        # the plain step of eight ragged sequences, small pages
        dict(name="weights 8 tokens", op="weights", S=8, N=1, H=16, HKV=8, D=128, page=16, lo=390, hi=1990, half=False, decay=1.0),
        # the other decoder's heads: the last 32 rows of four prompts score all of them
        dict(name="weights 4 windows of 32, D 64", op="weights", S=4, N=32, H=20, HKV=20, D=64, page=24, lo=700, hi=1468, half=False, decay=0.0),
        # a full server with long ragged caches, four tokens accepted a step, f16 queries, old weights fading
        dict(name="weights 16 long", op="weights", S=16, N=4, H=16, HKV=8, D=128, page=128, lo=4001, hi=8190, half=True, decay=0.99),
        # one sequence gives an eighth of its positions back
        dict(name="evict 1 sequence", op="evict", S=1, HKV=8, D=128, L=28, page=64, lo=512, hi=512, keep=448, sink=4, recent=64),
        # eight ragged sequences, some still below their budget, small pages
        dict(name="evict 8 sequences", op="evict", S=8, HKV=8, D=128, L=28, page=16, lo=390, hi=1990, keep=1024, sink=4, recent=128),
        # two long recordings to a quarter
        dict(name="evict 2 long", op="evict", S=2, HKV=4, D=128, L=12, page=64, lo=30011, hi=32003, keep=8000, sink=16, recent=1024),
    ]


def draw(rng):
    def span(lo, hi):  # spread over the logarithm, ends included
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.99)) - 0.001)))))

    op = rng.choice(["sample", "sample", "weights", "weights", "evict"])
    if op == "sample":
        V, kids = span(500, 260000), rng.choice([0, 0, 1, 1, 2, 4])
        most = 32 * 61 * 151936 // V if kids == 0 else 128 * 151936 // V // kids
        S = span(1, max(1, min(32, most)))
        N = span(1 if kids == 0 else 2, max(2, min(64, most // S)))
        return dict(op=op, S=S, N=N, V=V, kids=kids, greedy=rng.random() < 0.4)
    H, HKV, D = rng.choice([(16, 8, 128), (16, 8, 128), (20, 20, 64), (32, 4, 128), (6, 6, 64), (12, 2, 64), (8, 1, 128), (15, 5, 128)])
    page = rng.choice([8, 16, 16, 24, 32, 40, 64, 64, 128, 256])
    if op == "weights":
        S, N = span(1, 32), span(1, 64)
        most = min(32003, 16 * 6000 * 8 * 128 // (S * HKV * D))  # no more cache than the largest listed case
        most = min(most, 16 * 6000 * 4 * 16 * 128 // (S * N * H * D))
        hi = span(1, max(1, most))
        return dict(op=op, S=S, N=N, H=H, HKV=HKV, D=D, page=page, lo=rng.choice([hi, hi // 2, hi // 7, 0]), hi=hi,
                    half=rng.random() < 0.5, decay=rng.choice([0.0, 0.9, 1.0, 1.0]))
    L = rng.choice([1, 4, 12, 28])
    S = span(1, 16)
    hi = span(8, max(8, min(32003, 8 * 1024 * 28 * 8 * 128 // (S * L * HKV * D))))
    keep = span(max(1, hi // 16), hi)
    sink = min(keep, rng.choice([0, 1, 4, 16]))
    return dict(op=op, S=S, HKV=HKV, D=D, L=L, page=page, lo=rng.choice([hi, hi // 2, hi // 7, 0]), hi=hi, keep=keep, sink=sink,
                recent=min(keep - sink, rng.choice([0, 1, 32, keep // 4])))


# ---- what a case fixes: lengths (the seed makes values, trees and page orders) ----------
def pasts(c):
    """Committed positions per sequence: spread evenly over [lo, hi], shuffled by a stride."""
    S = c["S"]
    return [c["hi"] - (c["hi"] - c["lo"]) * ((s * 5) % S) // max(1, S - 1) if S > 1 else c["hi"] for s in range(S)]


def nodes(c):
    """Live nodes per sequence: every third sequence has about three quarters of the width."""
    return [c["N"] if s % 3 != 2 else max(1, c["N"] * 3 // 4) for s in range(c["S"])]


def work(case):
    c = case
    if c["op"] == "sample":
        n = sum(nodes(c))
        # every target row once; a draft's row only where its children are rejected, which is left out
        return {"bytes": n * (c["V"] * 4 + 8 + (8 if c["kids"] else 0)) + c["S"] * c["N"] * 8, "flops": 4 * n * c["V"]}
    HKV, D = c["HKV"], c["D"]
    if c["op"] == "weights":
        n = nodes(c)
        keys = [p + m for p, m in zip(pasts(c), n)]
        b = sum(keys) * HKV * D * 2 + sum(n) * c["H"] * D * (2 if c["half"] else 4)
        b += 4 * HKV * (sum(keys) + (sum(pasts(c)) if c["decay"] else 0))
        return {"bytes": b, "flops": 2 * c["H"] * D * sum(k * m for k, m in zip(keys, n))}
    full = [p for p in pasts(c) if p > c["keep"]]
    # the weights; then the kept rows and their weights, but the sinks in front, read and written
    return {"bytes": c["L"] * HKV * (4 * sum(full) + 2 * len(full) * (c["keep"] - c["sink"]) * (4 * D + 4)), "flops": 0}


# ---- inputs -------------------------------------------------------------------------------
def random_trees(r, S, N, kids):
    """Parents of random draft trees with at most `kids` children a node: node 0 is the root, a
    node's parent comes before it."""
    par = np.full((S, N), -1, np.int32)
    for s in range(S):
        free = np.full(N, kids)
        for i in range(1, N):
            up = i - 1 if r.rand() < 0.5 else int(r.rand() * i)
            while free[up] == 0:  # the node before always has room
                up += 1
            par[s, i] = up
            free[up] -= 1
    return par


def prepare(case, seed):
    c = case
    r = np.random.RandomState(seed % (1 << 32))
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device="cuda", dtype=dtype)

    def ints(a):
        return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()

    st = dict(c)
    S = c["S"]
    if c["op"] == "sample":
        N, V = c["N"], c["V"]
        # a flat vocabulary with a few likely tokens per row
        x = normal(S, N, V).mul_(2.0)
        at = torch.randint(0, V, (S, N, 8), generator=g, device="cuda")
        x.scatter_add_(2, at, 6.0 + 8.0 * torch.rand(S, N, 8, generator=g, device="cuda"))
        st["logits"] = x
        temp = np.array([0.2, 0.4, 0.6, 0.8, 1.0], np.float32)[r.randint(0, 5, S)]
        if c["greedy"]:
            temp[-1] = 0.0
        st["temperature"] = torch.from_numpy(temp).cuda()
        st["uniforms"] = torch.rand(S, N, 2, generator=g, device="cuda")
        st["n_nodes"] = ints(nodes(c))
        st["target"], st["logprob"] = ints(np.zeros((S, N))), torch.zeros(S, N, device="cuda")
        st["tokens"] = st["parents"] = st["draft"] = None
        if c["kids"]:
            par = random_trees(r, S, N, c["kids"])
            st["parents"] = ints(par)
            warm = torch.from_numpy(np.maximum(temp, 0.2)).cuda()[:, None, None]
            st["draft"] = torch.softmax((x + 0.4 * normal(S, N, V)) / warm, -1)
            up = st["draft"].gather(1, st["parents"].clamp(min=0).long()[..., None].expand(S, N, V))
            st["tokens"] = torch.multinomial(up.view(S * N, V), 1, generator=g).view(S, N).int()
        return st
    HKV, D, page, L = c["HKV"], c["D"], c["page"], c.get("L", 1)
    MP = -(-(c["hi"] + c.get("N", 0)) // page)
    P = S * MP + 2
    st["P"] = P
    st["k"] = normal(L * P, HKV, page, D, dtype=torch.float16)
    st["page_table"] = ints(r.permutation(P)[: S * MP].reshape(S, MP))
    st["n_past"] = ints(pasts(c))
    # accumulated weights: mostly small, a few large
    st["weights"] = normal(L * P, HKV, page).mul_(1.5).exp_()
    if c["op"] == "evict":
        st["v"] = normal(L * P, HKV, page, D, dtype=torch.float16)
        st["n_keep"] = ints(np.full(S, c["keep"]))
        st["n_past_out"] = ints(np.zeros(S))
        return st
    st["n_nodes"] = ints(nodes(c))
    # normed queries and keys: entries about 1, scores of a few units
    st["q"] = normal(S, c["N"], c["H"], D).to(torch.float16 if c["half"] else torch.float32).permute(0, 2, 1, 3)
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
        return {"sample": plain_sample, "weights": plain_weights, "evict": plain_evict}[st["op"]](st)
    be = backend()
    if st["op"] == "sample":
        be.tree_sample(st["logits"], st["temperature"], st["uniforms"], st["tokens"], st["parents"], st["draft"], st["n_nodes"], st["target"],
                       st["logprob"])
        return [st["target"], st["logprob"]]
    if st["op"] == "weights":
        be.attn_weights(st["q"], st["k"], st["page_table"], st["n_past"], st["n_nodes"], st["scale"], st["decay"], st["weights"])
        return st["weights"]
    be.kv_evict(st["weights"], st["page_table"], st["n_past"], st["n_keep"], st["sink"], st["recent"], st["k"], st["v"], st["L"],
                st["n_past_out"])
    return [st["k"], st["v"], st["weights"], st["n_past_out"]]


def plain_sample(st):
    S, N, V = st["S"], st["N"], st["V"]
    dev = st["logits"].device
    x, T = st["logits"].double(), st["temperature"].double()[:, None, None]
    ok = torch.isfinite(x)
    m = x.masked_fill(~ok, -math.inf).amax(-1, keepdim=True)
    w = torch.where(ok, torch.exp((x - m) / torch.where(T > 0, T, torch.ones_like(T))), torch.zeros_like(x))
    at = torch.arange(V, device=dev)
    first = torch.where(x == m, at, V).amin(-1, keepdim=True)
    w = torch.where(T > 0, w, (at == first).double())
    z = w.sum(-1, keepdim=True)
    r = w / z
    i = torch.arange(N, device=dev)
    live = i[None] < st["n_nodes"][:, None]
    target = torch.full((S, N), -1, device=dev, dtype=torch.long)
    if st["draft"] is not None:
        par, tok = st["parents"].long(), st["tokens"].long()
        same = (par[:, :, None] == par[:, None]) & (par >= 0)[:, :, None] & live[:, None] & (i[None, None] < i[None, :, None])
        rank = same.sum(-1)  # a child's place among its siblings
        open_ = torch.ones(S, N, dtype=torch.bool, device=dev)
        p = r
        for k in range(st["kids"]):
            child = live & (par >= 0) & (rank == k)
            kid = torch.full((S, N + 1), N, device=dev).scatter(1, torch.where(child, par, N), i.expand(S, N))[:, :N]
            has = open_ & (kid < N)
            kid = kid.clamp(max=N - 1)
            t = tok.gather(1, kid)
            u = st["uniforms"][..., 0].double().gather(1, kid)
            take = has & (u * st["draft"].gather(2, t[..., None])[..., 0].double() < r.gather(2, t[..., None])[..., 0])
            target = torch.where(take, t, target)
            open_ = open_ & ~take
            rest = (r - st["draft"].double()).clamp(min=0)
            total = rest.sum(-1, keepdim=True)
            # a residual without mass: the target's own probabilities
            rest = torch.where(total > 0, rest / total, p)
            r = torch.where((has & ~take)[..., None], rest, r)
    total = r.sum(-1)
    cum = r.cumsum(-1)
    drawn = (cum <= (st["uniforms"][..., 1].double() * total)[..., None]).sum(-1)
    last = torch.where(r > 0, at, 0).amax(-1)
    target = torch.where(target < 0, torch.minimum(drawn, last), target)
    logp = (x.gather(2, target[..., None]) - m) / torch.where(T > 0, T, torch.ones_like(T)) - z.log()
    logp = torch.where(live & (T[..., 0] > 0), logp[..., 0], torch.zeros_like(total))
    return [torch.where(live, target, torch.full_like(target, -1)).int(), logp.float()]


def plain_weights(st):
    S, N, H, HKV, D, page = (st[x] for x in ("S", "N", "H", "HKV", "D", "page"))
    dev = st["q"].device
    pt = st["page_table"].long()
    k = st["k"][pt].permute(0, 2, 1, 3, 4).reshape(S, HKV, -1, D).float()
    T = k.shape[2]
    at = torch.arange(T, device=dev)
    i = torch.arange(N, device=dev)
    end = st["n_past"] + st["n_nodes"]
    sees = (at <= st["n_past"][:, None, None] + i[None, :, None]) & (i[None] < st["n_nodes"][:, None])[..., None]  # (S, N, T)
    q = st["q"].float().reshape(S, HKV, -1, D)
    s = (torch.matmul(q, k.transpose(2, 3)) * st["scale"]).reshape(S, H, N, T).masked_fill(~sees[:, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m))
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / l, torch.zeros_like(p)).reshape(S, HKV, -1, T).sum(2)  # (S, HKV, T)
    w = st["weights"]
    old = w[pt].permute(0, 2, 1, 3).reshape(S, HKV, T)
    kept = (at < st["n_past"][:, None])[:, None]
    new = torch.where(kept, old * st["decay"], torch.zeros_like(old)) + p if st["decay"] else p
    new = torch.where((at < end[:, None])[:, None], new, old)
    w[pt] = new.reshape(S, HKV, -1, page).permute(0, 2, 1, 3)
    return w


def plain_evict(st):
    S, L, P, HKV, D, page, keep, sink, recent = (st[x] for x in ("S", "L", "P", "HKV", "D", "page", "keep", "sink", "recent"))
    pt, past = st["page_table"].long(), st["n_past"].long()
    w = st["weights"].view(L, P, HKV, page)
    T = pt.shape[1] * page
    at = torch.arange(T, device=w.device)
    order = w[:, pt].permute(0, 1, 3, 2, 4).reshape(L, S, HKV, T)
    always = (at < sink) | (at >= past[:, None] - recent)
    order = order.masked_fill(always[None, :, None], math.inf).masked_fill((at >= past[:, None])[None, :, None], -math.inf)
    pick = order.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(dim=-1).values  # (L, S, HKV, keep)
    full = past > keep
    j = torch.arange(pick.shape[-1], device=w.device)
    pick = torch.where(full[None, :, None, None], pick, j)  # below the budget all stay where they are
    s = torch.arange(S, device=w.device)[None, :, None, None]
    l, h = torch.arange(L, device=w.device)[:, None, None, None], torch.arange(HKV, device=w.device)[None, None, :, None]
    src = (l, pt[s, pick // page], h, pick % page)
    dst = (l, pt[s, j // page], h, j % page)
    for x in (st["k"].view(L, P, HKV, page, D), st["v"].view(L, P, HKV, page, D), w):
        x[dst] = x[src]
    return [st["k"], st["v"], st["weights"], torch.where(full, torch.full_like(past, keep), past).int()]


# ---- 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    c = case
    st = prepare(c, seed)
    S = c["S"]
    if c["op"] == "sample":
        N, V = c["N"], c["V"]
        out, logp = np.full((S, N), -1, np.int32), np.zeros((S, N))
        T, u = st["temperature"].tolist(), st["uniforms"].double().cpu().numpy()
        par = st["parents"].cpu().numpy() if c["kids"] else None
        tok = st["tokens"].cpu().numpy() if c["kids"] else None
        for s in range(S):
            for i in range(nodes(c)[s]):
                x = st["logits"][s, i]
                if T[s] == 0:
                    out[s, i] = int(torch.nonzero(x == x.max())[0])
                    continue
                p = torch.softmax(x.double() / T[s], -1)
                rest, found = p, None
                for j in [] if par is None else [j for j in range(i + 1, nodes(c)[s]) if par[s, j] == i]:
                    q = st["draft"][s, i].double()
                    t = int(tok[s, j])
                    if u[s, j, 0] * float(q[t]) < float(rest[t]):
                        found = t
                        break
                    rest = torch.relu(rest - q)
                    rest = rest / rest.sum() if float(rest.sum()) > 0 else p
                if found is None:
                    cum = rest.cumsum(0)
                    found = int(torch.searchsorted(cum, u[s, i, 1] * float(cum[-1]), right=True))
                    found = min(found, int(torch.nonzero(rest)[-1]))
                out[s, i] = found
                logp[s, i] = float(torch.log_softmax(x.double() / T[s], -1)[found])
        return [torch.from_numpy(out).cuda(), torch.from_numpy(logp).cuda()]
    HKV, D, page, P = c["HKV"], c["D"], c["page"], st["P"]
    past = pasts(c)
    table = st["page_table"].long()
    w = st["weights"].double()
    if c["op"] == "weights":
        G, N = c["H"] // HKV, c["N"]
        for s in range(S):
            n, T = nodes(c)[s], past[s] + nodes(c)[s]
            p = torch.arange(T, device="cuda")
            pg, off = table[s, p // page], p % page
            hide = p[None] > past[s] + torch.arange(n, device="cuda")[:, None]
            for h in range(HKV):
                k = st["k"][pg, h, off].double()
                got = torch.zeros(T, device="cuda", dtype=torch.float64)
                for a in range(h * G, (h + 1) * G):
                    score = (st["q"][s, a, :n].double() @ k.T * c_scale(D)).masked_fill(hide, -math.inf)
                    got += torch.softmax(score, -1).sum(0)
                old = w[pg, h, off] * c["decay"]
                old[past[s]:] = 0.0
                w[pg, h, off] = old + got
        return w
    L, keep = c["L"], c["keep"]
    k, v = (st[x].double() for x in ("k", "v"))
    for s in range(S):
        if past[s] <= keep:
            continue
        free = keep - c["sink"] - c["recent"]
        mid = torch.arange(c["sink"], past[s] - c["recent"], device="cuda")
        to = torch.arange(keep, device="cuda")
        for l in range(L):
            rows = table[s] + l * P
            for h in range(HKV):
                score = w[rows[mid // page], h, mid % page]
                best = mid[torch.argsort(-score, stable=True)[:free]].sort().values
                pick = torch.cat([to[:c["sink"]], best, torch.arange(past[s] - c["recent"], past[s], device="cuda")])
                for x in (k, v, w):
                    x[rows[to // page], h, to % page] = x[rows[pick // page], h, pick % page]
    return [k, v, w, torch.tensor([min(p, keep) for p in past], dtype=torch.int32, device="cuda")]


def c_scale(D):
    return 1.0 / math.sqrt(D)
