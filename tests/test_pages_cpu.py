"""Host side of the paged cache: tree masks (no device needed)."""
import numpy as np
import pytest

from openasr_b200 import backend as bk


@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 61, 200, 1024])
def test_tree_mask_is_each_node_with_its_ancestors(n):
    rng = np.random.default_rng(n)
    par = np.array([-1 if i == 0 or rng.random() < 0.05 else rng.integers(0, i) for i in range(n)], np.int32)
    words = bk.tree_mask(par).view(np.uint32)
    assert words.shape == (n, (n + 31) // 32)
    for i in range(n):
        want, j = set(), i
        while j >= 0:
            want.add(j)
            j = int(par[j])
        assert want == {j for j in range(n) if words[i, j // 32] >> np.uint32(j % 32) & np.uint32(1)}


@pytest.mark.parametrize("par", [[0], [-1, 1], [-1, 2, 0], [-2], list(range(-1, 1024))])
def test_tree_mask_refuses_what_is_no_tree(par):
    with pytest.raises(bk.UnsupportedInputs):
        bk.tree_mask(par)


# ---- page accounting -------------------------------------------------------------------------
class Cells:
    """What a pool stands for: every position of a sequence holds the value written last, by the
    sequence itself or by the one it was forked from; pages hold the values."""

    def __init__(self, n_pages, page, max_pages, max_seqs):
        self.pool = bk.KvPool(n_pages, page, max_pages, max_seqs)
        self.page = page
        self.mem = np.full((n_pages, page), -1)
        self.want = {}  # sequence -> list of values
        self.stamp = 0

    def write(self, s, start, end):
        for a, b in self.pool.extend(s, start, end):
            self.mem[b] = self.mem[a]
        row = self.pool.table([s])[0]
        v = self.want[s]
        del v[start:]
        for p in range(start, end):
            self.stamp += 1
            v.append(self.stamp)
            self.mem[row[p // self.page], p % self.page] = self.stamp

    def check(self):
        used = set()
        for s, v in self.want.items():
            row = self.pool.table([s])[0]
            assert [self.mem[row[p // self.page], p % self.page] for p in range(len(v))] == v
            used |= set(row[row >= 0].tolist())
        assert self.pool.pages_free() == len(self.mem) - len(used)


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("seed", range(4))
def test_pool_sequences_keep_their_values_through_forks_and_writes(page, seed):
    rng = np.random.default_rng(seed)
    c = Cells(40, page, 12, 6)
    full = 0
    for _ in range(400):
        act = rng.integers(0, 10)
        live = list(c.want)
        try:
            if act <= 1 or not live:
                c.want[c.pool.open()] = []
            elif act <= 3:
                s = live[rng.integers(len(live))]
                c.want[c.pool.fork(s)] = list(c.want[s])
            elif act == 4:
                s = live[rng.integers(len(live))]
                c.pool.close(s)
                del c.want[s]
            elif act == 5:  # a draft that was not accepted
                s = live[rng.integers(len(live))]
                n = int(rng.integers(0, len(c.want[s]) + 1))
                c.pool.truncate(s, n)
                del c.want[s][n:]
            else:
                s = live[rng.integers(len(live))]
                start = int(rng.integers(max(0, len(c.want[s]) - 3), len(c.want[s]) + 1))
                c.write(s, start, min(12 * page, start + int(rng.integers(0, 2 * page + 2))))
        except bk.AllocFailed:
            full += 1
        c.check()
    assert full > 0, "the pool never ran out"


def test_pool_fork_copies_one_page_only_when_it_is_written():
    p = bk.KvPool(10, 8, 5, 3)
    a = p.open()
    assert len(p.extend(a, 0, 20)) == 0 and p.pages_free() == 7
    b = p.fork(a)
    assert p.pages_free() == 7 and np.array_equal(p.table([a]), p.table([b]))
    assert p.extend(b, 20, 20).shape == (0, 2)
    pairs = p.extend(b, 20, 25)
    ta, tb = p.table([a, b])
    assert pairs.tolist() == [[ta[2], tb[2]]] and ta[:2].tolist() == tb[:2].tolist() and ta[2] != tb[2] and tb[3] >= 0
    assert len(p.extend(a, 20, 24)) == 0, "the other one is alone with its page now"
    assert p.extend(p.fork(a), 8, 24).shape == (0, 2), "whole pages are replaced, not copied"


def test_pool_refusals():
    p = bk.KvPool(3, 8, 2, 2)
    s = p.open()
    for bad in (lambda: p.extend(s, 1, 0), lambda: p.extend(s, -1, 3), lambda: p.extend(s, 9, 12), lambda: p.extend(s, 0, 17),
                lambda: p.extend(7, 0, 1), lambda: p.close(5), lambda: p.fork(-1), lambda: p.truncate(s, -1), lambda: p.table([1]),
                lambda: bk.KvPool(0, 8, 2, 2), lambda: bk.KvPool(4, 8, 1 << 30, 2)):
        with pytest.raises(bk.UnsupportedInputs):
            bad()
    p.extend(s, 0, 16)
    t = p.open()
    with pytest.raises(bk.AllocFailed):
        p.extend(t, 0, 9)
    assert p.pages_free() == 1 and (p.table([t]) == -1).all(), "a refused extend changes nothing"
    with pytest.raises(bk.AllocFailed):
        p.open()
    p.close(t)
    with pytest.raises(bk.UnsupportedInputs):
        p.close(t)


def test_the_extension_passes_what_describe_says():
    """tensors, strided views, ready descriptors and None through the extension and through ctypes"""
    import ctypes

    import torch

    from openasr_b200 import backend as bk

    ext = bk._ops()
    if isinstance(ext, bk._CtypesOps):
        pytest.skip("built without torch's headers")
    got = []

    @ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p, *[ctypes.c_void_p] * 2, ctypes.c_int32, ctypes.c_void_p)
    def copy(be, k, v, n_layers, pairs):
        got.append((be, n_layers, *(None if p is None else ctypes.string_at(p, ctypes.sizeof(bk.OasrTensor)) for p in (k, v, pairs))))
        return 7

    addr = ctypes.cast(copy, ctypes.c_void_p).value
    base = torch.zeros(3, 5, 4, 16, dtype=torch.float16)
    views = [base, base.permute(0, 2, 1, 3), base[1:, :, ::2], base[0, 0, 0], base[0, 0, 0, 0], torch.zeros(2, 0, 3),
             torch.zeros(7, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(1, 1, dtype=torch.float32)]
    try:
        ext.bind(bk._unsupported, addr, addr, addr, addr)
        for t in views:
            assert ext.kv_pages_copy(5, t, None, -2, bk.describe(t)) == 7
            want = bytes(bk.describe(t))
            assert got.pop() == (5, -2, want, None, want)
        with pytest.raises(bk.UnsupportedInputs, match="float64"):
            ext.kv_pages_copy(5, torch.zeros(2, dtype=torch.float64), None, 1, None)
        for args in ((5, "x", None, 1, None), (5, base, base, 2**31, base), (5, base), (5, base, base, 1.5, base)):
            with pytest.raises((TypeError, OverflowError)):
                ext.kv_pages_copy(*args)
        assert not got
    finally:
        bk._OPS = None
        bk._ops()


def test_both_ways_refuse_alike():
    import torch

    from openasr_b200 import backend as bk

    t = torch.zeros(2, 2)
    for ops in (bk._ops(), bk._CtypesOps()):  # no backend: refused before anything is read
        assert ops.kv_pages_copy(0, t, t, 1, t) == bk.STATUS_FAILED
        assert ops.flash_attn_tree(0, t, t, t, t, t, None, None, 0.5, t) == bk.STATUS_FAILED
        assert ops.qk_norm_rope(0, t, None, None, 0.5, t, t, t, t, t, t, t, t) == bk.STATUS_FAILED
        assert ops.tree_commit(0, t, t, t, t, t, t, t, t, 1, t, t, t, t) == bk.STATUS_FAILED
