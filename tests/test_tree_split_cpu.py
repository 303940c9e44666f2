"""How the tree attention shares its work out: the kernels' own arithmetic (csrc/tree_split.h), compiled
for the host.  Every unit of every item belongs to exactly one CTA that is launched, a CTA leaves at most
two unfinished segments in slots of its own, and the CTAs that share an item are the ones that the join
asks for."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "openasr_b200", "csrc")
CXX = shutil.which("g++", path="/usr/bin") or shutil.which("g++") or "g++"

SOURCE = r"""
#include <cstdint>
#include <vector>
#include "tree_split.h"
using namespace oasr;

// The call's split as the warps of fattn_tree.cuh work it out, their lanes one after the other: S
// sequences (past, n nodes of G rows each, HKV heads), tiles of R rows, `ctas` CTAs.
static TreeUnits count(int S, const int *past, const int *n, int G, int HKV, int R, int ctas, std::vector<int> &steps) {
    TreeUnits w = {};
    int64_t total = 0;
    int most = 0, units = 0;
    steps.resize(S);
    auto items = [&](int s) { return (n[s] * G + R - 1) / R * HKV; };
    for (int s = 0; s < S; ++s) {
        steps[s] = n[s] ? tree_steps(items(s), tree_units(past[s], n[s]), 0, R) : 0;
        total += steps[s];
        if (n[s]) most = std::max(most, tree_units(past[s], n[s]));
        if (n[s]) units += items(s) * tree_units(past[s], n[s]);
    }
    w.total = (int)total;
    if (S <= 32 && most < 32768) {
        const int run = (w.total + ctas - 1) / ctas, even = std::min(most, (units + ctas - 1) / ctas);
        unsigned least = ~0u;
        for (int l = 0; l < 32; ++l) {
            const int t = tree_try(even, most, l);
            int pieces = 0;
            for (int s = 0; s < S; ++s)
                if (n[s]) pieces += items(s) * tree_pieces(tree_units(past[s], n[s]), t, tree_rcp(t));
            least = std::min(least, tree_piece_cost(pieces, ctas, t, most) << 16 | (unsigned)t);
        }
        if (tree_in_pieces(least >> 16, run)) {
            w.piece = (int)(least & 65535u);
            w.total = 0;
            for (int s = 0; s < S; ++s) {
                steps[s] = n[s] ? tree_steps(items(s), tree_units(past[s], n[s]), w.piece, R) : 0;
                w.total += steps[s];
            }
            tree_set_pieces(w);
            return w;
        }
    }
    tree_set_runs(w, ctas);
    return w;
}

extern "C" int fits(int past, int n, int N, int MP, int page) { return kv_lengths_fit(past, n, N, MP, page); }

// 0: right, else a number that says what is not
extern "C" int check(int S, const int *past, const int *n, int G, int HKV, int R, int grid, int *in_pieces) {
    std::vector<int> steps;
    const TreeUnits w = count(S, past, n, G, HKV, R, grid, steps);
    *in_pieces = w.piece;
    int64_t items = 0;
    std::vector<int64_t> base(S + 1, 0);
    for (int s = 0; s < S; ++s) base[s + 1] = items += (int64_t)(n[s] * G + R - 1) / R * HKV;
    std::vector<int> next(items, 0), from(items, -1);  // units done of an item, and the CTA that began it
    std::vector<char> slot(2 * (size_t)grid, 0);
    if (w.ctas > grid) return 1;
    if (tree_start(w, grid) != w.total) return 2;
    for (int c = 0; c < grid; ++c) {
        int s = 0, first = 0;
        const int u0 = tree_start(w, c), u1 = tree_start(w, c + 1);
        if (u1 < u0) return 3;
        for (int u = u0; u < u1;) {
            while (u >= first + steps[s]) first += steps[s++];
            TreeSeg g = {};
            g.s = s, g.first = first, g.past = past[s], g.n = n[s];
            tree_cut(g, w.piece, n[s] * G, R, u, u1);
            if (g.k0 == g.k1) {  // the lead of an item alone: only where the CTA's range ends
                if (g.next != u1) return 4;
                break;
            }
            const int64_t item = base[s] + g.hk * ((n[s] * G + R - 1) / R) + g.rt;
            if (item < base[s] || item >= base[s + 1]) return 5;
            if (next[item] != g.k0) return 6;  // in order, none twice, none left out
            next[item] = g.k1;
            if (g.k0 == 0) from[item] = c;
            if (tree_owner(w, g.first + g.lead) != from[item]) return 7;
            if ((tree_owner(w, g.first + g.per - 1) == c) != (g.k1 == g.kt)) return 8;
            if (!(g.k0 == 0 && g.k1 == g.kt)) {
                const int at = tree_slot(w, c, g.first);
                if (at < 2 * c || at > 2 * c + 1 || slot[at]++) return 9;
                if (g.k0 > 0 && at != 2 * c) return 10;  // the join takes the later parts from there
            }
            u = g.next;
        }
    }
    for (int s = 0; s < S; ++s)
        for (int64_t i = base[s]; i < base[s + 1]; ++i)
            if (next[i] != tree_units(past[s], n[s])) return 11;
    return 0;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("split")
    (d / "split.cpp").write_text(SOURCE)
    subprocess.run([CXX, "-O2", "-std=c++17", "-fPIC", "-shared", "-I", CSRC, str(d / "split.cpp"), "-o", str(d / "split.so")], check=True)
    return ctypes.CDLL(str(d / "split.so"))


def split(lib, past, n, G, HKV, R, grid):
    past, n = np.ascontiguousarray(past, np.int32), np.ascontiguousarray(n, np.int32)
    piece = ctypes.c_int()
    rc = lib.check(len(past), past.ctypes.data_as(ctypes.c_void_p), n.ctypes.data_as(ctypes.c_void_p), G, HKV, R, grid, ctypes.byref(piece))
    return rc, piece.value


@pytest.mark.parametrize("past,n,G,HKV,R,grid", [
    ([390], [1], 2, 8, 16, 32), ([0], [1], 1, 1, 16, 1), ([30011, 32003], [5, 5], 8, 4, 64, 148),
    ([4001 + 261 * s for s in range(16)], [61] * 16, 2, 8, 128, 148), ([0] * 32, [43] * 32, 2, 8, 128, 148),
    ([4096] * 4, [512] * 4, 2, 8, 128, 148), ([5, 0, 0, 700], [16, 0, 3, 16], 2, 8, 32, 148),
    ([100000] * 32, [2048] * 32, 8, 4, 128, 148),   # more steps to a run than a piece's cost can say
    ([0], [131072], 2, 8, 128, 148),                # one chain as long
    ([2**22 - 200] * 2, [64 * 100] * 2, 2, 1, 128, 148),
    ([2**22 - 128], [128], 1, 1, 128, 148), ([2**22 - 100], [1], 1, 1, 16, 296),
])
def test_every_unit_is_done_once(lib, past, n, G, HKV, R, grid):
    assert split(lib, past, n, G, HKV, R, grid)[0] == 0


def test_every_unit_is_done_once_over_the_whole_range(lib):
    rng = np.random.default_rng(1)
    pieces = 0
    for _ in range(3000):
        S = int(np.exp(rng.uniform(0, np.log(70))))
        N = int(np.exp(rng.uniform(0, np.log(5000))))
        hi = int(np.exp(rng.uniform(0, np.log(3e5))))
        G, HKV, R = int(rng.integers(1, 9)), int(rng.choice([1, 2, 4, 8, 20])), int(rng.choice([16, 32, 64, 128]))
        past, n = rng.integers(0, hi + 1, S), rng.integers(0, N + 1, S)
        grid = int(rng.choice([1, 2, 7, 148, 296]))
        if sum(-(-int(x) * G // R) * HKV * ((int(p) + int(x)) // 128 + 10) for p, x in zip(past, n)) > 2**30:
            continue  # the launch refuses it
        rc, piece = split(lib, past, n, G, HKV, R, grid)
        assert rc == 0, (past, n, G, HKV, R, grid)
        pieces += piece > 0
    assert pieces > 300


@pytest.mark.parametrize("past,n,N,MP,page,want", [
    (0, 0, 1, 1, 8, True), (7, 1, 1, 1, 8, True), (8, 1, 1, 1, 8, False), (7, 2, 1, 1, 8, False), (-1, 1, 1, 1, 8, False),
    (3, -1, 1, 1, 8, False), (-2**31, 1, 1, 1, 8, False), (2**31 - 1, 1, 1, 4096, 2**20, False), (2**31 - 1, 1024, 1024, 2**24, 2**24, False),
    (2**31 - 1 - 128, 0, 5, 4096, 2**20, True), (2**31 - 1 - 129, 1, 1, 4096, 2**20, True), (2**31 - 1 - 128, 1, 1, 4096, 2**20, False),
])
def test_positions_stay_32_bit_numbers(lib, past, n, N, MP, page, want):
    """a cache of 2^31 positions and more (pages shared by many entries of a table) is in bounds, its last
    positions are not numbers that a kernel can hold"""
    assert bool(lib.fits(past, n, N, MP, page)) == want
