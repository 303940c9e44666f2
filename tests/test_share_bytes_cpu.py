"""Whether two tensors have a byte in common (op_checks.cuh), against the bytes themselves."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from openasr_b200 import backend as bk  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else shutil.which("nvcc"))

SOURCE = r"""
#include "op_checks.cuh"
extern "C" int shared(const oasr_tensor *a, const oasr_tensor *b) { return oasr::share_bytes(a, b); }
extern "C" int alone(const oasr_tensor *a) { return oasr::apart(a); }
"""


def build(d, source):
    (d / "s.cu").write_text(source)
    subprocess.run([NVCC, "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-ccbin", shutil.which("g++", path="/usr/bin") or "g++",
                    "-I", os.path.join(ROOT, "openasr_b200", "csrc"), str(d / "s.cu"), "-o", str(d / "s.so")], check=True)
    return ctypes.CDLL(str(d / "s.so"))


@pytest.fixture(scope="module")
def checks(tmp_path_factory):
    if not NVCC:
        pytest.skip("no nvcc")
    return build(tmp_path_factory.mktemp("share"), SOURCE)


@pytest.fixture(scope="module")
def shared(checks):
    return lambda a, b: bool(checks.shared(ctypes.byref(a) if a else None, ctypes.byref(b) if b else None))


SIZE = {bk.F32: 4, bk.F16: 2, bk.I32: 4, bk.I64: 8}


def tensor(ty, data, ne, nb):
    t = bk.OasrTensor()
    t.type, t.data = ty, data
    for i in range(4):
        t.ne[i], t.nb[i] = ne[i], nb[i]
    return t


def covered(t):
    at = {t.data}
    for n, b in zip(t.ne, t.nb):
        at = {x + i * b for x in at for i in range(n)}
    return {x + i for x in at for i in range(SIZE[t.type])}


def some(r):
    ty = r.choice(list(SIZE))
    ne = [r.choice([1, 1, 2, 3, 5]) for _ in range(4)]
    kind, nb, at = r.random(), [0] * 4, SIZE[ty]
    order = list(range(4))
    if r.random() < 0.5:
        r.shuffle(order)
    for i in order:  # one inside the other, now and then with room between
        nb[i] = at
        at = (at * ne[i]) + (r.choice([0, 0, 2, 4, 20]) if kind < 0.8 else 0)
    if kind > 0.9:
        nb = [r.choice([-12, -4, 0, 2, 4, 6, 8, 24, 60]) for _ in range(4)]
    if r.random() < 0.2:
        i = r.randrange(4)
        nb[i] = -nb[i]
    return tensor(ty, 100000 + 2 * r.randrange(-120, 120), ne, nb)


def test_random_tensors(shared):
    r = random.Random(1)
    seen = [0, 0]
    for _ in range(6000):
        a, b = some(r), some(r)
        if r.random() < 0.3:  # views of one shape and one set of strides
            b = tensor(a.type, b.data, list(a.ne), list(a.nb))
        want = bool(covered(a) & covered(b))
        seen[want] += 1
        assert shared(a, b) == want == shared(b, a), [(x.type, x.data, list(x.ne), list(x.nb)) for x in (a, b)]
    assert min(seen) > 1000


def test_nothing_shares_nothing(shared):
    a = tensor(bk.F32, 1000, [4, 1, 1, 1], [4, 16, 16, 16])
    empty = tensor(bk.F32, 1000, [4, 0, 1, 1], [4, 16, 16, 16])
    assert shared(a, a) and not shared(a, empty) and not shared(empty, a) and not shared(a, None) and not shared(None, a)
    assert not shared(a, tensor(bk.F32, None, [4, 1, 1, 1], [4, 16, 16, 16]))


@pytest.mark.parametrize("layout", [(1, 2, 8, 16), (4, 3, 2, 128), (16, 8, 1, 64)])
def test_views_of_one_buffer_of_pages(shared, layout):
    """K rows, V rows and weights of a page side by side, in any order of the dimensions; one step, however many pages"""
    pages, heads, page, D = layout[0] << 20, layout[1], 8 * layout[2], layout[3]
    row, block = 2 * D, 2 * D * 8 * layout[2]
    whole = 2 * heads * block + 4 * heads * page
    base = 1 << 44
    k = tensor(bk.F16, base, [D, page, heads, pages], [2, row, block, whole])
    v = tensor(bk.F16, base + heads * block, [D, page, heads, pages], [2, row, block, whole])
    w = tensor(bk.F32, base + 2 * heads * block, [page, heads, pages, 1], [4, 4 * page, whole, whole * pages])
    for a in (k, v, w):
        for b in (k, v, w):
            assert shared(a, b) == (a is b)
    w.data -= 4
    assert shared(w, v) and not shared(w, k)
    # rows of K and V in turn
    k = tensor(bk.F16, base, [D, page, heads, pages], [2, 2 * row, 2 * block, 2 * heads * block])
    v = tensor(bk.F16, base + row, [D, page, heads, pages], [2, 2 * row, 2 * block, 2 * heads * block])
    assert not shared(k, v)
    v.data -= 2
    assert shared(k, v)


def test_elements_in_one_place(checks):
    """what is said to be apart is; what is one dimension inside the other is found to be"""
    r = random.Random(2)
    seen = [0, 0]
    for _ in range(6000):
        t = some(r)
        n = t.ne[0] * t.ne[1] * t.ne[2] * t.ne[3]
        said = bool(checks.alone(ctypes.byref(t)))
        seen[said] += 1
        if said:
            assert len(covered(t)) == n * SIZE[t.type], (t.type, list(t.ne), list(t.nb))
        nested, size = True, SIZE[t.type]
        for b, m in sorted((abs(b), m) for b, m in zip(t.nb, t.ne) if m > 1):
            nested, size = nested and b >= size, size + (m - 1) * b
        assert said == nested, (t.type, list(t.ne), list(t.nb))
    assert min(seen) > 100
