"""A drawn number on the border of a stretch of values without weight.

Running sums over the lanes of a warp are rounded differently lane by lane: (v2 + v1) + v0 up to the third, then
(v3 + v2) + (v1 + v0), which may be greater although v3 is 0.  A number between the two belongs to v2 or to the next
value with weight, and to none of the fourth lane's."""
import math
from fractions import Fraction

import numpy as np
import pytest

from test_tree_sample_gpu import cuda

STEPS, MAGIC = 256, 6755399441055744.0


def fma(a, b, c):
    return float(Fraction(a) * Fraction(b) + Fraction(c))


def weight(x):
    """exp(x) as the kernel forms it: 2^(j / 256) from a table, the rest by a polynomial of degree 3"""
    C, A1 = STEPS / math.log(2), math.log(2) / STEPS
    A2 = A1 * A1 / 2
    A3 = A2 * A1 / 3
    z = fma(float(x), C, MAGIC)
    k = int(z - MAGIC)
    r = fma(float(x), C, MAGIC - z)
    p = fma(A3, r, A2)
    p = fma(p, r, A1)
    p = fma(p, r, 1.0)
    return math.ldexp(2.0 ** ((k % STEPS) / STEPS), k // STEPS) * p


def scanned(v):  # the last of eight running sums
    return ((v[7] + v[6]) + (v[5] + v[4])) + ((v[3] + v[2]) + (v[1] + v[0]))


def folded(v):
    return ((v[0] + v[4]) + (v[2] + v[6])) + ((v[1] + v[5]) + (v[3] + v[7]))


def trap(rng, total):
    """eight logits, the fourth -inf, and a number whose place in the running sum is (v2 + v1) + v0, below
    (v3 + v2) + (v1 + v0); None where these turn out alike, or roundings miss it"""
    x = np.full(8, -np.inf, np.float32)
    x[:3] = rng.uniform(-1, 1, 3)
    v = [weight(l) if np.isfinite(l) else 0.0 for l in x]
    at = (v[2] + v[1]) + v[0]
    if not at < (v[3] + v[2]) + (v[1] + v[0]):
        return None
    u = np.float32(rng.integers(1 << 22, 3 << 22) / (1 << 24))
    want = Fraction(at) / (Fraction(float(u)) + Fraction(2) ** -44)  # of all eight
    for i in range(4, 8):  # each fills what the ones before left to some 2^-20 of it
        rest = float(want - sum(map(Fraction, v)))
        if rest <= 0:
            return None
        x[i] = np.nextafter(np.float32(math.log(rest)), np.float32(-np.inf)) if i < 7 else np.float32(math.log(rest))
        v[i] = weight(x[i])
    t = total(v)
    return (x, u) if fma(float(u), t, t * 2.0**-44) == at == fma(t, 2.0**-44, float(u) * t) else None


def traps(total, n):
    rng = np.random.default_rng(1)
    found = []
    while len(found) < n:
        found += [t for t in [trap(rng, total)] if t]
    return np.stack([t[0] for t in found]), np.array([t[1] for t in found])


@pytest.mark.parametrize("total", [scanned, folded])
def test_the_numbers_lie_where_they_should(total):
    x, u = traps(total, 5)
    for i in range(5):
        p = np.exp(x[i].astype(np.float64))
        assert abs(u[i] * p.sum() - p[:3].sum()) <= 2.0**-43 * p.sum()


@pytest.mark.gpu
@pytest.mark.parametrize("total", [scanned, folded])
@pytest.mark.parametrize("width", [4, 8])
def test_a_stretch_without_weight_is_not_drawn_from(total, width):
    """`width` values for each of a CTA's warps (one vector of 4), or of a stretch's threads (8 values)"""
    import torch

    import openasr_b200 as ob

    n = 96
    small, u1 = traps(total, n)
    x = np.full((n, 1, 8 * width), -np.inf, np.float32)
    x[:, 0, ::width] = small
    if width == 8:  # all in the first warp's run: seven more runs of nothing
        x = np.concatenate([x, np.full((n, 1, 7 * 64), -np.inf, np.float32)], -1)
    u = np.zeros((n, 1, 2), np.float32)
    u[:, 0, 1] = u1
    be = ob.Backend(0)
    be.set_stream(torch.cuda.current_stream())
    t = torch.zeros(n, 1, dtype=torch.int32, device="cuda")
    be.tree_sample(cuda(x), None, cuda(u), None, None, None, None, t, None)
    be.synchronize()
    be.close()
    got = t.cpu().numpy()[:, 0]
    assert set(got.tolist()) <= {2 * width, 4 * width}, got
