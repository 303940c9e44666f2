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
