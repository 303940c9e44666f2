"""What the Python calls of the paged cache's operators refuse before anything reaches a device."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from openasr_b200 import backend as bk  # noqa: E402


def calls(be, t):
    """the four calls with tensor t everywhere"""
    return (lambda: be.kv_pages_copy(t, t, 1, t), lambda: be.flash_attn_tree(t, t, t, t, t, None, None, 0.5, t),
            lambda: be.qk_norm_rope(t, None, None, 0.5, t, t, t, t, t, t, t, t),
            lambda: be.tree_commit(t, t, t, t, t, t, t, t, 1, t, t, t, t))


@pytest.fixture(params=["extension", "ctypes"])
def ops(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(bk, "_OPS", bk._CtypesOps())
    elif isinstance(bk._ops(), bk._CtypesOps):
        pytest.skip("built without torch's headers")
    return request.param


def closed_backend():
    be = bk.Backend.__new__(bk.Backend)
    be.handle, be.ordinal = ctypes.c_void_p(0), 0
    return be


def test_a_closed_backend_is_the_librarys_error(ops):
    """as for the other operators: a status of the library, not a TypeError of the binding"""
    be = closed_backend()
    t = bk.describe(torch.zeros(2, 2))
    for call in calls(be, t):
        with pytest.raises(bk.GgmlBackendError, match="null backend"):
            call()


def test_a_tensor_on_the_host_is_refused(ops):
    """the kernels would read it at an address that the device does not have"""
    be = closed_backend()
    for call in calls(be, torch.zeros(2, 2)):
        with pytest.raises(bk.UnsupportedInputs, match="another device than the backend's: cpu"):
            call()
    ready = bk.describe(torch.zeros(2, 2))
    for a in ((torch.zeros(2, 2), ready, 1, ready), (ready, ready, 1, torch.zeros(1, 2, dtype=torch.int32))):
        with pytest.raises(bk.UnsupportedInputs, match="another device"):
            be.kv_pages_copy(*a)
    with pytest.raises(bk.GgmlBackendError, match="null backend"):  # nothing to read: as far as the library
        be.kv_pages_copy(ready, ready, 1, torch.zeros(0, 2, dtype=torch.int32))


def test_a_tensor_of_five_dimensions_is_refused(ops):
    """[layers, pages, heads, positions, D] is no pool of pages: its first layer alone would be taken"""
    be = closed_backend()
    ready = bk.describe(torch.zeros(2, 2))
    with pytest.raises(bk.UnsupportedInputs, match="at most 4 dimensions, not 5"):
        bk._ops().kv_pages_copy(be.handle.value or 0, torch.zeros(2, 3, 2, 8, 64, dtype=torch.float16), ready, 1, ready)


def test_tree_mask_takes_one_sequence():
    """of a table of sequences the first column's length was taken as the number of nodes"""
    for bad in ([[-1, 0, 1], [-1, 0, 0]], [[]]):
        with pytest.raises(bk.UnsupportedInputs):
            bk.tree_mask(bad)
    assert bk.tree_mask([]).shape == (0, 0) and bk.tree_mask([-1, 0]).tolist() == [[1], [3]]
    assert bk.tree_mask([[-1], [0]]).tolist() == [[1], [3]] and bk.tree_mask(-1).tolist() == [[1]], "as before"
