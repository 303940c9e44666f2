"""What tree_sample, attn_weights and kv_evict refuse before anything reaches a device: the entry points
themselves on a backend without one (a call that is in order gets as far as the device and no further),
and the Python calls."""
import ctypes
import os
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

import openasr_b200 as ob  # noqa: E402
from openasr_b200 import backend as bk  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else shutil.which("nvcc"))

BACKEND = r"""
#include "common.cuh"
extern "C" oasr_backend *backend_without_device() {
    oasr_backend *be = new oasr_backend();
    be->device = 1 << 20;  // no such one, also where there is a GPU
    be->sm_count = 148;
    return be;
}
"""


@pytest.fixture(scope="module")
def be(tmp_path_factory):
    if not NVCC:
        pytest.skip("no nvcc")
    d = tmp_path_factory.mktemp("backend")
    (d / "b.cu").write_text(BACKEND)
    subprocess.run([NVCC, "-std=c++17", "-shared", "-Xcompiler", "-fPIC", "-ccbin", shutil.which("g++", path="/usr/bin") or "g++",
                    "-I", os.path.join(ROOT, "openasr_b200", "csrc"), str(d / "b.cu"), "-o", str(d / "b.so")], check=True)
    make = ctypes.CDLL(str(d / "b.so")).backend_without_device
    make.restype = ctypes.c_void_p
    b = bk.Backend.__new__(bk.Backend)
    b.handle, b.ordinal = ctypes.c_void_p(make()), -1
    return b


def f(*d):
    return ob.describe(torch.zeros(*d))


def h(*d):
    return ob.describe(torch.zeros(*d, dtype=torch.float16))


def i(*d):
    return ob.describe(torch.zeros(*d, dtype=torch.int32))


def at(desc, data=None, **strides):
    """the descriptor at another address, or with another stride"""
    d = bk.OasrTensor.from_buffer_copy(desc)
    if data is not None:
        d.data = data
    for k, v in strides.items():
        d.nb[int(k[2:])] = v
    return d


@pytest.fixture(autouse=True)
def kept(monkeypatch):
    """descriptors of tensors whose memory nobody reads: give each an address of its own"""
    place = [1 << 40]

    def describe(t, ggml_type=None):
        d = real(t, ggml_type)
        if type(t) is not bk.OasrTensor:
            place[0] += 1 << 32
            d.data = place[0]
        return d

    real = bk.describe
    monkeypatch.setattr(ob, "describe", describe)


def sample(be, **change):
    S, N, V = 2, 3, 50
    a = dict(x=f(S, N, V), temp=f(S), u=f(S, N, 2), tok=i(S, N), par=i(S, N), q=f(S, N, V), live=i(S), t=i(S, N), lp=f(S, N))
    a.update({k: v(a) if callable(v) else v for k, v in change.items()})
    be.tree_sample(a["x"], a["temp"], a["u"], a["tok"], a["par"], a["q"], a["live"], a["t"], a["lp"])


def weights(be, **change):
    S, N, H, HKV, D, page, P = 2, 3, 4, 2, 64, 16, 6
    a = dict(q=f(S, H, N, D), k=h(P, HKV, page, D), table=i(S, 3), past=i(S), live=i(S), scale=0.1, decay=1.0, w=f(P, HKV, page))
    a.update({k: v(a) if callable(v) else v for k, v in change.items()})
    be.attn_weights(a["q"], a["k"], a["table"], a["past"], a["live"], a["scale"], a["decay"], a["w"])


def evict(be, **change):
    S, HKV, D, page, P = 2, 2, 128, 16, 6
    a = dict(w=f(P, HKV, page), table=i(S, 3), past=i(S), keep=i(S), sink=0, recent=0, k=h(P, HKV, page, D), v=h(P, HKV, page, D), L=1, out=i(S))
    a.update({k: v(a) if callable(v) else v for k, v in change.items()})
    be.kv_evict(a["w"], a["table"], a["past"], a["keep"], a["sink"], a["recent"], a["k"], a["v"], a["L"], a["out"])


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("call,change", [
    (sample, {}), (sample, dict(temp=None, live=None, lp=None)), (sample, dict(tok=None, par=None, q=None)),
    (sample, dict(x=lambda a: at(a["x"], data=a["x"].data + 4))),                 # rows of any 4-byte alignment
    (sample, dict(x=lambda a: at(a["x"], nb1=4 * 53, nb2=4 * 400))),
    (sample, dict(t=lambda a: at(a["t"], data=a["u"].data + 4096))),
    (weights, {}), (weights, dict(live=None, decay=0.0)), (weights, dict(q=lambda a: h(2, 4, 3, 64))),
    (weights, dict(w=lambda a: at(a["w"], nb1=384, nb2=64))), (weights, dict(w=lambda a: at(a["w"], nb1=68, nb2=132))),
    (evict, {}), (evict, dict(L=3)), (evict, dict(sink=5, recent=7)),
])
def test_calls_in_order_reach_the_device(be, call, change):
    with pytest.raises(ob.GgmlBackendError) as e:
        call(be, **change)
    assert e.value.status == bk.STATUS_DEVICE_LOST


@pytest.mark.parametrize("call,change,says", [
    (sample, dict(x=None), "null argument"), (sample, dict(u=None), "null argument"), (sample, dict(t=None), "null argument"),
    (sample, dict(tok=None), "come together"), (sample, dict(par=None), "come together"), (sample, dict(q=None), "come together"),
    (sample, dict(x=lambda a: h(2, 3, 50)), "logits must be F32"), (sample, dict(x=lambda a: at(a["x"], nb0=8)), "logits must be F32"),
    (sample, dict(x=lambda a: at(a["x"], data=a["x"].data + 2)), "logits must be F32"),
    (sample, dict(x=lambda a: at(a["x"], nb1=202)), "logits must be F32"), (sample, dict(x=lambda a: f(2, 3, 0)), "1 to 2"),
    (sample, dict(u=lambda a: f(2, 3, 3)), "uniforms"), (sample, dict(u=lambda a: f(2, 4, 2)), "uniforms"),
    (sample, dict(u=lambda a: at(a["u"], nb0=8)), "uniforms"),
    (sample, dict(temp=lambda a: f(3)), "temperature"), (sample, dict(temp=lambda a: i(2)), "temperature"),
    (sample, dict(temp=lambda a: at(a["temp"], nb0=8)), "temperature"), (sample, dict(live=lambda a: f(2)), "n_nodes"),
    (sample, dict(q=lambda a: f(2, 3, 51)), "draft_probs"), (sample, dict(tok=lambda a: i(2, 4)), "tokens and parents"),
    (sample, dict(t=lambda a: i(3, 2)), "target must be"), (sample, dict(t=lambda a: f(2, 3)), "target must be"),
    (sample, dict(t=lambda a: at(a["t"], nb1=8)), "must not overlap"), (sample, dict(t=lambda a: at(a["t"], nb1=0)), "must not overlap"),
    (sample, dict(lp=lambda a: i(2, 3)), "logprob"), (sample, dict(t=lambda a: a["tok"]), "overlap an input"),
    (sample, dict(t=lambda a: at(a["t"], data=a["x"].data + 4 * 299)), "overlap an input"),
    (sample, dict(t=lambda a: at(a["t"], data=a["q"].data + 4 * 149)), "overlap an input"),
    (sample, dict(lp=lambda a: at(a["lp"], data=a["u"].data + 44)), "overlap an input"),
    (sample, dict(lp=lambda a: at(a["lp"], data=a["live"].data)), "overlap an input"),
    (sample, dict(lp=lambda a: at(a["lp"], data=a["t"].data + 20)), "target and logprob must not overlap"),
    (weights, dict(q=None), "null argument"), (weights, dict(k=None), "null argument"), (weights, dict(w=None), "weights must be"),
    (weights, dict(table=None), "null argument"), (weights, dict(past=None), "null argument"),
    (weights, dict(q=lambda a: f(2, 3, 3, 64)), "q must be"), (weights, dict(q=lambda a: f(2, 4, 3, 128)), "q must be"),
    (weights, dict(q=lambda a: i(2, 4, 3, 64)), "q must be"), (weights, dict(q=lambda a: at(a["q"], nb0=8)), "contiguous"),
    (weights, dict(q=lambda a: at(a["q"], nb1=260)), "16-byte"), (weights, dict(q=lambda a: at(a["q"], data=a["q"].data + 8)), "16-byte"),
    (weights, dict(k=lambda a: f(6, 2, 16, 64)), "must be F16"), (weights, dict(k=lambda a: h(6, 2, 12, 64), w=lambda a: f(6, 2, 12)), "multiple of 8"),
    (weights, dict(k=lambda a: h(6, 2, 16, 96), q=lambda a: f(2, 4, 3, 96)), "64 or 128"),
    (weights, dict(w=lambda a: f(6, 2, 17)), "weights must be"), (weights, dict(w=lambda a: f(7, 2, 16)), "weights must be"),
    (weights, dict(w=lambda a: h(6, 2, 16)), "weights must be"), (weights, dict(w=lambda a: at(a["w"], nb0=8)), "weights must be"),
    (weights, dict(w=lambda a: at(a["w"], nb1=-64)), "weights must be"), (weights, dict(w=lambda a: at(a["w"], nb1=0)), "weights must be"),
    (weights, dict(w=lambda a: at(a["w"], nb2=64)), "weights must be"), (weights, dict(w=lambda a: at(a["w"], nb1=60, nb2=600)), "weights must be"),
    (weights, dict(w=lambda a: at(a["w"], nb1=380, nb2=64)), "weights must be"), (weights, dict(w=lambda a: at(a["w"], data=a["w"].data + 2)), "weights must be"),
    (weights, dict(scale=NAN), "scale"), (weights, dict(decay=-1.0), "decay"), (weights, dict(decay=NAN), "decay"), (weights, dict(decay=INF), "decay"),
    (weights, dict(table=lambda a: i(3, 3)), "page_table"), (weights, dict(past=lambda a: i(3)), "n_past"), (weights, dict(live=lambda a: f(2)), "n_nodes"),
    (evict, dict(past=None), "null argument"), (evict, dict(w=None), "weights must be"), (evict, dict(keep=None), "n_keep"),
    (evict, dict(out=None), "n_keep and n_past_out"), (evict, dict(v=lambda a: h(6, 2, 16, 64)), "one shape"),
    (evict, dict(k=lambda a: f(6, 2, 16, 128), v=lambda a: f(6, 2, 16, 128)), "must be F16"),
    (evict, dict(w=lambda a: f(6, 2, 24)), "weights must be"), (evict, dict(L=4), "n_layers"), (evict, dict(L=0), "n_layers"), (evict, dict(L=-1), "n_layers"),
    (evict, dict(sink=-1), "negative"), (evict, dict(recent=-1), "negative"), (evict, dict(keep=lambda a: f(2)), "n_keep"),
    (evict, dict(out=lambda a: a["past"]), "overlap"), (evict, dict(out=lambda a: a["keep"]), "overlap"),
    (evict, dict(out=lambda a: at(a["out"], data=a["table"].data + 16)), "overlap"), (evict, dict(table=lambda a: i(1, 3)), "page_table"),
])
def test_refusals(be, call, change, says):
    with pytest.raises(bk.UnsupportedInputs, match=says):
        call(be, **change)


def test_more_nodes_than_a_tree_may_have(be):
    big = dict(x=f(1, 1025, 4), temp=None, u=f(1, 1025, 2), live=None, t=i(1, 1025), lp=None)
    with pytest.raises(bk.UnsupportedInputs, match="1024"):
        sample(be, **big, tok=i(1, 1025), par=i(1, 1025), q=f(1, 1025, 4))
    with pytest.raises(ob.GgmlBackendError) as e:  # without a draft they are rows like any others
        sample(be, **big, tok=None, par=None, q=None)
    assert e.value.status == bk.STATUS_DEVICE_LOST


def calls(b, t):
    return (lambda: b.tree_sample(t, t, t, t, t, t, t, t, t), lambda: b.attn_weights(t, t, t, t, t, 0.5, 1.0, t),
            lambda: b.kv_evict(t, t, t, t, 0, 0, t, t, 1, t))


@pytest.fixture(params=["extension", "ctypes"])
def ops(request, monkeypatch):
    if request.param == "ctypes":
        monkeypatch.setattr(bk, "_OPS", bk._CtypesOps())
    elif isinstance(bk._ops(), bk._CtypesOps):
        pytest.skip("built without torch's headers")


def test_the_python_calls(ops):
    b = bk.Backend.__new__(bk.Backend)
    b.handle, b.ordinal = ctypes.c_void_p(0), 0
    for call in calls(b, bk.describe(torch.zeros(2, 2))):
        with pytest.raises(bk.GgmlBackendError, match="null backend"):
            call()
    for call in calls(b, torch.zeros(2, 2)):
        with pytest.raises(bk.UnsupportedInputs, match="another device than the backend's: cpu"):
            call()
    for call in calls(b, torch.zeros(2, 2, dtype=torch.bfloat16)):
        with pytest.raises(bk.UnsupportedInputs, match="dtype"):
            call()


def test_results_beside_many_rows_are_checked_at_once(be):
    """a column of results in the buffer of the logits: nothing is shared, and that does not take a step per pair of rows"""
    import time

    S, V = 1 << 17, 2
    x, t = f(S, 1, V), i(S, 1)
    at_once = dict(x=at(x, nb1=12, nb2=12), t=at(t, data=x.data + 8, nb1=12), u=f(S, 1, 2), temp=f(S), live=i(S), tok=None, par=None, q=None,
                   lp=f(S, 1))
    start = time.perf_counter()
    with pytest.raises(ob.GgmlBackendError) as e:
        sample(be, **at_once)
    assert e.value.status == bk.STATUS_DEVICE_LOST and time.perf_counter() - start < 1.0
    with pytest.raises(bk.UnsupportedInputs, match="overlap an input"):
        sample(be, **{**at_once, "t": at(t, data=x.data + 4, nb1=12)})


@pytest.mark.parametrize("change", [
    dict(w=lambda a: at(a["w"], data=a["q"].data + 4 * 1535)), dict(q=lambda a: at(a["q"], data=a["w"].data + 4 * 176)),
    dict(w=lambda a: at(a["w"], data=a["k"].data + 2 * 6 * 2 * 16 * 64 - 4)), dict(w=lambda a: at(a["w"], data=a["table"].data)),
    dict(w=lambda a: at(a["w"], data=a["past"].data + 4)), dict(live=lambda a: at(a["live"], data=a["w"].data + 764)),
    dict(k=lambda a: at(a["k"], nb3=4096 + 128), w=lambda a: at(a["w"], data=a["k"].data + 4092, nb1=64, nb2=4096 + 128)),
])
def test_weights_in_an_input_are_refused(be, change):
    with pytest.raises(bk.UnsupportedInputs, match="weights must not overlap an input"):
        weights(be, **change)


@pytest.mark.parametrize("change", [
    dict(w=lambda a: at(a["w"], data=a["q"].data + 4 * 1536)), dict(w=lambda a: at(a["w"], data=a["past"].data + 8)),
    dict(k=lambda a: at(a["k"], nb3=4096 + 128), w=lambda a: at(a["w"], data=a["k"].data + 4096, nb1=64, nb2=4096 + 128)),  # behind each page
])
def test_weights_beside_an_input_are_not(be, change):
    with pytest.raises(ob.GgmlBackendError) as e:
        weights(be, **change)
    assert e.value.status == bk.STATUS_DEVICE_LOST


EVICT_PAGES = 6 * 2 * 16 * 128 * 2  # bytes


@pytest.mark.parametrize("change,says", [
    (dict(out=lambda a: at(a["out"], data=a["w"].data + 764)), "n_past_out must not overlap an input"),
    (dict(out=lambda a: at(a["out"], data=a["k"].data + EVICT_PAGES - 4)), "n_past_out must not overlap an input"),
    (dict(out=lambda a: at(a["out"], data=a["v"].data)), "n_past_out must not overlap an input"),
    (dict(v=lambda a: a["k"]), "weights, k_pages and v_pages must not overlap"),
    (dict(v=lambda a: at(a["k"], data=a["k"].data + EVICT_PAGES - 16)), "weights, k_pages and v_pages must not overlap"),
    (dict(w=lambda a: at(a["w"], data=a["v"].data + 4096)), "weights, k_pages and v_pages must not overlap"),
    (dict(w=lambda a: at(a["w"], data=a["table"].data + 8)), "lengths or page table"),
    (dict(past=lambda a: at(a["past"], data=a["k"].data + 512)), "lengths or page table"),
    (dict(keep=lambda a: at(a["keep"], data=a["v"].data + EVICT_PAGES - 8)), "lengths or page table"),
    (dict(k=lambda a: at(a["k"], nb2=0)), "rows of the pages must not overlap"), (dict(v=lambda a: at(a["v"], nb3=0)), "rows of the pages must not overlap"),
    (dict(k=lambda a: at(a["k"], nb1=240)), "rows of the pages must not overlap"),
])
def test_evictions_over_what_is_still_read_are_refused(be, change, says):
    with pytest.raises(bk.UnsupportedInputs, match=says):
        evict(be, **change)


@pytest.mark.parametrize("change", [
    dict(v=lambda a: at(a["k"], data=a["k"].data + EVICT_PAGES)), dict(out=lambda a: at(a["out"], data=a["past"].data + 8)),
    # K and V rows in turn; K, V and weights of a page one after the other
    dict(k=lambda a: at(a["k"], nb1=512, nb2=8192, nb3=16384), v=lambda a: at(a["v"], data=a["k"].data + 256, nb1=512, nb2=8192, nb3=16384)),
    dict(k=lambda a: at(a["k"], nb3=16512), v=lambda a: at(a["v"], data=a["k"].data + 8192, nb3=16512),
         w=lambda a: at(a["w"], data=a["k"].data + 16384, nb2=16512)),
])
def test_evictions_in_one_buffer_are_not(be, change):
    with pytest.raises(ob.GgmlBackendError) as e:
        evict(be, **change)
    assert e.value.status == bk.STATUS_DEVICE_LOST


UNBOUND = """
import ctypes

import torch

from openasr_b200 import _torch_ops as ext, backend as bk

t = bk.describe(torch.zeros(2, 2))
calls = [lambda: ext.tree_sample(5, *[t] * 9), lambda: ext.attn_weights(5, *[t] * 5, 0.5, 1.0, t),
         lambda: ext.kv_evict(5, t, t, t, t, 0, 0, t, t, 1, t)]
first = [lambda: ext.kv_pages_copy(5, t, t, 1, t), lambda: ext.flash_attn_tree(5, *[t] * 7, 0.5, t),
         lambda: ext.qk_norm_rope(5, t, t, t, 0.5, *[t] * 8), lambda: ext.tree_commit(5, *[t] * 8, 1, *[t] * 4)]


def unbound(some):
    for call in some:
        try:
            call()
        except RuntimeError as e:
            assert "has not been bound" in str(e)
        else:
            raise SystemExit("no error")


unbound(calls + first)
copy = ctypes.CFUNCTYPE(ctypes.c_int, *[ctypes.c_void_p] * 3, ctypes.c_int32, ctypes.c_void_p)(lambda *a: 7)
addr = ctypes.cast(copy, ctypes.c_void_p).value
ext.bind(bk._unsupported, *[addr] * 4)
unbound(calls)
assert ext.kv_pages_copy(5, t, t, 1, t) == 7
ext.bind(bk._unsupported, *[addr] * 7)
ext.bind(bk._unsupported, *[addr] * 4)
unbound(calls)
print("done")
"""


def test_a_function_without_an_address_raises():
    """in a process of its own: bound to the first four functions, or to none, the others are not called"""
    if isinstance(bk._ops(), bk._CtypesOps):
        pytest.skip("built without torch's headers")
    import sys

    r = subprocess.run([sys.executable, "-c", UNBOUND], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "done", (r.returncode, r.stdout, r.stderr)
