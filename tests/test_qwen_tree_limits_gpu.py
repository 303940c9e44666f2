"""The Qwen decoder's verification pass where memory or the context ends."""
import numpy as np
import pytest

import openasr_b200 as ob
from openasr_b200 import models as om

pytestmark = pytest.mark.gpu


def test_a_pass_without_memory_is_refused_and_the_next_one_works(gpu_backend):
    """the first pass allocates what later ones reuse; all of it or nothing"""
    import torch

    cfg = om.QWEN3_ASR_0_6B.replace(n_layers=1, max_pos=64, max_prefill=32, max_batch=1)
    m = om.QwenModel(gpu_backend, cfg, om.qwen_synthetic_pack(cfg, seed=0x0A5A0003))
    try:
        _, first = m.prefill(om.qwen_synthetic_prefix(0x0A5A3000, 1, 8, cfg.d_model))
        tree = [[first[0], 5, 6]], [[-1, 0, 1]], [8]
        torch.cuda.empty_cache()
        free, _ = torch.cuda.mem_get_info()
        # leaves 64 MB: less than the 128 rows of logits that a pass needs, 78 MB
        hold = torch.empty(free - (64 << 20), dtype=torch.uint8, device="cuda")
        for _ in range(2):
            with pytest.raises(ob.backend.AllocFailed):
                m.verify_tree(*tree)
        del hold
        torch.cuda.empty_cache()
        path, acc, nxt = m.verify_tree(*tree)
        assert path[0, 0] == 0 and acc[0] >= 1 and 0 <= nxt[0] < cfg.n_vocab
    finally:
        m.close()


def test_prompt_and_tokens_may_fill_the_context(gpu_backend):
    """sequences that accept long drafts end early, at the context's end; the last one gets its tokens"""
    cfg = om.QWEN3_ASR_0_6B.replace(n_layers=1, n_vocab=4096, max_pos=40, max_prefill=16, max_batch=3)
    m = om.QwenModel(gpu_backend, cfg, om.qwen_synthetic_pack(cfg, seed=0x0A5A0003))
    try:
        emb, n_new = om.qwen_synthetic_prefix(0x0A5A3000, 3, 12, cfg.d_model), 28
        serial = m.generate(emb, n_new=n_new)

        def draft(s, tokens):  # the true continuation and some tokens more, one at a time, none
            tk = (serial[s, len(tokens):].tolist() + [1, 2, 3, 4])[:(20, 1, 0)[s]]
            return tk, list(range(-1, len(tk) - 1))

        got, passes = m.generate_speculative(emb, draft, n_new)
        assert got.shape == (3, n_new) and passes == n_new - 1
        assert np.array_equal(got[:, 0], serial[:, 0])
        with pytest.raises(ob.backend.UnsupportedInputs):
            m.generate(emb, n_new=n_new + 1)
    finally:
        m.close()


WITHOUT_HOST_MEMORY = """
import ctypes, resource
import numpy as np
import openasr_b200 as ob
from openasr_b200 import backend as bk, models as om

cfg = om.QWEN3_ASR_0_6B.replace(n_layers=1, n_vocab=4096, max_pos=1040, max_prefill=1024, max_batch=8)
be = ob.Backend(0)
m = om.QwenModel(be, cfg, om.qwen_synthetic_pack(cfg, seed=0x0A5A0003))
_, first = m.prefill(om.qwen_synthetic_prefix(0x0A5A3000, 8, 8, cfg.d_model))
tokens = np.tile(first[:, None], (1, 1024)).astype(np.int32)
parents = np.tile(np.arange(-1, 1023, dtype=np.int32), (8, 1))
pos, path, acc, nxt = np.full(8, 8, np.int32), np.empty_like(tokens), np.zeros(8, np.int32), np.zeros(8, np.int32)
args = (m.handle, tokens.ctypes.data, parents.ctypes.data, 8, 1024, pos.ctypes.data, path.ctypes.data, acc.ctypes.data, nxt.ctypes.data)
verify = bk.lib().oasr_b200_qwen_verify_tree
libc = ctypes.CDLL(None)
libc.malloc.restype, libc.malloc.argtypes, libc.free.argtypes = ctypes.c_void_p, [ctypes.c_size_t], [ctypes.c_void_p]
held, size = [], 1 << 20
pages = int(open("/proc/self/statm").read().split()[0])
_, hard = resource.getrlimit(resource.RLIMIT_AS)
resource.setrlimit(resource.RLIMIT_AS, (pages * 4096, hard))
while size >= 1 << 17:  # the masks of the trees alone take a megabyte
    p = libc.malloc(size)
    if p:
        held.append(p)
    else:
        size >>= 1
rc = verify(*args)
resource.setrlimit(resource.RLIMIT_AS, (hard, hard))
for p in held:
    libc.free(p)
assert rc == bk.STATUS_ALLOC_FAILED, rc
rc = verify(*args)
assert rc == 0 and (acc >= 1).all(), rc
m.close()
be.close()
print("passed")
"""


def test_a_pass_without_host_memory_is_a_status(gpu_backend):
    """not an exception through the C entry, which would end the process"""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(ob.__file__)))
    r = subprocess.run([sys.executable, "-c", WITHOUT_HOST_MEMORY], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("passed\n"), r.stderr[-2000:]


def test_a_pass_over_all_layers(gpu_backend):
    """28 layers: every token that a pass selects is within what the decoder's tensor-core prompt pass is
    held to at full depth (4e-2 of the largest logit, test_qwen_gpu.py) of a decode step's best"""
    bound, T, steps, n = 4e-2, 60, 20, 3
    cfg = om.QWEN3_ASR_0_6B.replace(n_vocab=4096, max_pos=128, max_prefill=64, max_batch=4)
    m = om.QwenModel(gpu_backend, cfg, om.qwen_synthetic_pack(cfg, seed=0x0A5A0003))
    try:
        emb = om.qwen_synthetic_prefix(0x0A5A5000, n, T, cfg.d_model)
        serial = m.generate(emb, n_new=steps)

        def draft(s, tokens):  # two right tokens, beside them a wrong one with a child
            tk = serial[s, len(tokens):len(tokens) + 2].tolist()
            return tk + [(tokens[-1] + 1) % cfg.n_vocab, 7], list(range(-1, len(tk) - 1)) + [-1, len(tk)]

        got, passes = m.generate_speculative(emb, draft, steps)
        assert passes < steps - 1
        logits, _ = m.prefill(emb)
        for i in range(steps):
            if i:
                logits, _ = m.decode_step(got[:, i - 1], T + i - 1)
            below = logits.max(1) - logits[np.arange(n), got[:, i]]
            assert (below <= bound * np.abs(logits).max(1)).all(), i
    finally:
        m.close()
