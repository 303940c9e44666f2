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
