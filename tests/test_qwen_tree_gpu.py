"""Drafted trees through the Qwen3-ASR decoder: a verification pass accepts what greedy
decoding would have produced and leaves the caches where decode steps would have.

The tree attention sums on the tensor cores, a decode step in its own order, and the int8
activations carry the last bits on: as for the tensor-core prompt pass (test_qwen_gpu.py),
logits agree to 2e-2 of the largest.  So a token is right when its logit in a decode step
over the same tokens is within that of the best, and has to be the greedy one where no
other comes that near."""
import numpy as np
import pytest

import openasr_b200 as ob
from openasr_b200 import models as om

pytestmark = pytest.mark.gpu

BOUND = 2e-2  # |logit difference| / max |logit|, as test_qwen_gpu.py has it for tensor-core attention
MID = om.QWEN3_ASR_0_6B.replace(n_layers=2, n_vocab=4096, max_pos=256, max_prefill=64, max_batch=4)


@pytest.fixture(scope="module")
def model(gpu_backend):
    m = om.QwenModel(gpu_backend, MID, om.qwen_synthetic_pack(MID, seed=0x0A5A0003))
    yield m
    m.close()


@pytest.fixture(scope="module")
def prompt():
    return om.qwen_synthetic_prefix(0x0A5A3000, 3, 30, 1024)


@pytest.fixture(scope="module")
def serial(model, prompt):
    return model.generate(prompt, n_new=40)


def slack(model, prompt, tokens):
    """[n_seq][n] how far each token's logit is below the best of the step, over max |logit|, in
    teacher-forced decode steps, and [n_seq][n] whether any other token comes within BOUND"""
    out, close = [], []
    logits, _ = model.prefill(prompt)
    for i in range(tokens.shape[1]):
        if i:
            logits, _ = model.decode_step(tokens[:, i - 1], prompt.shape[1] + i - 1)
        top = np.sort(logits, 1)
        size = np.abs(logits).max(1)
        out.append((top[:, -1] - logits[np.arange(len(tokens)), tokens[:, i]]) / size)
        close.append((top[:, -1] - top[:, -2]) / size <= BOUND)
    return np.stack(out, 1), np.stack(close, 1)


def test_a_tree_with_the_greedy_branch_is_accepted_to_its_end(model, prompt, serial):
    _, first = model.prefill(prompt)
    assert np.array_equal(first, serial[:, 0])
    # node 0, wrong nodes, and the greedy continuation scattered among them
    n, right = 12, [2, 5, 6, 9, 11]
    tokens, parents = np.zeros((3, n), np.int32), np.zeros((3, n), np.int32)
    for s in range(3):
        up = 0
        parents[s, 0], tokens[s, 0] = -1, first[s]
        for i in range(1, n):
            k = right.index(i) if i in right else None
            parents[s, i] = up if k is not None else max(0, i - 2)
            tokens[s, i] = serial[s, 1 + k] if k is not None else (serial[s, 20] + 7 * i) % MID.n_vocab
            up = i if k is not None else up
    path, acc, nxt = model.verify_tree(tokens, parents, [30, 30, 30])
    rows = [model.read_kv(layer, s, 30 + acc[s]) for s in range(3) for layer in range(2)]
    got = [np.concatenate([tokens[s, path[s, :acc[s]]], nxt[s:s + 1]]) for s in range(3)]
    _, close = slack(model, prompt, serial[:, :7])
    for s in range(3):
        assert path[s, :acc[s]].tolist() == ([0] + right)[:acc[s]] and (path[s, acc[s]:] == -1).all()
        assert acc[s] == 6 or close[s, acc[s]], "a step without a near tie must go on"
        assert acc[s] < 6 or nxt[s] == serial[s, 6] or close[s, 6]
        below, _ = slack(model, prompt[s:s + 1], got[s][None])
        assert (below <= BOUND).all()
        # the accepted rows are in place; layer 0 sees no attention before its K and V: the same
        # bits as decode steps write (slack() has just run them)
        for layer in range(2):
            for mine, want in zip(rows[2 * s + layer], model.read_kv(layer, 0, 30 + acc[s])):
                if layer == 0:
                    assert np.array_equal(mine.view(np.uint16), want.view(np.uint16))
                else:
                    assert np.abs(mine.astype(np.float32) - want.astype(np.float32)).max() <= BOUND * np.abs(want).max()
    assert (acc == 6).sum() >= 1


def test_decoding_goes_on_after_an_accepted_tree(model, prompt, serial):
    """the state after a pass is the state that decode steps over the same tokens leave"""
    s = 0
    _, first = model.prefill(prompt[:1])
    path, acc, nxt = model.verify_tree([[first[0], serial[s, 1], 5]], [[-1, 0, 1]], [30])
    out = [first[0], serial[s, 1]][:acc[0]] + [nxt[0]]
    at = 30 + acc[0]
    for i in range(8):
        out.append(model.decode_step(out[-1:], at + i)[1][0])
    below, _ = slack(model, prompt[:1], np.array([out], np.int32))
    assert (below <= BOUND).all()


def test_generate_speculative_is_greedy_decoding(model, prompt, serial):
    """drafts of any quality: the true continuation with a mistake at every fifth token, next to a
    branch of nonsense; sequences accept different numbers and end at different times"""
    def draft(s, tokens):
        at, nodes, parents = len(tokens), [], []
        for k in range(min(6, 39 - at) + 1 - s % 2):
            t = int(serial[s, min(at + k, 39)])
            nodes.append(t if (at + k) % 5 else (t + 1) % MID.n_vocab)
            parents.append(-1 if k == 0 else k - 1)
        for k in range(3):
            nodes.append((17 * at + k) % MID.n_vocab)
            parents.append(-1 if k == 0 else len(nodes) - 2)
        return nodes, parents

    got, passes = model.generate_speculative(prompt, draft, n_new=40)
    below, _ = slack(model, prompt, got)
    assert got.shape == (3, 40) and (below <= BOUND).all()
    assert passes < 39, "more than a token per pass"
    got, passes = model.generate_speculative(prompt, lambda s, t: ([], []), n_new=12)
    below, _ = slack(model, prompt, got)
    assert (below <= BOUND).all() and passes == 11


def test_verify_tree_refusals(model, prompt):
    model.prefill(prompt)
    ok = dict(tokens=np.zeros((2, 3)), parents=np.array([[-1, 0, 1]] * 2), pos=[30, 30])
    for kw in (dict(tokens=np.zeros((2, 4))), dict(parents=np.array([[-1, 0, 2]] * 2)), dict(parents=np.array([[0, 0, 1]] * 2)),
               dict(tokens=np.full((2, 3), MID.n_vocab)), dict(tokens=np.full((2, 3), -1)), dict(pos=[30, 254]), dict(pos=[-1, 3]),
               dict(pos=[30]), dict(tokens=np.zeros((5, 3)), parents=np.array([[-1, 0, 1]] * 5), pos=[30] * 5),
               dict(tokens=np.zeros((4, 65)), parents=np.array([list(range(-1, 64))] * 4), pos=[30] * 4)):
        with pytest.raises(ob.backend.UnsupportedInputs):
            model.verify_tree(*{**ok, **kw}.values())
    model.verify_tree(*ok.values())
