"""QwenModel.generate_speculative's own part, how it makes and keeps the trees: over a stand-in for the
decoder that checks what the entry point requires and forgets what it leaves undefined."""
import numpy as np
import pytest

from openasr_b200 import backend as bk
from openasr_b200 import models as om

VOCAB = 50


def greedy(context):
    """the model's choice after a list of tokens"""
    x = 17
    for t in context:
        x = (x * 31 + int(t) + 7) % 10007
    return x % VOCAB


def greedy_tokens(s, T, n):
    """what generate() would give for sequence s, whose prompt is T times 1000 + s"""
    c = [1000 + s] * T
    for _ in range(n):
        c.append(greedy(c))
    return c[T:]


class Decoder(om.QwenModel):
    def __init__(self, max_pos, max_prefill=64, max_batch=4):  # noqa: no device, no weights
        self.cfg = om.QWEN3_ASR_0_6B.replace(max_pos=max_pos, max_prefill=max_prefill, max_batch=max_batch)
        self.widths = []

    def prefill(self, emb):
        self.cache = [[1000 + s] * emb.shape[1] + [None] * (self.cfg.max_pos - emb.shape[1]) for s in range(emb.shape[0])]
        return None, np.array([greedy(c[:emb.shape[1]]) for c in self.cache], np.int32)

    def verify_tree(self, tokens, parents, pos):
        tokens, parents = np.asarray(tokens), np.asarray(parents)
        S, n = tokens.shape
        if S * n > self.cfg.max_batch * self.cfg.max_prefill or n > 1024:
            raise bk.UnsupportedInputs(bk.STATUS_FAILED, "verify_tree: bad arguments")
        self.widths.append(n)
        path, acc, nxt = np.full((S, n), -1, np.int32), np.zeros(S, np.int32), np.zeros(S, np.int32)
        for s in range(S):
            p, row = int(pos[s]), self.cache[s]
            assert parents[s, 0] == -1 and (parents[s] < np.arange(n)).all() and p + n <= self.cfg.max_pos
            assert None not in row[:p]
            walk = [0]
            while True:
                choice = greedy(row[:p] + [tokens[s, j] for j in walk])
                kids = [j for j in range(walk[-1] + 1, n) if parents[s, j] == walk[-1] and tokens[s, j] == choice]
                if not kids:
                    break
                walk.append(kids[0])
            path[s, :len(walk)], acc[s], nxt[s] = walk, len(walk), choice
            row[p:p + n] = [int(tokens[s, j]) for j in walk] + [None] * (n - len(walk))
        return path, acc, nxt


def drafter(T, length):
    """length(s, made) right tokens after those made so far"""
    def draft(s, tokens):
        k = length(s, len(tokens))
        return greedy_tokens(s, T, len(tokens) + k)[len(tokens):], list(range(-1, k - 1))
    return draft


@pytest.mark.parametrize("n_new", [1, 2, 11, 22])
@pytest.mark.parametrize("quick", [1, 3, 9])
def test_sequences_that_end_early_leave_the_others_their_room(n_new, quick):
    """one sequence accepts long drafts, past its last token and up to the context's end, the others none or
    two at a time: all get what generate() would give them, with prompt and tokens filling the context"""
    T, n = 10, 3
    m = Decoder(T + n_new)
    got, passes = m.generate_speculative(np.zeros((n, T, 4), np.float32), drafter(T, lambda s, made: (quick, 0, 2)[s]), n_new)
    assert got.tolist() == [greedy_tokens(s, T, n_new) for s in range(n)]
    assert passes == len(m.widths) == n_new - 1
    for s in range(n):  # and the caches hold the tokens, also of the one that ended first
        assert m.cache[s][T:T + n_new - 1] == got[s, :-1].tolist()


def test_a_sequence_that_ended_does_not_narrow_the_others_trees():
    T, n_new = 6, 40
    m = Decoder(T + n_new)
    m.generate_speculative(np.zeros((2, T, 4), np.float32), drafter(T, lambda s, made: 39 if s == 0 else 2 if made < 20 else 0), n_new)
    assert m.widths[0] == 40 and all(w == 3 for w in m.widths[1:7])


def test_the_context_is_full_only_for_a_sequence_that_goes_on():
    m = Decoder(20)
    with pytest.raises(bk.UnsupportedInputs, match="context is full"):
        m.generate_speculative(np.zeros((1, 10, 4), np.float32), drafter(10, lambda s, made: 0), 30)


@pytest.mark.parametrize("max_prefill,max_batch,n,most", [(8, 2, 2, 8), (5, 3, 2, 7), (1, 4, 3, 1), (2000, 2, 1, 1024)])
def test_drafts_wider_than_a_pass_are_cut(max_prefill, max_batch, n, most):
    """a pass takes max_batch * max_prefill nodes in all and 1024 of a sequence; the rest of a draft waits"""
    T, n_new = 1, 1100
    m = Decoder(4000, max_prefill, max_batch)
    if most < 100:
        n_new = 30
    draft = drafter(T, lambda s, made: n_new)
    got, passes = m.generate_speculative(np.zeros((n, T, 4), np.float32), draft, n_new)
    assert got.tolist() == [greedy_tokens(s, T, n_new) for s in range(n)]
    assert max(m.widths) == most and passes == -(-(n_new - 1) // most)
