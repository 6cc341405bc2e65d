"""Trees of drafted tokens from a text, and what the Python side checks before anything reaches the device (no GPU)."""
import pytest

from qraf_amd import engine as eng
from qraf_amd._lib import SamplingParams


@pytest.mark.parametrize("history,depth,width,ngram,most,want", [
    # the latest occurrence of the last three tokens first; what the continuations share is one node
    ([1, 2, 3, 4, 1, 2, 3, 5, 9, 1, 2, 3], 4, 3, 3, 63, ([5, 9, 1, 2, 4, 1, 2, 3], [0, 1, 2, 3, 0, 5, 6, 7])),
    ([1, 2, 3, 4, 8, 1, 2, 3, 4, 9, 1, 2, 3], 2, 3, 3, 63, ([4, 9, 8], [0, 1, 1])),
    ([1, 2, 3, 4, 1, 2, 3, 5, 9, 1, 2, 3], 4, 1, 3, 63, ([5, 9, 1, 2], [0, 1, 2, 3])),
    ([7, 7, 7, 7], 2, 8, 2, 3, ([7, 7], [0, 1])),
    ([5, 1, 6, 1, 7, 1], 1, 8, 3, 63, ([7, 6], [0, 0])),  # no three, no two: one
    ([5, 1, 6, 1, 7, 1], 1, 8, 3, 1, ([7], [0])),
    ([1, 2], 4, 3, 3, 63, ([], [])),
    ([1], 4, 3, 3, 63, ([], [])),
    ([1, 1], 0, 3, 3, 63, ([], [])),
    ([1, 1, 1], 3, 3, 3, 0, ([], [])),
])
def test_trees_of_a_text(history, depth, width, ngram, most, want):
    assert eng._TreeDrafter(None, depth, width, ngram).propose(history, depth, most) == want


def bare():
    e = eng.Engine.__new__(eng.Engine)
    e.h, e.vocab, e.max_batch = None, 100, 16
    return e


def test_step_tree_takes_an_entry_for_each_row():
    e = bare()
    for bad in (dict(tokens=[1]), dict(parents=[-1]), dict(positions=[0]), dict(want_logits=[1])):
        with pytest.raises(ValueError):
            e.step_tree(**{**dict(seq_ids=[0, 0], tokens=[1, 2], parents=[-1, 0], positions=[0, 0]), **bad})


def test_accept_tree_takes_a_history_and_a_draw_for_each_row():
    e = bare()
    e._trees = [2, 1]
    for bad in (dict(recent=[[1], [2]]), dict(uniforms=[0.5] * 4)):
        with pytest.raises(ValueError):
            e.accept_tree(SamplingParams(1.0, 0, 1.0, 1.2), **bad)


def test_logprobs_takes_a_token_for_each_row():
    e = bare()
    for bad in (dict(tokens=[1, 2], rows=3), dict(rows=-1), dict(top=-1)):
        with pytest.raises(ValueError):
            e.logprobs(**bad)


def test_generate_tree_and_score_refuse():
    class Model:
        engine = bare()
    g = eng.InferenceEngine(Model)
    for bad in (dict(prompt_tokens=[]), dict(depth=4, width=4), dict(depth=-1), dict(width=0), dict(depth=64, width=1)):
        with pytest.raises(ValueError):
            g.generate_tree(**{**dict(prompt_tokens=[1]), **bad})
    for text in ([], [1]):
        with pytest.raises(ValueError):
            g.score(text)
