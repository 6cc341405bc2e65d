"""What the engine's Python side checks and gives back before anything reaches the device (no GPU)."""
import pytest

from qraf_amd import engine as eng
from qraf_amd._lib import SamplingParams


@pytest.mark.parametrize("lists,rows", [([[1]], 2), ([[1], [2], [3]], 2), ([], 1)])
def test_probs_takes_a_history_for_each_row(lists, rows):
    """Fewer histories than rows would be read past their counts."""
    e = eng.Engine.__new__(eng.Engine)
    e.h = None
    with pytest.raises(ValueError):
        e.probs(SamplingParams(1.0, 0, 1.0, 1.2), 4096, lists, rows=rows)


def test_a_drafter_that_cannot_be_made_keeps_no_sequence(monkeypatch):
    class Model:
        class engine:
            held = []

            @classmethod
            def seq_create(cls):
                cls.held.append(7)
                return 7

            @classmethod
            def seq_release(cls, seq):
                cls.held.remove(seq)

    def none(size):
        raise MemoryError(size)
    from qraf_amd import backend
    monkeypatch.setattr(backend, "DeviceBuffer", none)
    with pytest.raises(MemoryError):
        eng._Drafter(Model, 100, 4, None, object(), 3)
    assert Model.engine.held == []
