"""Weights that the operators copy (they are kept contiguous) are there before a call on the handle's stream can read them: the
copy is issued on torch's current stream, which the handle's does not follow. Host only: the copies' stream is a stand-in."""
import pytest
import torch

from tsn import block_ops


class Host:
    """A handle whose tensors lie in host memory."""
    ordinal = -1


@pytest.fixture
def waited(monkeypatch):
    done = []

    class Stream:
        def synchronize(self):
            done.append("synchronized")

    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: Stream())
    return done


def test_a_copied_weight_is_waited_for(waited):
    table = torch.arange(32.0).view(16, 2)
    t = block_ops._weights(Host, "w", table[:, 1], (16,))
    assert t.is_contiguous() and torch.equal(t, table[:, 1]) and waited == ["synchronized"]


def test_a_contiguous_weight_is_taken_as_it_is(waited):
    w = torch.arange(16.0)
    assert block_ops._weights(Host, "w", w, (16,)) is w and waited == []
    assert block_ops._weights(Host, "w", None, (16,)) is None and waited == []
