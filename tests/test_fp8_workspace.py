"""The scratch that the E4M3 and balance forms hold, and what a graph keeps of it: on the host, with buffers that
are only counted."""
import gc
import weakref

import pytest
import torch

from moonshine_b200 import fp8


class Buffer:
    def __init__(self, need, device):
        self.need, self.device = need, device

    def record_stream(self, stream):
        pass


@pytest.fixture
def capturing(monkeypatch):
    """A list whose last entry says whether the current stream captures."""
    state = [False]
    monkeypatch.setattr(torch, "empty", lambda need, dtype, device: Buffer(need, device))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: None)
    monkeypatch.setattr(fp8, "_capturing", lambda: state[-1])
    return state


def alive(ref):
    gc.collect()
    return ref() is not None


def test_scratch_of_a_captured_call_outlives_larger_calls(capturing):
    ws = fp8._Workspace(lambda tokens: 100 * tokens)
    ws.of(50, "gpu")                             # what warming up allocates
    capturing.append(True)
    first = weakref.ref(ws.of(50, "gpu"))
    second = weakref.ref(ws.of(60, "gpu"))       # a call that grows it within the capture
    capturing.append(False)
    third = weakref.ref(ws.of(4096, "gpu"))
    assert first() is not second() and alive(first) and alive(second)
    ws.of(8192, "gpu")
    assert alive(first) and alive(second)
    assert not alive(third)                      # no graph has this one
    capturing.append(True)
    fourth = weakref.ref(ws.of(10, "gpu"))       # a second graph has the largest
    assert ws.of(20, "gpu") is fourth()
    capturing.append(False)
    ws.of(10000, "gpu")
    assert alive(fourth)
    assert len(ws._captured) == 3
    del ws
    assert not (alive(first) or alive(second) or alive(fourth))


def test_scratch_of_other_calls_is_given_back(capturing):
    ws = fp8._Workspace(lambda tokens, sequences: tokens * sequences)
    first = weakref.ref(ws.of(50, 2, "gpu"))
    assert ws.of(40, 1, "gpu") is first() and ws.bytes == 100
    second = weakref.ref(ws.of(40, 3, "gpu"))    # the larger of each size
    assert not alive(first) and ws.bytes == 150
    ws.of(50, 3, "other")
    assert not alive(second)
