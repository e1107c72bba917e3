"""Each thread has contexts of its own for the row operators, and threads that have
ended leave theirs to the next (a stand-in for the context: no GPU here)."""
import threading

import pytest

from vauss_b200 import ops


class FakeContext:
    made = 0

    def __init__(self, device):
        self.device = device
        FakeContext.made += 1

    def bind(self):
        self.stream = ops._raw_stream(self.device)
        return self

    def check(self, status):
        ops.N.check(None, status)


@pytest.fixture
def fake(monkeypatch):
    monkeypatch.setattr(ops, "Context", FakeContext)
    monkeypatch.setattr(ops, "_contexts", {})
    monkeypatch.setattr(ops, "_idle_contexts", [], raising=False)
    monkeypatch.setattr(FakeContext, "made", 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    if hasattr(ops, "_RowContexts"):
        monkeypatch.setattr(ops, "_row_contexts", ops._RowContexts())


def _in_threads(n, fn):
    """fn() of n threads that are all alive at once."""
    got, gate = [], threading.Barrier(n)

    def work():
        got.append(fn())
        gate.wait(10)

    threads = [threading.Thread(target=work) for _ in range(n)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    return got


def test_threads_do_not_share_a_context(fake):
    mine = ops._row_context(0)
    assert ops._row_context(0) is mine and ops._row_context(1) is not mine
    others = _in_threads(4, lambda: (ops._row_context(0), ops._row_context(0)))
    assert all(a is b for a, b in others)
    assert len({id(mine)} | {id(a) for a, _ in others}) == 5
    assert all(a.device == 0 for a, _ in others)


def test_threads_that_ended_leave_their_contexts(fake):
    first = _in_threads(3, lambda: ops._row_context(0))
    assert FakeContext.made == 3
    again = _in_threads(3, lambda: ops._row_context(0))
    assert FakeContext.made == 3 and {id(c) for c in again} == {id(c) for c in first}
    _in_threads(1, lambda: ops._row_context(2))  # no context of another device is taken
    assert FakeContext.made == 4


def test_a_wait_that_ran_out_is_reported(fake, monkeypatch):
    """check_device asks the thread's context of the row operators too, and raises what it reports."""
    asked = []

    class Lib:
        def vs_ctx_check(self, h):
            asked.append(h)
            return 4 if h == "row" else 0

    row, other = ops._row_context(0), FakeContext(0)
    monkeypatch.setattr(FakeContext, "lib", Lib(), raising=False)
    row.h, other.h = "row", "other"
    ops._contexts[0] = other
    with pytest.raises(ops.N.VsError, match="TIMEOUT"):
        ops.check_device(0)
    assert asked == ["other", "row"]
