"""PagedDecoder says so when an operator does not take a call (no GPU: the session's procs are replaced)."""
import pytest

from bybylang_amd import _abi, gpubackend as g
from bybylang_amd.paged_decoder import PagedDecoder


@pytest.mark.parametrize("proc,call", [("sessionCacheFork", lambda d: d.fork([0], [1])), ("sessionCacheFree", lambda d: d.free([1])),
                                       ("sessionCacheCompact", lambda d: d.compact())])
def test_a_call_that_is_not_taken_raises(monkeypatch, proc, call):
    d = PagedDecoder.__new__(PagedDecoder)
    d.pool = d.some = d.others = None
    monkeypatch.setattr(d, "_set", lambda handle, values: None, raising=False)
    monkeypatch.setattr(g, proc, lambda *a: True)
    call(d)
    monkeypatch.setattr(g, proc, lambda *a: False)
    with pytest.raises(_abi.HipUnsupported, match="does not take"):
        call(d)


def test_forks_without_a_parent_each_are_refused(monkeypatch):
    """The call would have taken the parents of the fork before it."""
    d = PagedDecoder.__new__(PagedDecoder)
    d.pool = d.some = d.others = None
    monkeypatch.setattr(d, "_set", lambda handle, values: None, raising=False)
    monkeypatch.setattr(g, "sessionCacheFork", lambda *a: pytest.fail("forked"))
    for parents, rows in (([0], [1, 2]), ([0, 3], [1]), ([], [1])):
        with pytest.raises(ValueError, match="forks of"):
            d.fork(parents, rows)


def test_a_step_without_rows_does_nothing(monkeypatch):
    d = PagedDecoder.__new__(PagedDecoder)
    d.rows, d.width, d.pool, d.all_rows, d.add, d.slots = 0, 8, None, None, None, 2
    for proc in ("sessionCacheGrow", "sessionNormBlock", "sessionMatmulQ4"):
        monkeypatch.setattr(g, proc, lambda *a: pytest.fail("queued"))
    d.encode()


def test_a_step_that_cannot_be_recorded_leaves_no_recording_open(monkeypatch):
    d = PagedDecoder.__new__(PagedDecoder)
    calls = []

    def encode():
        raise _abi.HipUnsupported("not taken")
    monkeypatch.setattr(d, "encode", encode, raising=False)
    monkeypatch.setattr(g, "sessionBeginRecording", lambda b: True)
    monkeypatch.setattr(g, "sessionRecoverQueue", lambda b: calls.append("recovered"))
    monkeypatch.setattr(g, "sessionEnd", lambda b: pytest.fail("kept"))
    with pytest.raises(_abi.HipUnsupported):
        d.record()
    assert calls == ["recovered"]
