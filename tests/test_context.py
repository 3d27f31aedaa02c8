"""Contexts shared by threads, without a GPU: a stub stands in for the library and for torch's current stream."""
import ctypes
import threading
import time

import pytest
import torch

from compression_amd import _lib


class StubLib:
    """The part of libmpc that a Context uses; every call leaves the interpreter to other threads in its middle, as a call
    through ctypes may."""

    def __init__(self):
        self.stream, self.error, self.created, self.ran_on = None, b"", 0, []

    def mpc_create(self, index, stream, out):
        time.sleep(0.001)
        self.created += 1
        out._obj.value, self.stream = 1, stream.value
        return 0

    def mpc_set_stream(self, handle, stream):
        self.stream = stream.value
        time.sleep(0.001)
        return 0

    def mpc_profile_mark(self, handle, who):
        time.sleep(0.0005)
        self.ran_on.append((who, self.stream))
        return 0

    def mpc_synchronize(self, handle, who):               # (fails, with a text of the caller's)
        self.error = b"for %d" % who
        time.sleep(0.0005)
        return -1

    def mpc_last_error(self, handle):
        return self.error

    def mpc_destroy(self, handle):
        return 0


@pytest.fixture
def stub(monkeypatch):
    lib, current = StubLib(), threading.local()
    monkeypatch.setattr(_lib, "load", lambda: lib)
    monkeypatch.setattr(_lib, "_contexts", {})
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: getattr(current, "stream", 0), raising=False)
    lib.current = current
    return lib


def in_threads(n, work):
    failed = []

    def guarded(i):
        try:
            work(i)
        except BaseException as e:                        # noqa: BLE001 (reported below)
            failed.append(e)
    threads = [threading.Thread(target=guarded, args=(i,)) for i in range(1, n + 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_calls_of_several_threads_run_on_their_own_streams(stub):
    def work(i):
        stub.current.stream = 100 + i
        for _ in range(30):
            _lib.context_at(0).call("mpc_profile_mark", i)
    in_threads(4, work)
    assert len(stub.ran_on) == 120 and all(stream == 100 + who for who, stream in stub.ran_on)
    assert stub.created == 1
    # nothing of it lasts: a call by this thread runs on this thread's stream
    _lib.context_at(0).call("mpc_profile_mark", -100)
    assert stub.ran_on[-1] in ((-100, 0), (-100, None))


def test_errors_are_those_of_the_call(stub):
    def work(i):
        for _ in range(20):
            with pytest.raises(_lib.MpcError, match=f"for {i}$"):
                _lib.context_at(0).call("mpc_synchronize", i)
    in_threads(4, work)


def test_the_stream_is_looked_up_at_the_call(stub):
    ctx = _lib.context_at(0)
    for s in (7, 8, 8, 7):
        stub.current.stream = s
        ctx.call("mpc_profile_mark", s)
    assert stub.ran_on == [(7, 7), (8, 8), (8, 8), (7, 7)]


def test_a_stream_given_by_hand(stub):
    """A context of one's own stays on the stream it was given, through either way of giving it; a shared one refuses."""
    own = _lib.Context(0, 5)
    own.call("mpc_profile_mark", 0)
    own.set_stream(6)
    own.call("mpc_profile_mark", 1)
    own.call("mpc_set_stream", ctypes.c_void_p(9))
    own.call("mpc_profile_mark", 2)
    assert stub.ran_on == [(0, 5), (1, 6), (2, 9)] and own.stream_handle == 9
    for give in (lambda c: c.set_stream(9), lambda c: c.call("mpc_set_stream", 9)):
        with pytest.raises(_lib.MpcError, match="current stream"):
            give(_lib.context_at(0))
