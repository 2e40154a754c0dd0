"""The call that launches on a tensor's own device: which library it goes through and what is current meanwhile."""
import contextlib
import ctypes

import pytest


class _Tensor:
    def __init__(self, index):
        self.index = index

    def get_device(self):
        return self.index


@pytest.fixture
def launches(monkeypatch):
    """What the library was called with, and the device that was current, for two devices that are not there."""
    from nlearn_amd import _lib

    current, seen = [0], []

    class Cuda:
        @staticmethod
        @contextlib.contextmanager
        def device(index):
            before, current[0] = current[0], index
            try:
                yield
            finally:
                current[0] = before

    class Library:
        @staticmethod
        def nl_fake(*args):
            seen.append((current[0], *args))
            return _lib.NL_OK

    monkeypatch.setattr(_lib, "_cuda", (Cuda, lambda: current[0], lambda index: 1000 + index))
    monkeypatch.setattr(_lib, "_lib", Library)
    return seen


def test_call_on_makes_the_tensors_device_current(launches):
    from nlearn_amd import _lib

    _lib.call_on(_Tensor(0), "nl_fake", 7)
    _lib.call_on(_Tensor(1), "nl_fake", 8)
    assert launches == [(0, 1000, 7), (1, 1001, 8)]


def test_call_on_with_a_probe(launches, monkeypatch):
    from nlearn_amd import _lib

    probed = []
    monkeypatch.setattr(_lib, "_probe", lambda name, args: probed.append((name, args)))
    # without the fakes' streams a probe's call looks the stream up here
    monkeypatch.setattr(_lib, "stream_of", lambda t: 1000 + t.get_device())
    _lib.call_on(_Tensor(1), "nl_fake", 9)
    assert launches == [(1, 1001, 9)] and probed == [("nl_fake", (1001, 9))]


def test_entry_points_leave_pythons_lock():
    """A launch can wait for room in the queue: other Python threads go on meanwhile."""
    from nlearn_amd import _lib

    L = _lib.load()
    keeps_lock = ctypes.PyDLL(str(_lib.LIB_PATH)).nl_last_error._flags_ & ~L.nl_last_error._flags_
    assert keeps_lock and not any(getattr(L, name)._flags_ & keeps_lock for name in _lib.EXPORTED)
    assert not any(isinstance(v, ctypes.PyDLL) for v in vars(_lib).values())
