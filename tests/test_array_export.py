"""CPU: device arrays that are handed to others by their array interface.  The library is a stand-in that records its
calls, so no address here is ever followed."""
import gc

import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd import _hip, xparray
from pytortto_amd.xparray import hiparray

F = tt.nn.functional


class _Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def function(*args):
            self.calls.append(name)
            if name == 'tt_malloc':
                args[0]._obj.value = 4096 * (1 + len(self.calls))
            return 0
        return function

    def since(self, *ignored):
        names = [n for n in self.calls if n not in ignored]
        self.calls.clear()
        return names


@pytest.fixture
def library(monkeypatch):
    stand_in = _Library()
    monkeypatch.setattr(_hip, '_lib', stand_in)
    monkeypatch.setattr(_hip, '_ready', True)
    monkeypatch.setattr(_hip, '_pending', None)
    monkeypatch.setattr(_hip, '_earlier', None)
    monkeypatch.setattr(xparray, '_one', None)
    yield stand_in
    _hip.take_pending()
    gc.collect()


def test_what_is_parked_runs_first(library):
    """A parked BatchNorm updates its running statistics when it runs."""
    norm = tt.nn.BatchNorm2d(3)
    norm.cuda()
    x = tt.Tensor(hiparray(np.ones((2, 3, 4, 4), np.float32)))
    y = norm(x)
    library.since()
    norm.running_mean.data.__cuda_array_interface__
    assert [n for n in library.since() if 'bn' in n], 'the array is handed out before its update was launched'
    del y
