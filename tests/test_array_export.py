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
        self.calls, self.blocks = [], 0

    def __getattr__(self, name):
        def function(*args):
            self.calls.append(name)
            if name == 'tt_malloc':
                self.blocks += 1
                args[0]._obj.value = 4096 * self.blocks
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


def _handed_out(array):
    return array.__cuda_array_interface__['data'][0]


def test_a_shared_array_is_handed_out_as_a_copy(library):
    """Others write past what the library notes of shared memory: neither holder may see the other's values change."""
    a = hiparray(np.ones(3, np.float32))
    b, c = a.alias(), a.lent()
    at = a.ptr
    library.since()
    assert _handed_out(b) not in (0, at) and library.since() == ['tt_malloc', 'tt_memcpy_d2d']
    assert _handed_out(b) == b.ptr and library.since() == []
    assert a.ptr == at and c.ptr == at
    assert _handed_out(c) not in (at, b.ptr) and library.since() == ['tt_malloc', 'tt_memcpy_d2d']


def test_loans_of_an_array_are_settled_before_it_is_handed_out(library):
    a = hiparray(np.ones(3, np.float32))
    loan = a.lent()
    library.since()
    at = a.ptr
    assert _handed_out(a) == at and library.since() == ['tt_malloc', 'tt_memcpy_d2d'] and loan.ptr != at


def test_the_ones_of_backward_passes_are_handed_out_as_copies(library):
    first = xparray.one(0)
    assert _handed_out(first) != xparray._one.ptr and not xparray.is_one(first) and xparray.is_one(xparray.one(1))


@pytest.mark.parametrize('share', ['alias', 'lent'])
def test_what_was_handed_out_is_not_shared_afterwards(library, share):
    """... and so never moves: its receiver keeps the array, which keeps the block."""
    first, _ = hiparray.carve(((3,), np.float32), ((5,), np.float32))
    for a in (hiparray(np.ones(3, np.float32)), first, hiparray(np.ones((3, 1), np.float32)).reshape(3)):
        at = _handed_out(a)
        other = getattr(a, share)()
        assert other.ptr != at and not a._shared
        a += other
        assert a.ptr == at
        np.testing.assert_array_equal(a.shape, other.shape)


def test_a_gradient_that_was_handed_out(library):
    x = tt.Tensor(hiparray(np.ones(3, np.float32)), requires_grad=True)
    g = tt.Tensor(hiparray(np.ones(3, np.float32)))
    at = _handed_out(g.data)
    x.backward(g)
    assert x.grad.ptr != at
    kept = _handed_out(x.grad)
    x.backward(g)
    assert x.grad.ptr == kept and g.data.ptr == at


def test_blocks_of_arrays_that_were_handed_out_wait_for_others(library):
    """... whoever holds the array last, also where it is a part of a block."""
    freed = ('tt_malloc', 'tt_memcpy_h2d', 'tt_memcpy_d2d')
    a, b = hiparray(np.ones(3, np.float32)), hiparray(np.ones(3, np.float32))
    view = a.reshape(1, 3)
    view.__cuda_array_interface__
    del view
    library.since()
    del b
    assert library.since(*freed) == ['tt_free']
    del a
    assert library.since(*freed) == ['tt_free_exported']
    parts = hiparray.carve(((3,), np.float32), ((5,), np.float32))
    parts[1].__cuda_array_interface__
    del parts[1]
    assert library.since(*freed) == []
    del parts
    assert library.since(*freed) == ['tt_free_exported']


def test_memory_of_others_that_is_handed_out_again(library):
    class Foreign:
        __cuda_array_interface__ = {'shape': (3,), 'typestr': '<f4', 'data': (1 << 20, False), 'version': 3}
    a = hiparray.borrow(Foreign())
    assert _handed_out(a) == 1 << 20
    del a
    assert library.since() == []


def test_the_stream_is_named(library, monkeypatch):
    monkeypatch.setattr(_hip, '_stream', None)

    def tt_get_stream(handle):
        handle._obj.value = 77
        library.calls.append('tt_get_stream')
        return 0

    library.tt_get_stream = tt_get_stream
    a = hiparray(np.ones(3, np.float32))
    about = a.__cuda_array_interface__
    assert about['stream'] == 77 and about['version'] == 3 and a.__cuda_array_interface__['stream'] == 77
    assert library.calls.count('tt_get_stream') == 1
    monkeypatch.setattr(_hip, '_stream', None)
    monkeypatch.setattr(_hip, '_ready', False)      # nothing has been launched: there is no stream to wait for
    assert _hip.stream() is None


def test_read_only_memory_of_others_is_not_written(library):
    class Foreign:
        def __init__(self, read_only):
            self.__cuda_array_interface__ = {'shape': (3,), 'typestr': '<f4', 'data': (1 << 20, read_only), 'version': 3}

    for write in (lambda a: a.fill(1.0), lambda a: a.__iadd__(1.0), lambda a: a.set(np.ones(3)), lambda a: a.own(),
                  lambda a: a.__cuda_array_interface__):
        a, b = hiparray.borrow(Foreign(True)), hiparray.borrow(Foreign(False))
        assert a.ptr == b.ptr == 1 << 20
        library.since()
        write(a)
        assert a.ptr != 1 << 20 and library.since()[:2] == ['tt_malloc', 'tt_memcpy_d2d']
        write(b)
        assert b.ptr == 1 << 20 and 'tt_memcpy_d2d' not in library.since()
