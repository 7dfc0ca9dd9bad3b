"""CPU: what holds the arrays of the operators over a vocabulary.  The library is a stand-in: nothing is computed."""
import gc
import weakref

import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd import _hip
from pytortto_amd.xparray import hiparray

F = tt.nn.functional


class _Library:
    blocks = 0

    def __getattr__(self, name):
        def function(*args):
            if name == 'tt_malloc':
                self.blocks += 1
                args[0]._obj.value = 4096 * self.blocks
            return 0
        return function


@pytest.fixture
def library(monkeypatch):
    monkeypatch.setattr(_hip, '_lib', _Library())
    monkeypatch.setattr(_hip, '_ready', True)
    monkeypatch.setattr(_hip, '_pending', None)
    yield
    gc.collect()


def _tensor(shape, dtype=np.float32, grad=False):
    return tt.Tensor(hiparray(np.zeros(shape, dtype)), dtype=dtype, requires_grad=grad)


@pytest.mark.parametrize('call', [
    lambda x: F.layer_norm(x, 5),
    lambda x: F.token_log_prob(x, _tensor(3, np.int64)),
    lambda x: F.token_log_prob(x, _tensor(3, np.int64), top=2),
    lambda x: F.distill_loss(x, _tensor((3, 2)), _tensor((3, 2), np.int64)),
])
def test_a_call_that_is_never_run_backward_leaves_nothing(library, call):
    """The logits go with the last result, not when the cycle collector comes."""
    gc.collect()
    gc.disable()
    try:
        x = _tensor((3, 5), grad=True)
        held = weakref.ref(x.data)
        result = call(x)
        del x
        assert held() is not None
        del result
        assert held() is None
    finally:
        gc.enable()


def test_a_result_that_was_changed_in_place_is_still_noticed(library):
    """The entropy is needed again by the backward pass."""
    x = _tensor((3, 5), grad=True)
    logp, entropy = F.token_log_prob(x, _tensor(3, np.int64))
    entropy.data._version[0] += 1
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        logp.backward(_tensor(3))
