"""GPU: arrays on memory of others, and the stream of its writers."""

import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray

pytestmark = pytest.mark.gpu


class _Owner:
    def __init__(self, array, **more):
        self.array = array
        self.__cuda_array_interface__ = dict(array.__cuda_array_interface__, version=3, **more)


@pytest.mark.parametrize('stream', [None, 1, 2])
def test_operators_on_borrowed_memory(stream):
    z = np.random.default_rng(0).standard_normal((5, 33)).astype(np.float32)
    x = tt.as_tensor(_Owner(hiparray(z), stream=stream), requires_grad=True)
    y = tt.nn.functional.layer_norm(x, (33,))
    want = (z - z.mean(1, keepdims=True)) / np.sqrt(z.var(1, keepdims=True) + 1e-5)
    np.testing.assert_allclose(y.data.get(), want, atol=1e-5)
    y.backward(tt.as_tensor(_Owner(hiparray(z), stream=stream)))
    assert x.grad.shape == z.shape


def test_no_stream():
    with pytest.raises(RuntimeError, match='0 is no stream'):
        tt.as_tensor(_Owner(hiparray(np.ones(3, np.float32)), stream=0))
