"""GPU: the operators over a vocabulary on borrowed memory that begins at any multiple of its type, as slices of others'
arrays do."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu
F = tt.nn.functional


class _Slice:
    """The values of ``a`` behind ``offset`` others."""

    def __init__(self, a, offset):
        self.block = hiparray(np.concatenate([np.full(offset, 7, a.dtype), a.ravel(), np.full(5, 7, a.dtype)]))
        about = self.block.__cuda_array_interface__
        self.__cuda_array_interface__ = dict(about, shape=a.shape, data=(about['data'][0] + offset * a.itemsize, False))


def _tensor(a, offset, grad=False):
    return tt.as_tensor(_Slice(a, offset), requires_grad=grad)


@pytest.mark.parametrize('offset', [1, 3, 4, 7, 8])
@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,cols', [(5, 33), (3, 1000), (2, 5001)])
def test_slices(rows, cols, dtype, offset):
    rng = np.random.default_rng(offset)
    z, dy = (rng.standard_normal((rows, cols)).astype(dtype) for _ in range(2))
    w, b, g = (rng.standard_normal(n).astype(np.float32) for n in (cols, cols, rows))
    x, wt, bt = (_tensor(a, offset, True) for a in (z, w, b))
    y = F.layer_norm(x, cols, wt, bt)
    want, off, *_ = plain64.layer_norm(z, w, b, 1e-5)
    plain64.check(y.data.get(), want, plain64.stored(off, want, dtype), 'y')
    y.backward(_tensor(dy, offset))
    for got, value, bound, kind in zip((x, wt, bt), *plain64.layer_norm_grad(z, dy, w, 1e-5), (dtype, np.float32, np.float32)):
        plain64.check(got.grad.get(), value, plain64.stored(bound, value, kind), 'gradient of layer_norm')

    tokens = rng.integers(0, cols, rows)
    x = _tensor(z, offset, True)
    got = F.token_log_prob(x, _tensor(tokens, offset), 4)
    values, bounds = plain64.token_log_prob(z, tokens, 4)
    for y, value, off in zip(got, values, bounds):
        plain64.check(y.data.get(), value, off)
    np.testing.assert_array_equal(got[3].data.get(), values[3])
    tt.backward(got[:2], [_tensor(g, offset), _tensor(g, offset)])
    dz, bound = plain64.token_log_prob_grad(z, tokens, 0, g, g, None)
    plain64.check(x.grad.get(), dz, plain64.stored(bound, dz, dtype), 'gradient of token_log_prob')

    teacher, index = rng.standard_normal((rows, 6)).astype(dtype), (tokens[:, None] + np.arange(6)) % cols
    for scale in (None, np.asarray(0.5, np.float32)):
        x = _tensor(z, offset, True)
        loss = F.distill_loss(x, _tensor(teacher, offset), _tensor(index, offset), 2.0, 'sum')
        (value, off), (dz, bound) = plain64.distill(z, teacher, index, 2.0, 'sum')
        plain64.check(loss.data.get(), value, off)
        loss.backward(None if scale is None else _tensor(scale, offset))
        dz, bound = (v if scale is None else v * 0.5 for v in (dz, bound))
        plain64.check(x.grad.get(), dz, plain64.stored(bound, dz, dtype), 'gradient of distill_loss')
