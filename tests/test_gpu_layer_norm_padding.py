"""GPU: layer normalisation's gradient where a row does not fill its last sixteen bytes and its mean is so large that what
stands in for the missing columns would overflow."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu


def _tensor(a, grad=False):
    return tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


WIDTHS = [5, 17, 33, 70, 131, 257, 390, 1025, 2050, 3301, 5001, 9001, 13001, 17001, 40001]


@pytest.mark.parametrize('rows,cols,level,eps', [(3, d, 2.0 ** 100, 1e-20) for d in WIDTHS]
                         + [(300, 70, 2.0 ** 100, 1e-20)] + [(2, d, 2.0 ** 121, 1e-5) for d in WIDTHS[:4]])
def test_constant_rows(rows, cols, level, eps):
    """Every sum of a row's values is a multiple of one power of two that float32 holds exactly, so mean and variance are
    the row's value and zero."""
    rng = np.random.default_rng(cols)
    z = np.full((rows, cols), level, np.float32)
    dy, w = rng.standard_normal((rows, cols)).astype(np.float32), rng.standard_normal(cols).astype(np.float32)
    (dx, _, db), (_, _, off) = plain64.layer_norm_grad(z, dy, w, float(np.float32(eps)))
    x, wt, bt = _tensor(z, True), _tensor(w, True), _tensor(np.zeros(cols, np.float32), True)
    y = tt.nn.functional.layer_norm(x, cols, wt, bt, eps)
    np.testing.assert_array_equal(y.data.get(), np.zeros((rows, cols)))
    y.backward(_tensor(dy))
    # the values less their mean are zero exactly: dx = (h - mean h) / sqrt(eps), which the mean's rounding does not move
    h, r = dy.astype(np.float64) * w, 1.0 / np.sqrt(float(np.float32(eps)))
    bound = plain64.U * r * (plain64.chain(cols) * np.abs(h).mean(1, keepdims=True) + 8 * np.abs(h)) + 8 * plain64.U * np.abs(dx)
    plain64.check(x.grad.get(), dx, bound, 'dx')
    np.testing.assert_array_equal(wt.grad.get(), np.zeros(cols))
    plain64.check(bt.grad.get(), db, off, 'db')
