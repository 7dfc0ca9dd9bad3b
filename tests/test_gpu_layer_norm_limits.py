"""GPU: layer normalisation at every width where more threads, or more values of each, take a row."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu


def _tensor(a):
    return tt.Tensor(hiparray(a), requires_grad=True, dtype=a.dtype)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('packs', [4, 8, 16, 24, 32, 48, 64, 96, 128, 192, 256, 320, 384, 512, 768, 960, 2048, 3072, 4096])
@pytest.mark.parametrize('odd', [-1, 0, 1])
def test_limits(packs, odd, dtype):
    """Rows of whole packs of sixteen bytes, and of one value less or more; more rows than a block takes at once."""
    cols, rows = packs * (16 // np.dtype(dtype).itemsize) + odd, 150 if packs <= 96 else 13
    rng = np.random.default_rng(cols)
    x, dy = (rng.standard_normal((rows, cols)) * 2 + 0.5).astype(dtype), rng.standard_normal((rows, cols)).astype(dtype)
    w, b = rng.uniform(0.5, 1.5, cols).astype(np.float32), rng.standard_normal(cols).astype(np.float32)
    xt, wt, bt = _tensor(x), _tensor(w), _tensor(b)
    y = tt.nn.functional.layer_norm(xt, cols, wt, bt)
    y.backward(_tensor(dy))
    want, bound, *_ = plain64.layer_norm(x, w, b, 1e-5)
    plain64.check(y.data.get(), want, plain64.stored(bound, want, dtype), 'y')
    grads, bounds = plain64.layer_norm_grad(x, dy, w, 1e-5)
    for got, value, off, kind in zip((xt, wt, bt), grads, bounds, (dtype, np.float32, np.float32)):
        plain64.check(got.grad.get(), value, plain64.stored(off, value, kind), 'gradient')
