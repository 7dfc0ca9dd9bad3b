"""GPU: distillation of logits that are large beside the temperature.  A probability depends on differences of logits
alone, so neither the loss nor the gradient may lose accuracy to the size of the logits themselves."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu
F = tt.nn.functional


def _tensor(a, grad=False):
    return tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _compare(z, teacher, index, temperature, reduction, scale):
    rows = len(z)
    g = np.full(rows, scale, np.float32) if reduction == 'none' else None
    (loss, off), (dz, bound) = plain64.distill(z, teacher, index, temperature, reduction, g)
    if reduction != 'none':
        dz, bound = dz * scale, bound * scale
    x = _tensor(z, True)
    got = F.distill_loss(x, _tensor(teacher), _tensor(index), temperature, reduction)
    plain64.check(got.data.get(), loss, off, 'loss')
    if reduction != 'none':
        g = None if scale == 1 else np.asarray(scale, np.float32)
    got.backward(None if g is None else _tensor(g))
    plain64.check(x.grad.get(), dz, plain64.stored(bound, dz, z.dtype), 'dx')


# rows by some lanes of a wave, by a wave, by blocks of 256 and of 512, longer than the registers, shared by blocks
SIZES = [(20, 100), (9, 1000), (5, 3000), (3, 20000), (300, 9000), (3, 70000)]
LARGE = (130, 66000)


@pytest.mark.parametrize('reduction,scale', [('sum', 1), ('sum', 2), ('mean', 1), ('none', 1)])
@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,vocab', SIZES + [LARGE])
def test_large_logits_at_temperature_one(rows, vocab, dtype, reduction, scale):
    """Values of one size, the type's lowest among them, as a mask leaves them: probabilities of 1 / V, times 4096 that a
    half holds them."""
    z = np.full((rows, vocab), np.finfo(dtype).min, dtype)
    z[1::3] = 20000.0
    z[2::3] = 60000.0
    index = np.arange(4)[None, :] + np.zeros((rows, 1), np.int64)
    teacher = np.zeros((rows, 4), dtype)
    _compare(z, teacher, index, 1.0, reduction, scale * (4096.0 if reduction != 'sum' or scale != 1 else 1.0))


def _logits(rows, vocab, dtype, size, temperature):
    """A few classes of the largest logit share the probability, the others have none, or, where the logits' spacing
    allows it, a part that the temperature decides."""
    rng = np.random.default_rng(rows * vocab)
    z = np.full((rows, vocab), size, np.float64)
    z -= rng.choice([0.0, 1.0, 2.0, 5.0], (rows, vocab)) * temperature
    z[:, ::2] -= 100.0 * temperature
    index = rng.integers(0, vocab // 4, (rows, 1)) + np.arange(6) * (vocab // 8)
    return z.astype(dtype), (rng.integers(0, 3, (rows, 6)) * temperature).astype(dtype), index


SCALES = [(60.0, 1e-3), (20000.0, 0.1), (60000.0, 1e-2), (-60000.0, 1e-4), (30000.0, 1e-5), (3.0, 1e-6), (50.0, 20.0), (-65504.0, 1e-6)]


@pytest.mark.parametrize('reduction', ['sum', 'mean', 'none'])
@pytest.mark.parametrize('size,temperature', SCALES)
@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,vocab', SIZES[:-1])
def test_low_temperatures(rows, vocab, dtype, size, temperature, reduction):
    _compare(*_logits(rows, vocab, dtype, size, temperature), temperature, reduction, 1.0)


@pytest.mark.parametrize('size,temperature', SCALES[1::3])
def test_low_temperatures_of_long_rows(size, temperature):
    _compare(*_logits(*LARGE, np.float16, size, temperature), temperature, 'sum', 1.0)
