"""GPU: rows of logits that are NaN throughout, or NaN where they are not -inf: their gradients are NaN, not those of a row
that a mask has left with nothing.  Sizes for every number of threads that takes a row."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu
F = tt.nn.functional
# (rows, values): a few lanes of a wave, a wave that keeps the row, a wave, blocks that share a row, a block
SIZES = [(37, 1), (21, 2), (33, 10), (20, 100), (19, 700), (9, 1000), (18, 3000), (9, 9000), (300, 9000)]


def _tensor(a, grad=False):
    return tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _logits(rows, vocab, dtype):
    """Rows in turn: NaN throughout, NaN and -inf, one NaN, -inf throughout, ordinary ones."""
    rng = np.random.default_rng(rows * vocab)
    z = (rng.standard_normal((rows, vocab)) * 2).astype(dtype)
    z[0::6] = np.nan
    z[1::6] = -np.inf
    z[1::6, vocab // 2] = np.nan
    z[2::6, vocab - 1] = np.nan
    z[3::6] = -np.inf
    return z, rng


@pytest.mark.parametrize('top', [0, 5, 40])
@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,vocab', SIZES)
def test_token_log_prob(rows, vocab, dtype, top):
    z, rng = _logits(rows, vocab, dtype)
    top = min(top, vocab)
    tokens = rng.integers(0, vocab, rows)
    g = [rng.standard_normal(s).astype(np.float32) for s in ((rows,), (rows,), (rows, top))]
    x = _tensor(z, True)
    got = F.token_log_prob(x, _tensor(tokens), top)
    with np.errstate(invalid='ignore'):
        values, bounds = plain64.token_log_prob(z, tokens, top)
        dz, bound = plain64.token_log_prob_grad(z, tokens, top, g[0], g[1], g[2] if top else None)
    for y, want, off in zip(got, values, bounds):
        plain64.check(y.data.get(), want, off)
    if top:
        np.testing.assert_array_equal(got[3].data.get(), values[3])
    tt.backward(got[:3 if top else 2], [_tensor(v) for v in g[:3 if top else 2]])
    plain64.check(x.grad.get(), dz, plain64.stored(bound, dz, dtype), 'dx')


@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,vocab', SIZES)
def test_distill_loss(rows, vocab, dtype, reduction):
    z, rng = _logits(rows, vocab, dtype)
    k = min(vocab, 7)
    teacher = (rng.standard_normal((rows, k)) * 2).astype(dtype)
    index = (rng.integers(0, vocab, (rows, 1)) + np.arange(k) * (vocab // k)) % vocab
    index[(np.arange(rows) // 6) % 3 == 1] = -1             # every kind of row with and without a teacher, and with
    index[(np.arange(rows) // 6) % 3 == 2, 0] = vocab       # one of another vocabulary
    g = rng.standard_normal(rows).astype(np.float32) if reduction == 'none' else None
    with np.errstate(invalid='ignore'):
        (loss, off), (dz, bound) = plain64.distill(z, teacher, index, 2.0, reduction, g)
    x = _tensor(z, True)
    got = F.distill_loss(x, _tensor(teacher), _tensor(index), 2.0, reduction)
    plain64.check(got.data.get(), loss, off, 'loss')
    got.backward(None if g is None else _tensor(g))
    plain64.check(x.grad.get(), dz, plain64.stored(bound, dz, dtype), 'dx')


@pytest.mark.parametrize('rows,vocab', SIZES)
def test_distill_loss_for_another_gradient_than_one(rows, vocab):
    z, rng = _logits(rows, vocab, np.float32)
    index, teacher = np.zeros((rows, 1), np.int64), np.zeros((rows, 1), np.float32)
    with np.errstate(invalid='ignore'):
        _, (dz, bound) = plain64.distill(z, teacher, index, 1.0, 'sum')
    x = _tensor(z, True)
    F.distill_loss(x, _tensor(teacher), _tensor(index), 1.0, 'sum').backward(_tensor(np.asarray(0.5, np.float32)))
    plain64.check(x.grad.get(), dz * 0.5, bound, 'dx')
