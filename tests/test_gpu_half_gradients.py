"""GPU: gradients of float16 tensors that are used more than once."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd import ops
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu
F = tt.nn.functional


def _tensor(a, grad=False):
    return tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _halves(rng, n):
    """Bit patterns of every finite size, with infinities and NaN."""
    bits = rng.integers(0, 1 << 16, n).astype(np.uint16)
    return bits.view(np.float16)


def _sum(a, b):
    """Rounded once: in 64 bits every sum of two halves is exact."""
    with np.errstate(invalid='ignore', over='ignore'):
        return (a.astype(np.float64) + b.astype(np.float64)).astype(np.float16)


@pytest.mark.parametrize('n', [0, 1, 7, 8, 9, 15, 16, 1000, 4099, (1 << 21) + 5])
def test_sums(n):
    rng = np.random.default_rng(n)
    a, b = _halves(rng, n), _halves(rng, n)
    x, y = hiparray(a), hiparray(b)
    want = _sum(a, b)
    got = ops.add(x, y)
    assert got.dtype == np.float16 and got.shape == (n,)
    np.testing.assert_array_equal(got.get(), want)
    x += y
    np.testing.assert_array_equal(x.get(), want)
    np.testing.assert_array_equal(y.get(), b)


def test_refusals():
    x = hiparray(np.zeros(4, np.float16))
    with pytest.raises(ValueError, match='equal shapes and dtypes'):
        x += hiparray(np.zeros(4, np.float32))
    with pytest.raises(ValueError, match='equal shapes and dtypes'):
        x += hiparray(np.zeros(5, np.float16))
    with pytest.raises(TypeError, match='float32'):
        x += 1.0
    with pytest.raises(TypeError):
        ops.add(x, hiparray(np.zeros(4, np.float32)))
    with pytest.raises(TypeError):
        y = hiparray(np.zeros(4, np.int64))
        y += y


def _inputs(rows, vocab):
    rng = np.random.default_rng(rows)
    z = (rng.standard_normal((rows, vocab)) * 2).astype(np.float16)
    tokens = rng.integers(0, vocab, rows)
    g = rng.standard_normal(rows).astype(np.float32)
    teacher, index = rng.standard_normal((rows, 3)).astype(np.float16), rng.integers(0, vocab, (rows, 3))
    return z, tokens, g, teacher, index


def _two_losses(x, tokens, g, teacher, index):
    logp, _ = F.token_log_prob(x, _tensor(tokens))
    loss = F.distill_loss(x, _tensor(teacher), _tensor(index), 1.0, 'sum')
    return [logp, loss], [_tensor(g), None]


def _gradients(z, tokens, g, teacher, index):
    """Both losses' gradients of the logits with their bounds, and how far their sum may be off."""
    a, off_a = plain64.token_log_prob_grad(z, tokens, 0, g, None, None)
    _, (b, off_b) = plain64.distill(z, teacher, index, 1.0, 'sum')
    return a + b, plain64.stored(plain64.stored(off_a, a, np.float16) + plain64.stored(off_b, b, np.float16), a + b, np.float16)


@pytest.mark.parametrize('rows,vocab', [(5, 33), (4, 1000)])
def test_two_operators_on_one_leaf(rows, vocab):
    z, *rest = _inputs(rows, vocab)
    x = _tensor(z, True)
    tt.backward(*_two_losses(x, *rest))
    want, bound = _gradients(z, *rest)
    plain64.check(x.grad.get(), want, bound)


@pytest.mark.parametrize('rows,vocab', [(5, 33), (4, 1000)])
def test_two_operators_on_one_inner_tensor(rows, vocab):
    """Layer normalisation gives the logits; its own gradient is that of the sum of theirs."""
    z, *rest = _inputs(rows, vocab)
    x = _tensor(z, True)
    logits = F.layer_norm(x, vocab)
    tt.backward(*_two_losses(logits, *rest))
    held = logits.data.get()
    total, off = _gradients(held, *rest)
    (dx, _, _), (bound, _, _) = plain64.layer_norm_grad(z, total, None, 1e-5)
    _, _, n, r, _ = plain64.layer_norm(z, None, None, 1e-5)
    moved = r * (off + off.mean(1, keepdims=True) + np.abs(n) * (off * np.abs(n)).mean(1, keepdims=True))
    plain64.check(x.grad.get(), dx, plain64.stored(bound + moved, dx, np.float16))


def test_two_passes_into_one_leaf():
    z, *rest = _inputs(6, 50)
    x = _tensor(z, True)
    for _ in range(2):
        tt.backward(*_two_losses(x, *rest))
    want, bound = _gradients(z, *rest)
    plain64.check(x.grad.get(), 2 * want, plain64.stored(2 * bound, 2 * want, np.float16))
