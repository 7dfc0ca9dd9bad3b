"""GPU: logits of ``F.linear_cross_entropy`` that are infinite: as softmax has it, -inf is a class without probability, and +inf, or none but
-inf, is NaN for its position and for what that position's gradient reaches."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray

pytestmark = pytest.mark.gpu
F = tt.nn.functional
# one block to a row, tiles of 64 and the larger ones; whole lines of 64 features and others
SIZES = [(40, 2048, 300), (40, 70, 300), (300, 256, 4100), (1100, 128, 9000)]


def _tensor(a, grad=False):
    return tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _inputs(rows, width, vocab, dtype):
    rng = np.random.default_rng(rows + width)
    w = (rng.standard_normal((vocab, width)) * width ** -0.5).astype(dtype)
    x = rng.standard_normal((rows, width)).astype(dtype)
    return x, w, rng.integers(3, vocab, rows)


def _losses(x, w, target):
    return F.linear_cross_entropy(_tensor(x), _tensor(w), _tensor(target), reduction='none').data.get()


def _infinite(x, w, sign, dtype):
    """Positions 0, 3, 6, ... have an infinite logit of class 1, of the sign; of the others it is finite, or -inf in float16."""
    x, w = x.copy(), w.copy()
    if dtype == np.float32:         # a product past the type's range, of finite values
        x[:, 0], w[:, 0] = 0.0, 0.0
        x[::3, 0], w[1, 0] = 2.0 ** 20, sign * 2.0 ** 120
    else:
        w[1, 0] = sign * np.inf
        x[:, 0] = -1.0 if sign > 0 else 1.0
        x[::3, 0] = 1.0
    return x, w


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,width,vocab', SIZES)
def test_plus_infinity(rows, width, vocab, dtype):
    x, w, target = _inputs(rows, width, vocab, dtype)
    x, w = _infinite(x, w, 1, dtype)
    target[:9] = [1, 1, 1, 2, 2, 2, 5, 5, 5]
    got = _losses(x, w, target)
    hit = np.arange(rows) % 3 == 0
    assert np.isnan(got[hit]).all()
    if dtype == np.float32:
        assert np.isfinite(got[~hit]).all()
    else:                           # class 1 is at -inf there: no probability, and a loss of inf as a target
        assert np.isinf(got[[1, 2]]).all() and np.isfinite(np.delete(got[~hit], [0, 1])).all()
    # the gradients of those positions, and of the weight, are NaN
    xt, wt = _tensor(x, True), _tensor(w, True)
    F.linear_cross_entropy(xt, wt, _tensor(target), reduction='none').backward(_tensor(np.ones(rows, np.float32)))
    assert np.isnan(xt.grad.get()[hit]).all() and np.isnan(wt.grad.get()).all()
    assert np.isnan(F.linear_cross_entropy(_tensor(x), _tensor(w), _tensor(target)).item())
    # without those positions nothing is
    if dtype == np.float32:
        target[hit] = -100
        xt, wt = _tensor(x, True), _tensor(w, True)
        F.linear_cross_entropy(xt, wt, _tensor(target)).backward()
        assert np.isfinite(xt.grad.get()).all() and np.isfinite(wt.grad.get()).all()


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,width,vocab', SIZES)
def test_minus_infinity(rows, width, vocab, dtype):
    x, w, target = _inputs(rows, width, vocab, dtype)
    x, w = _infinite(x, w, -1, dtype)
    target[0] = 1
    got = _losses(x, w, target)
    assert got[0] == np.inf
    # the class is not there: losses over the others
    fewer = np.delete(w, 1, 0)
    x64, w64 = x.astype(np.float64), fewer.astype(np.float64)
    if dtype == np.float32:
        x64[:, 0] = 0.0
    z = x64 @ w64.T
    lse = np.log(np.exp(z - z.max(1, keepdims=True)).sum(1)) + z.max(1)
    which = np.arange(0, rows, 3)[1:] if dtype == np.float32 else np.arange(1, rows)
    want = lse[which] - z[which, target[which] - 1]
    off = (44 + 6 * width / 32) * 2.0 ** -24 * (np.abs(x64) @ np.abs(w64).T).max() * 3 + 24 * 2.0 ** -24 * np.abs(lse).max()
    if dtype == np.float32:         # (the other features are held to 2^-40 of the row's first)
        off += 3 * 2.0 ** -40 * 2.0 ** 20 * np.abs(w64).sum(1).max()
    assert (np.abs(got[which] - want) <= off).all()


@pytest.mark.parametrize('rows,width,vocab', SIZES)
def test_no_class_at_all(rows, width, vocab):
    x, w, target = _inputs(rows, width, vocab, np.float16)
    w[:, 0] = -np.inf
    x[:, 0] = 1.0
    assert np.isnan(_losses(x, w, target)).all()


@pytest.mark.parametrize('rows,width,vocab', [(1, 8, 5), (3, 72, 70), (40, 2056, 300), (9, 1000, 33000), (300, 200, 4100), (1100, 56, 9000),
                                              (2048, 72, 4200), (2048, 184, 4321), (513, 248, 30000)])
def test_rows_of_float16_that_end_inside_a_line(rows, width, vocab):
    """A weight's row ends where the next begins, which may begin with what is not finite: the same bits as of rows with zeros behind them."""
    x, w, target = _inputs(rows, width, vocab, np.float16)
    x[:, 0] = 1.0
    w[2::5, 0] = -np.inf
    target[target % 5 == 2] -= 1
    more = (0, -width % 64)
    got, want = _losses(x, w, target), _losses(np.pad(x, ((0, 0), more)), np.pad(w, ((0, 0), more)), target)
    assert np.isfinite(want).all()
    np.testing.assert_array_equal(got, want)
    # a finite weight's gradients, too
    w[2::5, 0] = 0.5
    results = []
    for a, b in ((x, w), (np.pad(x, ((0, 0), more)), np.pad(w, ((0, 0), more)))):
        xt, wt = _tensor(a, True), _tensor(b, True)
        F.linear_cross_entropy(xt, wt, _tensor(target)).backward()
        results.append((xt.grad.get()[:, :width].astype(np.float64), wt.grad.get()[:, :width].astype(np.float64)))
    for one, other in zip(*results):
        assert np.abs(one - other).max() <= 2.0 ** -10 * np.abs(other).max() + 2.0 ** -24
