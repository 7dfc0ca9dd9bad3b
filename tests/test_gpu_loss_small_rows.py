"""GPU: gradients of ``F.linear_cross_entropy`` in float32 where rows of the weight, of the features or of the incoming gradient are small
beside the others: each is held to its own digits, against the formulas in 64 bits.

The bounds, u = 2^-24.  Operands are held to 2^-22 of each value (two of them and what is left out of the product: 12 u), or to 2^-40 of the
largest of the row (logits) or matrix (gradients); a sum of K terms takes 32 + 6 K / 32 roundings.  So a logit is off by d = (44 + 6 H / 32) u |x| |w|,
and G = softmax(z) - [v = t] by 2 d and twelve roundings of itself, and by 2^-40."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray

pytestmark = pytest.mark.gpu
F = tt.nn.functional
U = 2.0 ** -24


def _tensor(a, grad=False):
    return tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _inputs(rows, width, vocab, seed):
    rng = np.random.default_rng(seed)
    w = (rng.standard_normal((vocab, width)) * width ** -0.5).astype(np.float32)
    target = rng.integers(0, vocab, rows)
    x = (rng.standard_normal((rows, width)) + 2.0 * w[target]).astype(np.float32)
    return x, w, target


def _check(x, w, target, g=None, scale=1.0):
    rows, vocab = len(x), len(w)
    kept = target != -100
    clean = np.where(kept[:, None], x, 0).astype(np.float64)
    weight = np.where(kept, scale if g is None else g.astype(np.float64), 0.0)
    w64 = w.astype(np.float64)
    z = clean @ w64.T
    d = (44 + 6 * x.shape[1] / 32) * U * (np.abs(clean) @ np.abs(w64).T)
    # (floors of the logits' operands)
    d += 2.0 ** -39 * (np.abs(clean).max(1)[:, None] * np.abs(w64).sum(1) + np.abs(clean).sum(1)[:, None] * np.abs(w64).max(1))
    big = z.max(1, keepdims=True)
    dz = np.exp(z - big)
    dz /= dz.sum(1, keepdims=True)
    off = dz * (d + (dz * d).sum(1, keepdims=True) + U * (12 + 4 * np.abs(z - big)))
    at = np.flatnonzero(kept)
    dz[at, target[at]] -= 1.0
    off[at, target[at]] = d[at].max(1) * 2 + 8 * U
    off += 2.0 ** -40
    size = np.abs(dz)
    sums = lambda k: (44 + 6 * k / 32) * U
    dx = weight[:, None] * (dz @ w64)
    off_x = np.abs(weight)[:, None] * (off @ np.abs(w64) + sums(vocab) * (size @ np.abs(w64)) + 2.0 ** -39 * np.abs(w64).max() * size.sum(1, keepdims=True))
    gx = weight[:, None] * clean
    dw = dz.T @ gx
    off_w = off.T @ np.abs(gx) + sums(rows) * (size.T @ np.abs(gx)) + 2.0 ** -39 * np.abs(gx).max() * size.sum(0)[:, None]

    xt, wt = _tensor(x, True), _tensor(w, True)
    loss = F.linear_cross_entropy(xt, wt, _tensor(target), reduction='sum' if g is None else 'none')
    loss.backward(_tensor(np.asarray(scale, np.float32) if g is None else g))
    for name, got, want, bound in (('dx', xt.grad.get(), dx, off_x), ('dw', wt.grad.get(), dw, off_w)):
        bound = bound + 4 * U * np.abs(want) + 1e-44
        over = np.abs(got.astype(np.float64) - want) - bound
        assert np.isfinite(got).all(), name
        worst = np.unravel_index(np.argmax(over), over.shape)
        assert (over <= 0).all(), (name, worst, got[worst], want[worst], bound[worst])
    return xt.grad.get(), wt.grad.get(), dx, dw


# one block to a row of logits, tiles of 64, of 128 and of 256
SIZES = [(40, 1100, 300), (90, 70, 110), (256, 128, 9000), (1024, 64, 9000), (700, 300, 17000)]


@pytest.mark.parametrize('rows,width,vocab', SIZES)
def test_small_rows_of_the_weight(rows, width, vocab):
    """2^-8 to 2^-60 of the others' size, with targets and without: their gradients have as many digits as the others'."""
    x, w, target = _inputs(rows, width, vocab, rows)
    for k, shift in enumerate((-8, -12, -16, -20, -24, -30, -40, -60)):
        w[k::40] = np.ldexp(w[k::40], shift)
    target[1::2] = target[1::2] // 40 * 40 + 8 + target[1::2] % 30      # (half of the targets are large rows)
    np.clip(target, 0, vocab - 1, out=target)
    _, got, _, want = _check(x, w, target)
    # of each row by itself: sums of hundreds of terms of one sign or two
    quiet = np.setdiff1d(np.arange(vocab), target)
    for k in range(8):
        rows_of = quiet[quiet % 40 == k]
        assert rows_of.size == 0 or np.linalg.norm(got[rows_of] - want[rows_of]) <= 2.0 ** -16 * np.linalg.norm(want[rows_of]), k


@pytest.mark.parametrize('rows,width,vocab', SIZES)
def test_small_rows_of_the_features(rows, width, vocab):
    x, w, target = _inputs(rows, width, vocab, rows + 1)
    for k, shift in enumerate((-8, -16, -24, -32, -48, -60, 10)):
        x[k::9] = np.ldexp(x[k::9], shift)
    target[5::17] = -100
    got, _, want, _ = _check(x, w, target)
    kept = np.flatnonzero(target != -100)
    # (a position that is sure of its target has a G, and with it a gradient, below 2^-40: that is the least it is held to)
    least = 2.0 ** -40 * np.linalg.norm(np.abs(w.astype(np.float64)).sum(0))
    for i in kept[:60]:
        assert np.linalg.norm(got[i] - want[i]) <= 2.0 ** -16 * np.linalg.norm(want[i]) + least, i


@pytest.mark.parametrize('rows,width,vocab', SIZES[:4])
def test_small_and_large_gradients_of_losses(rows, width, vocab):
    x, w, target = _inputs(rows, width, vocab, rows + 2)
    g = np.random.default_rng(rows).standard_normal(rows).astype(np.float32)
    g[::5] = np.ldexp(g[::5], -60)
    g[1::5] = np.ldexp(g[1::5], -100)
    g[2::5] = 0.0
    got, _, want, _ = _check(x, w, target, g)
    for i in np.flatnonzero(np.arange(rows) % 5 < 2)[:60]:
        assert np.linalg.norm(got[i] - want[i]) <= 2.0 ** -16 * np.linalg.norm(want[i]), i
    _check(x, w, target, np.ldexp(g, 80).astype(np.float32))
    _check(x, w, target, np.ldexp(g, -40).astype(np.float32))


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,width,vocab', SIZES[:3])
def test_any_gradient_of_a_position_without_a_target(rows, width, vocab, dtype):
    """A position without a target has no gradient, whatever its loss's incoming gradient is."""
    x, w, target = _inputs(rows, width, vocab, 7)
    x, w = x.astype(dtype), w.astype(dtype)
    target[::4] = -100
    results = []
    for value in (0.0, 1.0, np.nan, np.inf, 1e38):
        g = np.random.default_rng(8).standard_normal(rows).astype(np.float32)
        g[::4] = value
        xt, wt = _tensor(x, True), _tensor(w, True)
        F.linear_cross_entropy(xt, wt, _tensor(target), reduction='none').backward(_tensor(g))
        results.append((xt.grad.get(), wt.grad.get()))
        assert not results[-1][0][::4].any()
    for dx, dw in results:
        np.testing.assert_array_equal(dx, results[0][0])
        np.testing.assert_array_equal(dw, results[0][1])


def test_a_weight_that_began_at_zeros():
    """A few classes have been trained for a step, the others are zeros or nearly so."""
    x, w, target = _inputs(200, 96, 4000, 9)
    w *= 1e-9
    w[:50] = _inputs(1, 96, 50, 10)[1]
    w[100:200] = 0.0
    _check(x, w, target)
