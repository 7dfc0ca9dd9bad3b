"""GPU: ``F.layer_norm`` and ``nn.LayerNorm`` against the formulas in 64 bits (``plain64``, where the bounds are derived)
and against differences of the forward pass."""
import numpy as np
import pytest

from tests import plain64
import pytortto_amd as tt
from pytortto_amd.xparray import hiparray

pytestmark = pytest.mark.gpu
F = tt.nn.functional
EPS = 1e-5


def _inputs(rows, cols, dtype, seed=0, affine=True):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((rows, cols)) * rng.uniform(0.5, 2.0, cols) + rng.uniform(-1, 1, cols)).astype(dtype)
    dy = rng.standard_normal((rows, cols)).astype(dtype)
    w = rng.uniform(0.5, 1.5, cols).astype(np.float32) if affine else None
    b = rng.standard_normal(cols).astype(np.float32) if affine else None
    return x, dy, w, b


def _tensor(a, grad=False):
    if a is None:
        return None
    return tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


SHAPES = [(1, 1), (1, 2), (3, 1), (5, 3), (2, 7), (17, 8), (4, 15), (1, 16), (9, 17), (33, 31), (130, 32), (7, 33), (5, 63),
          (6, 64), (700, 65), (3, 96), (2, 127), (65, 128), (4, 129), (3, 255), (258, 256), (2, 257), (7, 511), (3, 513),
          (4, 768), (2, 1000), (65, 1024), (3, 1025), (5, 1537), (2, 2047), (37, 2048), (2, 2049), (3, 4095), (11, 4096),
          (2, 4097), (2, 5000), (3, 8192), (2, 8193), (4, 12289), (3, 16384), (2, 16385), (3, 40000), (1, 131073),
          (1025, 24), (4099, 40), (600, 1537)]


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,cols', SHAPES)
def test_forward_and_gradients(rows, cols, dtype):
    x, dy, w, b = _inputs(rows, cols, dtype, rows * 7919 + cols)
    xt, wt, bt = _tensor(x, True), _tensor(w, True), _tensor(b, True)
    y = F.layer_norm(xt, cols, wt, bt, EPS)
    y.backward(_tensor(dy))
    assert y.dtype == dtype and xt.grad.dtype == dtype and wt.grad.dtype == np.float32
    want, bound, *_ = plain64.layer_norm(x, w, b, EPS)
    plain64.check(y.data.get(), want, plain64.stored(bound, want, dtype), 'y')
    grads, bounds = plain64.layer_norm_grad(x, dy, w, EPS)
    plain64.check(xt.grad.get(), grads[0], plain64.stored(bounds[0], grads[0], dtype), 'dx')
    plain64.check(wt.grad.get(), grads[1], bounds[1], 'dw')
    plain64.check(bt.grad.get(), grads[2], bounds[2], 'db')


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('weight,bias', [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize('cols', [24, 1537])
def test_without_some_parameters(cols, weight, bias, dtype):
    x, dy, w, b = _inputs(50, cols, dtype, 5)
    w, b = w if weight else None, b if bias else None
    xt, wt, bt = _tensor(x, True), _tensor(w, True), _tensor(b, True)
    y = F.layer_norm(xt, (cols,), wt, bt, EPS)
    y.backward(_tensor(dy))
    want, bound, *_ = plain64.layer_norm(x, w, b, EPS)
    plain64.check(y.data.get(), want, plain64.stored(bound, want, dtype), 'y')
    grads, bounds = plain64.layer_norm_grad(x, dy, w, EPS)
    plain64.check(xt.grad.get(), grads[0], plain64.stored(bounds[0], grads[0], dtype), 'dx')
    if weight:
        plain64.check(wt.grad.get(), grads[1], bounds[1], 'dw')
    if bias:
        plain64.check(bt.grad.get(), grads[2], bounds[2], 'db')


@pytest.mark.parametrize('wanted', [(True, False, False), (False, True, False), (False, False, True), (False, True, True)])
def test_only_what_is_needed_is_computed_and_it_is_the_same(wanted):
    x, dy, w, b = _inputs(300, 515, np.float32, 6)

    def step(needs):
        tensors = [_tensor(a, n) for a, n in zip((x, w, b), needs)]
        F.layer_norm(tensors[0], 515, tensors[1], tensors[2], EPS).backward(_tensor(dy))
        return [None if t.grad is None else t.grad.get() for t in tensors]

    whole, some = step((True, True, True)), step(wanted)
    for a, s, n in zip(whole, some, wanted):
        assert (s is not None) == n
        if n:
            np.testing.assert_array_equal(a, s)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('cols', [5, 200, 3000])
def test_rows_of_one_value_and_large_offsets(cols, dtype):
    x, dy, w, b = _inputs(6, cols, dtype, 7)
    x[0] = 0
    x[1] = 3.25                       # no variance: rstd is 1 / sqrt(eps)
    x[2] += 200 if dtype == np.float16 else 1e4
    x[3] *= 100
    x[4] *= 1e-3
    xt, wt, bt = _tensor(x, True), _tensor(w, True), _tensor(b, True)
    y = F.layer_norm(xt, cols, wt, bt, EPS)
    y.backward(_tensor(dy))
    want, bound, *_ = plain64.layer_norm(x, w, b, EPS)
    plain64.check(y.data.get(), want, plain64.stored(bound, want, dtype), 'y')
    grads, bounds = plain64.layer_norm_grad(x, dy, w, EPS)
    plain64.check(xt.grad.get(), grads[0], plain64.stored(bounds[0], grads[0], dtype), 'dx')
    plain64.check(wt.grad.get(), grads[1], bounds[1], 'dw')


@pytest.mark.parametrize('cols', [9, 100, 1000, 20000])
def test_nan_and_infinity_stay_in_their_row(cols):
    x, dy, w, b = _inputs(5, cols, np.float32, 8)
    x[1, cols // 2], x[3, 0] = np.nan, np.inf
    xt = _tensor(x, True)
    y = F.layer_norm(xt, cols, _tensor(w), _tensor(b), EPS)
    y.backward(_tensor(dy))
    for out in (y.data.get(), xt.grad.get()):
        assert np.isnan(out[[1, 3]]).any(1).all() and np.isfinite(out[[0, 2, 4]]).all()


def test_gradient_against_differences():
    """L = sum(y * c); (L(x + e v) - L(x - e v)) / 2e for random directions.  The rounding of y (2^-24 of values up to 4,
    1000 of them, at random) moves the quotient by about 1e-5 / e, the third derivative by e^2: with e = 1e-2 both are far
    below the 1e-2 asked for of a directional derivative of size 10."""
    x, c, w, b = _inputs(4, 250, np.float32, 9)
    rng = np.random.default_rng(10)
    tensors = [_tensor(a, True) for a in (x, w, b)]
    F.layer_norm(tensors[0], 250, tensors[1], tensors[2], EPS).backward(_tensor(c))
    for i, base in enumerate((x, w, b)):
        v = rng.standard_normal(base.shape).astype(np.float32)
        ends = []
        for e in (1e-2, -1e-2):
            moved = [x, w, b]
            moved[i] = (base + np.float32(e) * v).astype(np.float32)
            y = F.layer_norm(*[_tensor(moved[0]), 250, _tensor(moved[1]), _tensor(moved[2])], EPS).data.get()
            ends.append((y.astype(np.float64) * c).sum())
        slope = (tensors[i].grad.get().astype(np.float64) * v).sum()
        assert abs((ends[0] - ends[1]) / 2e-2 - slope) <= 1e-2 * max(1.0, abs(slope))


def test_several_trailing_dimensions_views_and_the_module():
    rng = np.random.default_rng(11)
    x = rng.standard_normal((2, 3, 5, 7)).astype(np.float32)
    layer = tt.nn.LayerNorm((5, 7))
    with tt.no_grad():
        layer.weight.copy_(rng.uniform(0.5, 1.5, (5, 7)).astype(np.float32))
        layer.bias.copy_(rng.standard_normal((5, 7)).astype(np.float32))
    w, b = np.asarray(layer.weight.data).copy(), np.asarray(layer.bias.data).copy()
    layer.cuda()
    xt = _tensor(x, True)
    y = layer(xt)
    assert y.shape == x.shape
    want, bound, *_ = plain64.layer_norm(x.reshape(6, 35), w.ravel(), b.ravel(), layer.eps)
    plain64.check(y.data.get().reshape(6, 35), want, bound, 'y')
    dy = rng.standard_normal(x.shape).astype(np.float32)
    y.backward(_tensor(dy))
    grads, bounds = plain64.layer_norm_grad(x.reshape(6, 35), dy.reshape(6, 35), w.ravel(), layer.eps)
    assert layer.weight.grad.shape == (5, 7) and layer.bias.grad.shape == (5, 7)
    plain64.check(layer.weight.grad.get().ravel(), grads[1], bounds[1], 'dw')
    plain64.check(xt.grad.get().reshape(6, 35), grads[0], bounds[0], 'dx')
    assert list(layer.state_dict()) == ['weight', 'bias']


def test_gradients_accumulate_and_repeat_bit_for_bit():
    x, dy, w, b = _inputs(777, 1030, np.float32, 12)
    wt, bt = _tensor(w, True), _tensor(b, True)
    first = None
    for _ in range(3):
        xt = _tensor(x, True)
        wt.grad = bt.grad = None
        F.layer_norm(xt, 1030, wt, bt, EPS).backward(_tensor(dy))
        got = [t.grad.get() for t in (xt, wt, bt)]
        if first is None:
            first = got
        for a, c in zip(first, got):
            np.testing.assert_array_equal(a, c)
    F.layer_norm(_tensor(x), 1030, wt, bt, EPS).backward(_tensor(dy))
    np.testing.assert_array_equal(wt.grad.get(), 2 * first[1])


def test_no_rows():
    xt, wt, bt = _tensor(np.zeros((0, 12), np.float32), True), _tensor(np.ones(12, np.float32), True), \
        _tensor(np.zeros(12, np.float32), True)
    y = F.layer_norm(xt, 12, wt, bt)
    assert y.shape == (0, 12)
    y.backward(_tensor(np.zeros((0, 12), np.float32)))
    np.testing.assert_array_equal(wt.grad.get(), np.zeros(12))
    np.testing.assert_array_equal(bt.grad.get(), np.zeros(12))


def test_normalises_the_output_of_a_parked_operation():
    """The residual sum in front of it has not been launched when layer_norm is called."""
    x, r, w, b = _inputs(40, 96, np.float32, 13)
    xt, rt = _tensor(x, True), _tensor(r, True)
    total = xt + rt
    y = F.layer_norm(total, 96, _tensor(w), _tensor(b), EPS)
    want, bound, *_ = plain64.layer_norm((x + r).astype(np.float32), w, b, EPS)
    plain64.check(y.data.get(), want, bound, 'y')
    y.backward(_tensor(r))
    np.testing.assert_array_equal(xt.grad.get(), rt.grad.get())


def test_refusals():
    x, w = _tensor(np.zeros((4, 8), np.float32)), _tensor(np.ones(8, np.float32))
    with pytest.raises(RuntimeError, match='expected input with shape'):
        F.layer_norm(x, 4)
    with pytest.raises(RuntimeError, match='expected input with shape'):
        F.layer_norm(x, ())
    with pytest.raises(RuntimeError, match='weight to be of same shape'):
        F.layer_norm(x, 8, _tensor(np.ones(4, np.float32)))
    with pytest.raises(RuntimeError, match='same device'):
        F.layer_norm(x, 8, tt.ones(8))
    with pytest.raises(RuntimeError, match='at least one value'):
        F.layer_norm(_tensor(np.zeros((4, 0), np.float32)), 0)
    with pytest.raises(TypeError, match='float32 or float16'):
        F.layer_norm(_tensor(np.zeros((4, 8), np.float64)), 8)
    with pytest.raises(TypeError, match='float32 only'):
        F.layer_norm(x, 8, _tensor(np.ones(8, np.float16)))
    from pytortto_amd import _hip
    for args, message in (((x.data.ptr, None, None, x.data.ptr, None, None, 1e-5, 7, 4, 8), 'unknown type'),
                          ((None, None, None, x.data.ptr, None, None, 1e-5, 0, 4, 8), 'null pointer'),
                          ((x.data.ptr, None, None, x.data.ptr, None, None, 1e-5, 0, 0, 8), 'rows must be'),
                          ((x.data.ptr, None, None, x.data.ptr, None, None, 1e-5, 0, 4, 0), 'columns must be'),
                          ((x.data.ptr + 4, None, None, x.data.ptr, None, None, 1e-5, 0, 1, 4), '16-byte aligned'),
                          ((x.data.ptr, None, None, x.data.ptr, w.data.ptr, None, 1e-5, 0, 4, 8), 'come together')):
        with pytest.raises(RuntimeError, match=message):
            _hip.call('tt_layer_norm_fwd', *args)
