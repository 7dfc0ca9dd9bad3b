"""GPU: ``optim.orthogonalize`` and ``optim.Muon`` where a matrix's norm, or eps, is near the ends of float32's range or past them."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests.test_gpu_muon import _compare, _matrix, _tensor

pytestmark = pytest.mark.gpu
# one block's LDS, and several blocks
SIZES = [(20, 30), (64, 384), (70, 70), (300, 130)]


@pytest.mark.parametrize('rows,columns', SIZES)
@pytest.mark.parametrize('scale', [1e-44, 1e-40, 1e-38, 1e-35, 1e-33, 1e33, 1e36, 1e38])
def test_any_norm(scale, rows, columns):
    """(Values of 1e-44 are a few units of the smallest float32.)"""
    x = np.clip(_matrix(rows, columns, np.float64, scale=1.0) * scale, -3e38, 3e38).astype(np.float32)
    assert x.any() and np.isfinite(x).all()
    _compare(x, eps=1e-300)
    if scale < 1e-30:
        _compare(x, eps=1e-33)


@pytest.mark.parametrize('rows,columns', SIZES)
@pytest.mark.parametrize('eps', [5e-324, 1e-300, 1e-46, 1e-45, 1e-40, 1e-36, 1e-20, 1e30])
def test_zeros_stay_zeros(eps, rows, columns):
    for dtype in (np.float32, np.float16):
        got = tt.optim.orthogonalize(_tensor(np.zeros((rows, columns), dtype)), eps=eps).data.get()
        assert not got.any()


@pytest.mark.parametrize('eps', [5e-324, 1e-40, 1e-36, 1e-7])
def test_a_parameter_without_a_gradient_keeps_its_values(eps):
    """All gradients are zeros, as those of a part that is not used: the decay is all that a step does."""
    values = [np.random.default_rng(i).standard_normal(s).astype(np.float32) for i, s in enumerate(SIZES)]
    leaves = [_tensor(v, True) for v in values]
    opt = tt.optim.Muon(leaves, lr=0.5, weight_decay=0.125, eps=eps)
    for leaf in leaves:
        leaf.grad = hiparray(np.zeros(leaf.shape, np.float32))
    opt.step()
    for leaf, v in zip(leaves, values):
        np.testing.assert_array_equal(leaf.data.get(), v * np.float32(1 - 0.5 * 0.125))


@pytest.mark.parametrize('rows,columns', SIZES)
def test_what_is_not_finite_is_nan_for_any_eps(rows, columns):
    for value in (np.nan, np.inf, -np.inf):
        for eps in (5e-324, 1e-7, 1e30):
            x = _matrix(rows, columns)
            x[3, 4] = value
            assert np.isnan(tt.optim.orthogonalize(_tensor(x), eps=eps).data.get()).all()


def test_a_step_has_its_memory_before_it_begins():
    """Several batches of matrices: asked for without tables, a step's scratch memory does not grow any more."""
    import ctypes

    from pytortto_amd import _hip

    def taken():
        sizes = [ctypes.c_size_t() for _ in range(3)]
        _hip.call('tt_mem_stats', *[ctypes.byref(n) for n in sizes])
        return sizes[2].value

    shapes = [(3, 5)] * 3 + [(100, 70 + i) for i in range(50)] + [(900, 1000)] * 50
    leaves = [_tensor(_matrix(*s), True) for s in shapes]
    opt = tt.optim.Muon([{'params': leaves[:60]}, {'params': leaves[60:], 'lr': 0.25}])
    before = [leaf.data.get() for leaf in leaves]
    _hip.call('tt_empty_cache')
    for i in (slice(0, 60), slice(60, None)):
        count = len(shapes[i])
        _hip.call('tt_muon_step_multi_f32', count, None, None, None, (ctypes.c_int * count)(*[s[0] for s in shapes[i]]),
                  (ctypes.c_int * count)(*[s[1] for s in shapes[i]]), (ctypes.c_double * count)(*[1.0] * count), 0.1, 0.9, 0.0, 1, 5,
                  3.4445, -4.7750, 2.0315, 1e-7)
    asked = taken()
    assert asked > 0
    for leaf, v in zip(leaves, before):
        np.testing.assert_array_equal(leaf.data.get(), v)
        leaf.grad = hiparray(v)
    opt.step()
    assert taken() == asked
    assert all((leaf.data.get() != v).any() for leaf, v in zip(leaves, before))
    with pytest.raises(RuntimeError, match='null table'):
        _hip.call('tt_muon_step_multi_f32', 1, leaves[0].data.ptr, None, None, None, None, None, 0.1, 0.9, 0.0, 1, 5, 3.4445, -4.7750, 2.0315, 1e-7)


def test_tied_weights():
    """Two parameters on one array are stepped one after the other."""
    for rows, columns in SIZES:
        w, g = _matrix(rows, columns, scale=1.0), [_matrix(rows, columns, seed=1), _matrix(rows, columns, seed=2)]
        one, other = _tensor(w, True), _tensor(w, True)
        tied = tt.nn.Parameter(one)
        tt_opt, turns = tt.optim.Muon([one, tied], lr=0.1), [tt.optim.Muon([other], lr=0.1) for _ in range(2)]
        for _ in range(2):
            one.grad, tied.grad = hiparray(g[0]), hiparray(g[1])
            tt_opt.step()
            for k in range(2):
                other.grad = hiparray(g[k])
                turns[k].step()
            np.testing.assert_array_equal(one.data.get(), other.data.get())
