"""CPU: what the loss from features, the orthogonalisation and its optimiser refuse and hold without a device."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd import _hip

F = tt.nn.functional


class _Foreign:
    def __init__(self, shape, kind='<f4'):
        self.__cuda_array_interface__ = {'shape': shape, 'typestr': kind, 'data': (4096, False), 'version': 3}


def _tensor(shape, kind='<f4', grad=False):
    """(No address here is ever followed.)"""
    return tt.as_tensor(_Foreign(shape, kind), requires_grad=grad)


@pytest.fixture
def nothing_is_called(monkeypatch):
    def call(name, *args):
        raise AssertionError(f'{name} was called')
    monkeypatch.setattr(_hip, 'call', call)


def test_host_tensors_are_refused():
    x, w, target = tt.randn(3, 5), tt.randn(7, 5), tt.tensor(np.zeros(3, np.int64))
    with pytest.raises(RuntimeError, match='linear_cross_entropy: .*device \\(HIP\\) path only'):
        F.linear_cross_entropy(x, w, target)
    with pytest.raises(RuntimeError, match='device \\(HIP\\) path only'):
        tt.nn.LinearCrossEntropy(5, 7)(x, target)
    with pytest.raises(RuntimeError, match='same device'):
        F.linear_cross_entropy(_tensor((3, 5)), w, target)
    with pytest.raises(RuntimeError, match='same device'):
        F.linear_cross_entropy(_tensor((3, 5)), _tensor((7, 5)), target)
    with pytest.raises(RuntimeError, match='device \\(HIP\\) path only'):
        tt.optim.orthogonalize(x)
    with pytest.raises(RuntimeError, match='device \\(HIP\\) path only'):
        tt.optim.orthogonalize(np.zeros((3, 5), np.float32))
    leaf = tt.randn(3, 5, requires_grad=True)
    leaf.grad = np.zeros((3, 5), np.float32)
    with pytest.raises(RuntimeError, match='float32 device parameters only'):
        tt.optim.Muon([leaf]).step()


def test_shapes_and_types(nothing_is_called):
    x, w, target = _tensor((4, 6)), _tensor((9, 6)), _tensor((4,), '<i8')
    for a, b, c in ((x, w, _tensor((4, 1), '<i8')), (x, w, _tensor((5,), '<i8')), (x, _tensor((9, 5)), target), (x, _tensor((6,)), target),
                    (x, _tensor((1, 9, 6)), target), (_tensor(()), w, target), (_tensor((4, 0)), _tensor((9, 0)), target),
                    (x, _tensor((0, 6)), target)):
        with pytest.raises(RuntimeError, match='linear_cross_entropy takes input'):
            F.linear_cross_entropy(a, b, c)
    with pytest.raises(TypeError, match='one type, got float32 and float16'):
        F.linear_cross_entropy(x, _tensor((9, 6), '<f2'), target)
    with pytest.raises(TypeError, match='float32 or float16, got float64'):
        F.linear_cross_entropy(_tensor((4, 6), '<f8'), _tensor((9, 6), '<f8'), target)
    with pytest.raises(TypeError, match='int64 or int32, got int16'):
        F.linear_cross_entropy(x, w, _tensor((4,), '<i2'))
    with pytest.raises(ValueError, match='not a valid value for reduction'):
        F.linear_cross_entropy(x, w, target, reduction='batchmean')
    with pytest.raises(RuntimeError, match='takes a matrix'):
        tt.optim.orthogonalize(_tensor((2, 3, 4)))
    with pytest.raises(TypeError, match='float32 or float16, got int64'):
        tt.optim.orthogonalize(_tensor((2, 3), '<i8'))


@pytest.mark.parametrize('n', [(1 << 20) + 1, (1 << 31) + 8, (1 << 32) + 8])
def test_sizes_that_no_int_holds(nothing_is_called, n):
    target = _tensor((4,), '<i8')
    for kind in ('<f4', '<f2'):
        with pytest.raises(RuntimeError, match=f'classes at most, got {n}'):
            F.linear_cross_entropy(_tensor((4, 6), kind), _tensor((n, 6), kind), target)
        with pytest.raises(RuntimeError, match=f'features at most, got {n}'):
            F.linear_cross_entropy(_tensor((4, n), kind), _tensor((9, n), kind), target)
        for shape in ((n, 3), (3, n)):
            with pytest.raises(RuntimeError, match=f'rows and columns at most, got {n}'):
                tt.optim.orthogonalize(_tensor(shape, kind))
    rows = (1 << 30) + n
    with pytest.raises(RuntimeError, match=f'positions at most, got {rows}'):
        F.linear_cross_entropy(_tensor((rows, 6)), _tensor((9, 6)), _tensor((rows,), '<i8'))


def test_arguments_of_the_orthogonalisation(nothing_is_called):
    x = _tensor((4, 6))
    for steps in (0, -1, 101, 2.0, True):
        with pytest.raises(ValueError, match='steps'):
            tt.optim.orthogonalize(x, steps)
    for eps in (0.0, -1.0, float('nan'), float('inf')):
        with pytest.raises(ValueError, match='epsilon'):
            tt.optim.orthogonalize(x, eps=eps)
    for coefficients in ((1.0, 2.0), (1.0, 2.0, 3.0, 4.0), (1.0, float('nan'), 0.0), (float('inf'), 0.0, 0.0)):
        with pytest.raises(ValueError, match='three coefficients'):
            tt.optim.orthogonalize(x, coefficients=coefficients)


def test_arguments_of_the_optimiser():
    p = _tensor((4, 6), grad=True)
    for wrong in (dict(lr=-1.0), dict(momentum=1.0), dict(momentum=-0.1), dict(weight_decay=-1.0), dict(eps=0.0), dict(ns_steps=0),
                  dict(ns_steps=2.5), dict(adjust_lr_fn='other'), dict(ns_coefficients=(1.0,))):
        with pytest.raises(ValueError):
            tt.optim.Muon([p], **wrong)
    with pytest.raises(ValueError, match='takes matrices'):
        tt.optim.Muon([p, _tensor((4,), grad=True)])
    opt = tt.optim.Muon([p, tt.nn.Parameter(tt.randn(3, 2, 2, 2))], lr=0.1)
    assert len(opt.param_groups) == 1
    with pytest.raises(ValueError, match='takes matrices'):
        opt.add_param_group({'params': [_tensor((3,), grad=True)]})
    assert len(opt.param_groups) == 1 and "ns_steps: 5" in repr(opt)
    opt.step()                  # (no gradients: nothing to do)


def test_module_state():
    layer = tt.nn.LinearCrossEntropy(4, 10, ignore_index=-1, reduction='sum')
    assert layer.weight.shape == (10, 4) and list(layer.state_dict()) == ['weight'] and np.asarray(layer.weight.data).any()
    assert repr(layer) == 'LinearCrossEntropy(in_features=4, num_classes=10, ignore_index=-1, reduction=sum)'
