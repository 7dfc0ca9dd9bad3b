"""CPU: what the operators over a vocabulary and the passes from several tensors do without a device."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests import plain64

F = tt.nn.functional


def test_host_tensors_are_refused():
    x = tt.randn(3, 5)
    with pytest.raises(RuntimeError, match='layer_norm: .*device \\(HIP\\) path only'):
        F.layer_norm(x, 5)
    with pytest.raises(RuntimeError, match='device \\(HIP\\) path only'):
        tt.nn.LayerNorm(5)(x)
    with pytest.raises(RuntimeError, match='token_log_prob: .*device \\(HIP\\) path only'):
        F.token_log_prob(x, tt.tensor(np.zeros(3, np.int64)))
    with pytest.raises(RuntimeError, match='distill_loss: .*device \\(HIP\\) path only'):
        F.distill_loss(x, x, tt.tensor(np.zeros((3, 5), np.int64)))


def test_layer_norm_module_state():
    layer = tt.nn.LayerNorm((3, 4), eps=1e-3)
    assert layer.weight.shape == (3, 4) and list(layer.state_dict()) == ['weight', 'bias']
    np.testing.assert_array_equal(layer.weight.data, np.ones((3, 4)))
    np.testing.assert_array_equal(layer.bias.data, np.zeros((3, 4)))
    assert repr(layer) == 'LayerNorm((3, 4), eps=0.001, elementwise_affine=True)'
    assert list(tt.nn.LayerNorm(4, elementwise_affine=False).parameters()) == []
    assert list(tt.nn.LayerNorm(4, bias=False).state_dict()) == ['weight']


def test_one_pass_from_several_tensors():
    """The sum of the passes from each, with every node visited once."""
    def graph():
        x = tt.tensor(np.array([1.0, -2.0, 3.0], np.float32), requires_grad=True)
        a = x + x
        b = F.relu(a)
        return x, a, b, b + x

    g = [tt.tensor(np.array(v, np.float32)) for v in ((1, 2, 3), (4, 5, 6), (7, 8, 9))]
    x, a, b, c = graph()
    tt.backward([a, b, c], g)
    mask = np.array([1, 0, 1])
    np.testing.assert_array_equal(x.grad, 2 * (np.array([1, 2, 3]) + mask * (np.array([4, 5, 6]) + np.array([7, 8, 9]))) + np.array([7, 8, 9]))
    x, a, b, c = graph()
    tt.backward([c, a, a], [g[2], g[0], g[1]])
    np.testing.assert_array_equal(x.grad, 2 * (np.array([5, 7, 9]) + mask * np.array([7, 8, 9])) + np.array([7, 8, 9]))
    x, *_ = graph()
    tt.backward(x, g[0])
    np.testing.assert_array_equal(x.grad, [1, 2, 3])
    x = tt.tensor(np.array(2.0, np.float32), requires_grad=True)
    tt.backward([x + x, x])
    assert x.grad == 3
    with pytest.raises(RuntimeError, match='got 2 tensors and 1 gradients'):
        tt.backward([x, x], [None])
    with pytest.raises(RuntimeError, match='does not require grad'):
        tt.backward([tt.zeros(2)], [tt.zeros(2)])


class _Foreign:
    def __init__(self, **about):
        self.__cuda_array_interface__ = dict({'shape': (2, 3), 'typestr': '<f4', 'data': (4096, False), 'version': 3,
                                              'strides': None}, **about)


def test_borrowed_memory():
    """(No address here is ever followed.)"""
    owner = _Foreign()
    t = tt.as_tensor(owner, requires_grad=True)
    assert t.shape == (2, 3) and t.dtype == np.float32 and t.is_cuda and t.requires_grad and t.data_ptr() == 4096
    assert t.data._buf.owner is owner and t.data.reshape((3, 2))._buf.owner is owner
    about = t.data.__cuda_array_interface__
    assert about['shape'] == (2, 3) and about['typestr'] == '<f4' and about['data'] == (4096, False)
    assert tt.as_tensor(t) is t
    assert tt.as_tensor(_Foreign(strides=(12, 4))).shape == (2, 3)
    assert tt.as_tensor(_Foreign(shape=(1, 3), strides=(400, 4))).shape == (1, 3)
    for strides in ((4, 8), (24, 4), (0, 4)):
        with pytest.raises(ValueError, match='C-contiguous'):
            tt.as_tensor(_Foreign(strides=strides))
    with pytest.raises(ValueError, match='masked'):
        tt.as_tensor(_Foreign(mask=owner))
    with pytest.raises(RuntimeError, match='floating point'):
        tt.as_tensor(_Foreign(typestr='<i8'), requires_grad=True)
    with pytest.raises(AttributeError):
        tt.as_tensor(np.zeros(3))


def test_the_plain_forms_gradients_are_those_of_their_values():
    """plain64 itself: each gradient against differences of its function, in 64 bits."""
    rng = np.random.default_rng(0)
    e = 1e-5

    def slope(f, x, v):
        return (f(x + e * v) - f(x - e * v)) / (2 * e)

    x, dy, w = rng.standard_normal((4, 7)), rng.standard_normal((4, 7)), rng.standard_normal(7)
    (dx, dw, db), _ = plain64.layer_norm_grad(x, dy, w, 1e-5)
    v, vw = rng.standard_normal((4, 7)), rng.standard_normal(7)
    np.testing.assert_allclose(slope(lambda a: (plain64.layer_norm(a, w, None, 1e-5)[0] * dy).sum(), x, v), (dx * v).sum(), rtol=1e-6)
    np.testing.assert_allclose(slope(lambda a: (plain64.layer_norm(x, a, None, 1e-5)[0] * dy).sum(), w, vw), (dw * vw).sum(), rtol=1e-6)
    tokens = np.array([0, -1, -100, 3])
    g = [rng.standard_normal(4), rng.standard_normal(4), rng.standard_normal((4, 3))]

    def value(z):
        a, h, top, _ = plain64.token_log_prob(z, tokens, 3)[0]
        return (a * g[0]).sum() + (h * g[1]).sum() + (top * g[2]).sum()

    dz, _ = plain64.token_log_prob_grad(x, tokens, 3, *g)
    np.testing.assert_allclose(slope(value, x, v), (dz * v).sum(), rtol=1e-6)
    teacher, index = rng.standard_normal((4, 3)), np.array([[0, 1, 2], [3, 3, 1], [-1, 6, 5], [-1, -1, -1]])
    for reduction in ('sum', 'mean'):
        _, (dz, _) = plain64.distill(x, teacher, index, 2.0, reduction)
        np.testing.assert_allclose(slope(lambda a: plain64.distill(a, teacher, index, 2.0, reduction)[0][0], x, v), (dz * v).sum(), rtol=1e-6)


def test_the_ones_that_backward_passes_start_with(monkeypatch):
    """One block, shared: who writes it gets a copy.  (Allocation and launches are recorded, not carried out.)"""
    from pytortto_amd import _hip, xparray
    calls = []

    def call(name, *args):
        calls.append(name)
        if name == 'tt_malloc':
            args[0]._obj.value = 4096 * (1 + len(calls))

    monkeypatch.setattr(_hip, 'call', call)
    monkeypatch.setattr(xparray, '_one', None)
    monkeypatch.setattr(xparray._Buffer, '__del__', lambda self: None)
    a, b = xparray.one(0), xparray.one(2)
    assert a.shape == () and b.shape == (1, 1) and a.ptr == b.ptr and calls == ['tt_malloc', 'tt_fill_f32']
    assert xparray.is_one(a) and xparray.is_one(b) and not xparray.is_one(hiparray.empty((1,)))
    b += 1.0
    assert b.ptr != a.ptr and not xparray.is_one(b) and xparray.is_one(xparray.one(1))
    assert calls[-2:] == ['tt_memcpy_d2d', 'tt_add_scalar_f32']
    first, second, third = hiparray.carve(((3,), np.float32), ((0, 2), np.float32), ((2, 2), np.int64))
    assert first.ptr % 256 == second.ptr % 256 == third.ptr % 256 == 0 and third.ptr >= first.ptr + 12
    assert first._buf.owner is third._buf.owner and third.nbytes == 32 and third.dtype == np.int64
    assert third.ptr + third.nbytes <= first._buf.owner._ptr + first._buf.owner.nbytes
