"""CPU: ``optim.Muon`` refuses what it cannot do before anything has moved, and asks for a step's memory before its first launch."""
from itertools import count

import pytest

import pytortto_amd as tt
from pytortto_amd import _hip

_addresses = count(1 << 20, 1 << 20)


class _Foreign:
    def __init__(self, shape, kind):
        self.__cuda_array_interface__ = {'shape': shape, 'typestr': kind, 'data': (next(_addresses), False), 'version': 3}


def _tensor(shape, kind='<f4', grad=False):
    """(No address here is ever followed.)"""
    return tt.as_tensor(_Foreign(shape, kind), requires_grad=grad)


def _leaf(*shape):
    leaf = _tensor(shape, grad=True)
    leaf.grad = _tensor(shape).data
    return leaf


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(_hip, 'call', lambda name, *args: made.append((name, args)))
    return made


def _steps(made):
    return [args for name, args in made if name == 'tt_muon_step_multi_f32']


def test_coefficients_that_let_values_grow():
    p = _leaf(4, 6)
    for bad in ((4.0, 0.0, 0.0), (-3.0, 0.0, 0.0), (1.0, 0.0, 30.0), (1e300, -1e300, 1e300)):
        with pytest.raises(ValueError, match='grow past'):
            tt.optim.Muon([p], ns_coefficients=bad)
    with pytest.raises(ValueError, match='grow past'):
        tt.optim.Muon([p], ns_coefficients=(1.2, 0.0, 0.0), ns_steps=8)
    tt.optim.Muon([p], ns_coefficients=(1.2, 0.0, 0.0), ns_steps=3)
    for steps in (1, 5, 100):
        tt.optim.Muon([p], ns_steps=steps)
        tt.optim.Muon([p], ns_coefficients=(1.5, -0.5, 0.0), ns_steps=steps)


WRONG = [dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-1.0), dict(eps=0.0), dict(eps=float('nan')), dict(ns_steps=0), dict(ns_steps=2.0),
         dict(adjust_lr_fn='other'), dict(ns_coefficients=(1.0,)), dict(ns_coefficients=(9.0, 0.0, 0.0))]


@pytest.mark.parametrize('wrong', WRONG, ids=lambda d: f'{next(iter(d))}')
def test_options_of_a_group(wrong, calls):
    a, b = _leaf(4, 6), _leaf(5, 3)
    with pytest.raises(ValueError):
        tt.optim.Muon([{'params': [a]}, {'params': [b], **wrong}])
    opt = tt.optim.Muon([a])
    with pytest.raises(ValueError):
        opt.add_param_group({'params': [b], **wrong})
    assert len(opt.param_groups) == 1
    # changed, or loaded, afterwards: the step is refused whole
    opt.add_param_group({'params': [b]})
    opt.param_groups[1].update(wrong)
    with pytest.raises(ValueError):
        opt.step()
    assert not calls and not any('momentum_buffer' in opt.state[p] for p in (a, b))


def test_gradients_that_do_not_fit(calls):
    for shape, kind, error in (((3, 5), '<f4', "parameter's shape"), ((5, 3), '<f2', 'float32 device parameters only')):
        a, b = _leaf(4, 6), _leaf(5, 3)
        b.grad = _tensor(shape, kind).data
        opt = tt.optim.Muon([{'params': [a]}, {'params': [b]}])
        with pytest.raises(RuntimeError, match=error):
            opt.step()
        assert not calls and 'momentum_buffer' not in opt.state[a]


@pytest.mark.parametrize('shape,what', [(((1 << 20) + 1, 2), 'rows'), ((2, (1 << 20) + 1), 'columns'), ((1 << 17, 1 << 16), 'values')])
def test_sizes(shape, what, calls):
    a, b = _leaf(4, 6), _leaf(*shape)
    with pytest.raises(RuntimeError, match=f'{what} at most'):
        tt.optim.Muon([{'params': [a]}, {'params': [b]}]).step()
    assert not calls


def test_memory_is_asked_for_before_anything_moves(calls, monkeypatch):
    a, b, c = _leaf(4, 6), _leaf(5, 3), _leaf(7, 2)
    opt = tt.optim.Muon([{'params': [a, c]}, {'params': [b], 'lr': 0.5}])
    opt.step()
    made = _steps(calls)
    assert [m[0] for m in made] == [2, 1, 2, 1]
    assert all(m[1:4] == (None, None, None) for m in made[:2]) and all(None not in m[1:4] for m in made[2:])
    assert [m[4:] for m in made[:2]] == [m[4:] for m in made[2:]]
    assert [name for name, _ in calls].index('tt_muon_step_multi_f32') > max(
        (i for i, (name, _) in enumerate(calls) if name in ('tt_malloc', 'tt_memset')), default=0)
    # one call asks by itself
    del calls[:]
    b.grad = None
    opt.step()
    assert [m[0] for m in _steps(calls)] == [2] and None not in _steps(calls)[0][1:4]

    def refuse(name, *args):
        calls.append((name, args))
        if name == 'tt_muon_step_multi_f32' and args[0] == 1:
            raise RuntimeError('out of memory')

    del calls[:]
    b.grad = _tensor((5, 3)).data
    monkeypatch.setattr(_hip, 'call', refuse)
    with pytest.raises(RuntimeError, match='out of memory'):
        opt.step()
    assert all(m[1] is None for m in _steps(calls))


def test_a_parameter_that_comes_twice(calls):
    a, b = _leaf(4, 6), _leaf(5, 3)
    with pytest.warns(UserWarning):
        opt = tt.optim.Muon([a, b, a])
    opt.step()
    made = _steps(calls)
    assert [m[0] for m in made] == [2, 1, 2, 1] and [m[1] is None for m in made] == [True, True, False, False]


def test_parameters_on_the_same_memory(calls):
    """Tied weights: one after the other, as the same parameter twice is."""
    a, b = _leaf(4, 6), _leaf(5, 3)
    tied, turned = tt.nn.Parameter(a), tt.Tensor.on(a.data.reshape(6, 4), True)
    tied.grad, turned.grad = _tensor((4, 6)).data, _tensor((6, 4)).data
    opt = tt.optim.Muon([a, tied, b, turned])
    opt.step()
    made = _steps(calls)
    assert [m[0] for m in made] == [2, 1, 1] * 2
    assert all(len(set(m[1])) == m[0] for m in made[3:])


def test_nothing_to_do(calls):
    a = _leaf(0, 6)
    opt = tt.optim.Muon([a, _tensor((3, 4), grad=True)])
    opt.step()
    assert not _steps(calls)
