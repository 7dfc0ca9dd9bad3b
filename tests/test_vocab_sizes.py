"""CPU: rows that are longer than the kernels count are refused, whatever a C int would make of their length."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd import _hip

F = tt.nn.functional


class _Foreign:
    def __init__(self, shape, kind='<f4'):
        self.__cuda_array_interface__ = {'shape': shape, 'typestr': kind, 'data': (4096, False), 'version': 3}


def _tensor(shape, kind='<f4', grad=False):
    return tt.as_tensor(_Foreign(shape, kind), requires_grad=grad)


@pytest.fixture(autouse=True)
def nothing_is_called(monkeypatch):
    def call(name, *args):
        raise AssertionError(f'{name} was called')
    monkeypatch.setattr(_hip, 'call', call)


@pytest.mark.parametrize('n', [(1 << 30) + 1, (1 << 31) + 8, (1 << 32) + 8, 1 << 40])
@pytest.mark.parametrize('kind', ['<f4', '<f2'])
@pytest.mark.parametrize('grad', [False, True])
def test_long_rows(n, kind, grad):
    x = _tensor((2, n), kind, grad)
    with pytest.raises(RuntimeError, match=f'layer_norm: .*2\\^30.* got {n}'):
        F.layer_norm(x, n)
    with pytest.raises(RuntimeError, match=f'layer_norm: .*2\\^30.* got {n * 2}'):
        F.layer_norm(_tensor((3, 2, n), kind, grad), (2, n))
    with pytest.raises(RuntimeError, match=f'token_log_prob: .*2\\^30.* got {n}'):
        F.token_log_prob(x, _tensor((2,), '<i8'))
    with pytest.raises(RuntimeError, match=f'distill_loss: .*2\\^30.* got {n}'):
        F.distill_loss(x, _tensor((2, 3)), _tensor((2, 3), '<i8'))
