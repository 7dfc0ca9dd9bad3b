"""CPU: ``tt.as_tensor`` of tensors and of what has no device memory."""
import numpy as np
import pytest

import pytortto_amd as tt


def test_a_leaf_on_the_memory_of_a_tensor():
    t = tt.tensor(np.array([1.0, 2.0], np.float32))
    leaf = tt.as_tensor(t, requires_grad=True)
    assert leaf.requires_grad and leaf.grad_fn is None and leaf.data is t.data
    assert not t.requires_grad and tt.as_tensor(t) is t
    assert tt.as_tensor(leaf, requires_grad=True) is leaf and tt.as_tensor(leaf) is leaf
    (leaf + leaf).backward(tt.tensor(np.ones(2, np.float32)))
    np.testing.assert_array_equal(leaf.grad, [2, 2])
    inner = leaf + leaf
    assert tt.as_tensor(inner, requires_grad=True) is inner
    with pytest.raises(RuntimeError, match='floating point'):
        tt.as_tensor(tt.tensor(np.arange(3), dtype=np.int64), requires_grad=True)


@pytest.mark.parametrize('data', [np.zeros(3), [1.0, 2.0], None])
def test_host_data(data):
    with pytest.raises(AttributeError, match='takes device memory.*tt.tensor'):
        tt.as_tensor(data)
