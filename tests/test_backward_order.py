"""CPU: the order in which a backward pass visits nodes whose outputs are also used by what takes no part in the pass."""
import itertools

import numpy as np
import pytest

import pytortto_amd as tt

F = tt.nn.functional


def _leaf(values=(1.0, -2.0, 3.0)):
    return tt.tensor(np.array(values, np.float32), requires_grad=True)


def _ones(n=3):
    return tt.tensor(np.ones(n, np.float32))


@pytest.mark.parametrize('order', list(itertools.permutations(range(3))))
def test_several_end_nodes_with_other_consumers(order):
    """Each end node has a consumer outside the pass, and one leads to the next.  (Their order must not depend on where
    the nodes lie in memory: several graphs are kept.)"""
    kept = []
    for _ in range(30):
        x = _leaf()
        y = x + x
        z = y + y
        u = F.relu(z)
        ends = [y, z, u]
        kept.append((ends, [F.relu(t) for t in ends]))
        tt.backward([ends[i] for i in order], [_ones() for _ in order])
        np.testing.assert_array_equal(x.grad, [10, 6, 10])      # 2 + 4 + 4 where positive


def test_one_end_node_and_two_branches_with_other_consumers():
    """Nothing is ready where both branches wait, and one of them leads to the other."""
    kept = []
    for _ in range(60):
        x = _leaf()
        a = x + x
        b = a + a
        kept.append((a, b, F.relu(a), F.relu(b)))
        (a + b).backward(_ones())
        np.testing.assert_array_equal(x.grad, [6, 6, 6])


def test_a_long_chain_of_waiting_nodes():
    kept, x = [], _leaf()
    h, total = x, None
    for _ in range(12):
        h = h + x
        total = h if total is None else total + h
        kept.append(F.relu(h))
    total.backward(_ones())
    np.testing.assert_array_equal(x.grad, np.full(3, sum(range(2, 14)), np.float32))


def test_what_stays_behind_is_there_for_a_later_pass():
    """Two passes from what shares only its leaf; a node's consumers outside the pass are counted as before."""
    x = _leaf()
    a, b = x + x, F.relu(x)
    stray = [F.relu(a), F.relu(b)]
    tt.backward([a, b], [_ones(), _ones()])
    np.testing.assert_array_equal(x.grad, [3, 2, 3])
    c = x + x
    c.backward(_ones())
    np.testing.assert_array_equal(x.grad, [5, 4, 5])
    assert len(stray) == 2
