"""GPU: ``optim.orthogonalize`` and ``optim.Muon`` against the formulas in 64 bits (``products64``, where the bounds are
derived)."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd import _hip
from pytortto_amd.xparray import hiparray
from tests import products64

pytestmark = pytest.mark.gpu
ABC = (3.4445, -4.7750, 2.0315)


def _tensor(a, grad=False):
    return tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _matrix(rows, columns, dtype=np.float32, seed=0, scale=1e-2):
    rng = np.random.default_rng(seed + 31 * rows + columns)
    return (rng.standard_normal((rows, columns)) * scale + rng.standard_normal((rows, 1)) * rng.standard_normal(columns) * scale).astype(dtype)


def _compare(x, steps=5, coefficients=ABC, eps=1e-7):
    got = tt.optim.orthogonalize(_tensor(x), steps, coefficients, eps)
    assert got.dtype == x.dtype and got.shape == x.shape and not got.requires_grad
    want, off = products64.newton_schulz(x, steps, coefficients, eps)
    got = got.data.get().astype(np.float64)
    assert np.isfinite(got).all()
    if x.dtype == np.float16:
        off = off + 2.0 ** -11 * (np.linalg.norm(want) + off) + 2.0 ** -25 * np.sqrt(x.size)
    assert np.linalg.norm(got - want) <= off, (x.shape, np.linalg.norm(got - want), off)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,columns', [(1, 1), (1, 7), (9, 1), (2, 2), (3, 64), (64, 3), (16, 16), (31, 33), (64, 64), (65, 65), (63, 129),
                                          (128, 128), (130, 60), (127, 257), (256, 256), (300, 200), (64, 1000), (1000, 64), (5, 3000),
                                          (3000, 5), (511, 513), (700, 333)])
def test_sizes(rows, columns, dtype):
    _compare(_matrix(rows, columns, dtype))


@pytest.mark.parametrize('rows,columns', [(64, 384), (64, 385), (65, 384), (384, 64), (385, 64), (63, 192), (192, 64), (60, 193), (193, 33),
                                          (1, 384), (384, 1), (17, 383)])
def test_around_what_one_block_takes(rows, columns):
    _compare(_matrix(rows, columns))
    _compare(_matrix(rows, columns, np.float16), 2)


@pytest.mark.parametrize('rows,columns', [(1, 70000), (70000, 1), (40, 60001), (60001, 40), (130, 20000)])
def test_long_reductions(rows, columns):
    """Many blocks share a tile."""
    _compare(_matrix(rows, columns))


@pytest.mark.parametrize('rows,columns', [(1300, 1300), (1025, 2100), (2300, 900)])
def test_larger(rows, columns):
    _compare(_matrix(rows, columns), 3)


@pytest.mark.parametrize('steps,coefficients', [(1, ABC), (2, ABC), (7, ABC), (12, (1.5, -0.5, 0.0)), (8, (15 / 8, -10 / 8, 3 / 8)),
                                                (3, (1.0, 0.0, 0.0))])
def test_steps_and_coefficients(steps, coefficients):
    for rows, columns in ((40, 70), (70, 40)):
        _compare(_matrix(rows, columns), steps, coefficients)


def test_singular_values_come_to_one():
    """The classic coefficients converge: U V^T of the decomposition."""
    rng = np.random.default_rng(3)
    u, _ = np.linalg.qr(rng.standard_normal((96, 40)))
    v, _ = np.linalg.qr(rng.standard_normal((40, 40)))
    x = ((u * np.linspace(0.5, 2.0, 40)) @ v.T).astype(np.float32)
    got = tt.optim.orthogonalize(_tensor(x), 30, (1.5, -0.5, 0.0)).data.get()
    # from 0.5 / |X| on they have converged; what is left are the roundings of the last steps, whose slope is 0 to 1.5
    np.testing.assert_allclose(got, u @ v.T, atol=1e-5)


@pytest.mark.parametrize('scale', [1e-30, 1e-12, 1.0, 1e15, 1e30])
def test_sizes_of_values(scale):
    x = (_matrix(50, 90, scale=1.0) * scale).astype(np.float32)
    _compare(x, eps=1e-7 if scale >= 1e-3 else 1e-36)


def test_a_norm_below_eps():
    """Divided by eps then; a matrix of zeros stays one."""
    _compare(_matrix(20, 30, scale=1e-9), eps=1e-3)
    for dtype in (np.float32, np.float16):
        assert not tt.optim.orthogonalize(_tensor(np.zeros((20, 30), dtype))).data.get().any()


def test_values_that_are_not_finite():
    for value in (np.nan, np.inf, -np.inf):
        x = _matrix(20, 30)
        x[3, 4] = value
        assert np.isnan(tt.optim.orthogonalize(_tensor(x)).data.get()).all()


def test_low_rank_and_unlike_rows():
    rng = np.random.default_rng(4)
    _compare((rng.standard_normal((80, 2)) @ rng.standard_normal((2, 120))).astype(np.float32))
    x = _matrix(80, 120)
    x[::3] = 0.0
    x[:, 7] *= 1000.0
    _compare(x)


def test_empty_matrices():
    assert tt.optim.orthogonalize(_tensor(np.zeros((0, 5), np.float32))).shape == (0, 5)


def test_equal_calls_have_equal_bits():
    x = _matrix(700, 300)
    first = tt.optim.orthogonalize(_tensor(x)).data.get()
    _compare(_matrix(130, 60))
    np.testing.assert_array_equal(tt.optim.orthogonalize(_tensor(x)).data.get(), first)


# ---- the optimiser ---------------------------------------------------------------------------------

def _step64(p, g, m, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, steps=5, eps=1e-7, adjust='original'):
    """(p, m, bound of p in the Frobenius norm, bound of m)"""
    shape = p.shape
    p, g, m = (a.astype(np.float64).reshape(shape[0], -1) for a in (p, g, m))
    new = m + (1 - momentum) * (g - m)
    u = g + momentum * (new - g) if nesterov else new
    rows, columns = p.shape
    scale = np.sqrt(max(1.0, rows / columns)) if adjust == 'original' else 0.2 * np.sqrt(max(rows, columns))
    o, off = products64.newton_schulz(u, steps, ABC, eps)
    # u has a few roundings of float32 of its own; through the steps each grows by 3.4445 at most
    off += 3.4445 ** steps * 8 * products64.U * (np.linalg.norm(g) + np.linalg.norm(m)) / max(np.linalg.norm(u), eps)
    q = p * (1 - lr * weight_decay) - lr * scale * o
    bound = lr * scale * off + 4 * products64.U * (np.linalg.norm(p) + lr * scale * np.linalg.norm(o))
    return q.reshape(shape), new.reshape(shape), bound, 6 * products64.U * (np.linalg.norm(g) + np.linalg.norm(m))


def _near(got, want, bound, what):
    off = np.linalg.norm(got.astype(np.float64) - want)
    assert off <= bound, (what, got.shape, off, bound)


SHAPES = [(40, 70), (70, 40), (64, 64), (16, 3, 3, 3), (8, 16, 1, 1), (1, 5), (130, 257), (300, 128), (33, 2, 5)]


@pytest.mark.parametrize('options', [{}, dict(nesterov=False), dict(momentum=0.0), dict(adjust='match_rms_adamw', lr=0.02),
                                     dict(weight_decay=0.0, lr=0.5, momentum=0.5), dict(steps=2, eps=1e-3)])
def test_steps_of_a_group(options):
    rng = np.random.default_rng(5)
    values = [rng.standard_normal(s).astype(np.float32) for s in SHAPES]
    leaves = [_tensor(v, True) for v in values]
    names = {'adjust': 'adjust_lr_fn', 'steps': 'ns_steps'}
    opt = tt.optim.Muon(leaves, **{names.get(k, k): v for k, v in options.items()})
    momenta = [np.zeros_like(v) for v in values]
    for step in range(3):
        gradients = [_matrix(s[0], int(np.prod(s[1:])), seed=step).reshape(s) for s in SHAPES]
        for leaf, g in zip(leaves, gradients):
            leaf.grad = hiparray(g)
        opt.step()
        for i, leaf in enumerate(leaves):
            want, m, bound, off = _step64(values[i], gradients[i], momenta[i], **options)
            values[i], momenta[i] = leaf.data.get(), opt.state[leaf]['momentum_buffer'].get()
            _near(values[i], want, bound, 'parameter')
            _near(momenta[i], m, off, 'momentum')


def test_more_matrices_than_a_launch_takes():
    rng = np.random.default_rng(6)
    shapes = [(int(r), int(c)) for r, c in rng.integers(1, 90, (61, 2))]
    values = [rng.standard_normal(s).astype(np.float32) for s in shapes]
    leaves = [_tensor(v, True) for v in values]
    leaves[7].grad = None
    opt = tt.optim.Muon(leaves, lr=0.1)
    gradients = [_matrix(*s) for s in shapes]
    for i, leaf in enumerate(leaves):
        leaf.grad = None if i == 7 else hiparray(gradients[i])
    opt.step()
    for i, leaf in enumerate(leaves):
        if i == 7:
            np.testing.assert_array_equal(leaf.data.get(), values[i])
            assert 'momentum_buffer' not in opt.state[leaf]
            continue
        want, _, bound, _ = _step64(values[i], gradients[i], np.zeros_like(values[i]), lr=0.1)
        _near(leaf.data.get(), want, bound, 'parameter')


def test_a_matrix_steps_the_same_alone_and_among_others():
    rng = np.random.default_rng(7)
    shapes = [(300, 200), (40, 900), (64, 64), (513, 511)]
    values, gradients = [rng.standard_normal(s).astype(np.float32) for s in shapes], [_matrix(*s) for s in shapes]

    def stepped(which):
        leaves = [_tensor(values[i], True) for i in which]
        for leaf, i in zip(leaves, which):
            leaf.grad = hiparray(gradients[i])
        tt.optim.Muon(leaves, lr=0.1).step()
        return [leaf.data.get() for leaf in leaves]

    together = stepped(range(4))
    for i in range(4):
        np.testing.assert_allclose(stepped([i])[0], together[i], atol=2.0 ** -18)


def test_groups_checkpoints_and_values_that_others_hold():
    rng = np.random.default_rng(8)
    a, b = (rng.standard_normal(s).astype(np.float32) for s in ((12, 20), (30, 10)))
    ga, gb = _matrix(12, 20), _matrix(30, 10)

    def make():
        leaves = [_tensor(a, True), _tensor(b, True)]
        opt = tt.optim.Muon([{'params': [leaves[0]]}, {'params': [leaves[1]], 'lr': 0.3, 'nesterov': False}], lr=0.1)
        leaves[0].grad, leaves[1].grad = hiparray(ga), hiparray(gb)
        return leaves, opt

    leaves, opt = make()
    held = leaves[0].data.lent()
    opt.step()
    np.testing.assert_array_equal(held.get(), a)
    _near(leaves[0].data.get(), *_step64(a, ga, np.zeros_like(a), lr=0.1)[::2], 'first group')
    _near(leaves[1].data.get(), *_step64(b, gb, np.zeros_like(b), lr=0.3, nesterov=False)[::2], 'second group')
    saved = opt.state_dict()
    others, again = make()
    for mine, theirs in zip(others, leaves):
        mine.data.set(theirs.data.get())
    again.load_state_dict(saved)
    for o in (opt, again):
        o.step()
    for mine, theirs in zip(others, leaves):
        np.testing.assert_array_equal(mine.data.get(), theirs.data.get())


def test_a_training_step_of_a_head():
    """Layer normalisation, the loss straight from features, the optimiser: a few steps against the formulas."""
    from tests.plain64 import layer_norm
    rng = np.random.default_rng(9)
    rows, width, vocab = 120, 40, 300
    tt.manual_seed(1)
    norm, head = tt.nn.LayerNorm(width).cuda(), tt.nn.LinearCrossEntropy(width, vocab).cuda()
    opt = tt.optim.Muon([head.weight], lr=0.1)
    x = rng.standard_normal((rows, width)).astype(np.float32)
    target = rng.integers(0, vocab, rows)
    m = np.zeros((vocab, width), np.float32)
    for _ in range(3):
        w = head.weight.data.get()
        xt = _tensor(x, True)
        h = norm(xt)
        loss = head(h, _tensor(target))
        opt.zero_grad()
        loss.backward()
        n = layer_norm(x, None, None, 1e-5)[0]
        want = products64.linear_cross_entropy(h.data.get(), w, target, 'mean')
        # the normalised features are off by a few units: so are the logits and the loss
        assert abs(loss.data.get() - products64.linear_cross_entropy(n.astype(np.float32), w, target, 'mean')[0][0]) < 1e-5
        assert (np.abs(head.weight.grad.get() - want[2][0]) <= want[2][1]).all()
        g = head.weight.grad.get()
        opt.step()
        q, m64, bound, _ = _step64(w, g, m, lr=0.1)
        _near(head.weight.data.get(), q, bound, 'weight')
        m = opt.state[head.weight]['momentum_buffer'].get()
        assert np.isfinite(xt.grad.get()).all()


def test_refusals():
    x = _tensor(_matrix(4, 6))
    with pytest.raises(RuntimeError, match='takes a matrix'):
        tt.optim.orthogonalize(_tensor(np.zeros(5, np.float32)))
    with pytest.raises(TypeError, match='float32 or float16'):
        tt.optim.orthogonalize(_tensor(np.zeros((5, 5))))
    for bad in ((4.0, 0.0, 0.0), (-3.0, 0.0, 0.0), (1.0, 0.0, 30.0), (1e300, -1e300, 1e300)):
        with pytest.raises(RuntimeError, match='grow past'):
            tt.optim.orthogonalize(x, 5, bad)
    leaf = _tensor(_matrix(4, 6), True)
    opt = tt.optim.Muon([leaf])
    leaf.grad = hiparray(np.zeros((4, 5), np.float32))
    with pytest.raises(RuntimeError, match="parameter's shape"):
        opt.step()
    leaf.grad = hiparray(np.zeros((4, 6), np.float16))
    with pytest.raises(RuntimeError, match='float32 device parameters only'):
        opt.step()
    a = hiparray(np.zeros(64, np.float32))
    for kind, rows, columns, steps, eps in ((2, 2, 2, 1, 1.0), (0, 0, 2, 1, 1.0), (0, 2, 0, 1, 1.0), (0, 2, 2, 0, 1.0), (0, 2, 2, 101, 1.0),
                                            (0, 2, 2, 1, 0.0), (0, (1 << 20) + 1, 2, 1, 1.0)):
        with pytest.raises(RuntimeError, match='orthogonalize'):
            _hip.call('tt_orthogonalize', a.ptr, a.ptr, kind, rows, columns, steps, 1.0, 0.0, 0.0, eps)
