"""GPU: ``F.linear_cross_entropy`` and ``nn.LinearCrossEntropy`` against the formulas in 64 bits (``products64``, where the
bounds are derived), against differences of the loss, and what its rows, targets and calls may be."""
import numpy as np
import pytest

torch = pytest.importorskip('torch')
import pytortto_amd as tt
from pytortto_amd import _hip
from pytortto_amd.xparray import hiparray
from tests import products64
from tests.plain64 import check, stored

pytestmark = pytest.mark.gpu
F = tt.nn.functional


def _tensor(a, grad=False):
    return None if a is None else tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _inputs(rows, width, vocab, dtype, seed=0, padded=0.0, index=np.int64):
    rng = np.random.default_rng(seed)
    w = (rng.standard_normal((vocab, width)) * width ** -0.5 * rng.uniform(0.3, 2.0, (vocab, 1))).astype(dtype)
    target = rng.integers(0, vocab, rows)
    x = (rng.standard_normal((rows, width)) * 1.5 + 4.0 * rng.random((rows, 1)) * w[target]).astype(dtype)
    target[rng.random(rows) < padded] = -100
    return x, w, target.astype(index)


def _compare(x, w, target, reduction='mean', g=None, scale=1.0, need=(True, True), ignore_index=-100):
    want = products64.linear_cross_entropy(x, w, target, reduction, g, scale, ignore_index)
    with tt.no_grad():
        plain = F.linear_cross_entropy(_tensor(x), _tensor(w), _tensor(target), ignore_index, reduction)
    xt, wt = _tensor(x, need[0]), _tensor(w, need[1])
    loss = F.linear_cross_entropy(xt, wt, _tensor(target), ignore_index, reduction)
    assert loss.dtype == np.float32 and loss.shape == want[0][0].shape and not plain.requires_grad
    check(plain.data.get(), *want[0], 'loss without gradients')
    check(loss.data.get(), *want[0], 'loss')
    if reduction == 'none':
        loss.backward(_tensor(np.ones(len(x), np.float32) if g is None else g))
    else:
        loss.backward(None if scale == 1.0 else _tensor(np.asarray(scale, np.float32)))
    for name, leaf, (value, bound), wanted in (('dx', xt, want[1], need[0]), ('dw', wt, want[2], need[1])):
        if not wanted:
            assert leaf.grad is None
            continue
        assert leaf.grad.dtype == x.dtype and leaf.grad.shape == leaf.shape
        check(leaf.grad.get(), value, stored(bound, np.nan_to_num(value), x.dtype), name)
    return loss


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,width,vocab', [
    (1, 1, 1), (1, 1, 2), (2, 3, 5), (1, 8, 63), (3, 64, 64), (5, 65, 65), (16, 7, 127), (17, 33, 128), (63, 72, 129), (64, 128, 255),
    (65, 100, 257), (128, 31, 300), (129, 250, 65), (200, 513, 1000), (255, 64, 10), (257, 40, 2049), (300, 17, 4100), (7, 2000, 500),
    (2, 1025, 9001), (1, 300, 33333), (1000, 9, 3)])
def test_sizes(rows, width, vocab, dtype):
    _compare(*_inputs(rows, width, vocab, dtype, rows + vocab))
    _compare(*_inputs(rows, width, vocab, dtype, rows + width, padded=0.3), reduction='sum')


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,width,vocab', [(1000, 1000, 4300), (777, 800, 17001)])
def test_rounds_that_are_not_whole(rows, width, vocab, dtype):
    """A few tiles more than the compute units can take at once: the last classes are left to smaller tiles."""
    x, w, target = _inputs(rows, width, vocab, dtype, 3, padded=0.1)
    target[:40] = vocab - 1 - np.arange(40) * 13
    _compare(x, w, target, 'sum')


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,width,vocab', [(1, 4096, 64), (3, 2048, 63), (7, 1100, 7003), (33, 2048, 4097), (64, 2048, 1000), (65, 1025, 130),
                                              (1, 2049, 8190), (128, 1500, 1), (256, 1024, 200), (257, 1536, 77), (500, 1040, 500)])
def test_few_positions_and_wide_features(rows, width, vocab, dtype):
    """Few small tiles, whose reduction several blocks share."""
    x, w, target = _inputs(rows, width, vocab, dtype, rows + vocab, padded=0.2)
    _compare(x, w, target)
    _compare(x, w, target, 'sum', scale=0.25, need=(False, True))
    g = np.random.default_rng(rows).standard_normal(rows).astype(np.float32)
    g[::3] = 0.0
    _compare(x, w, target, 'none', g)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
def test_few_positions_with_what_is_not_finite_or_not_there(dtype):
    """The rows of the test before: NaN stays in its row's loss, a class outside is NaN, and so is a class whose logits are."""
    x, w, target = _inputs(40, 2000, 300, dtype, 5)
    x[3, 7] = np.nan
    target[5], target[9] = 300, -301
    target[11:14] = -100
    x[12] = np.inf
    loss = F.linear_cross_entropy(_tensor(x), _tensor(w), _tensor(target), reduction='none').data.get()
    assert np.isnan(loss[[3, 5, 9]]).all() and (loss[11:14] == 0).all()
    assert np.isfinite(np.delete(loss, [3, 5, 9])).all()
    w[17, 0] = np.nan
    loss = F.linear_cross_entropy(_tensor(x), _tensor(w), _tensor(target), reduction='none').data.get()
    assert np.isnan(np.delete(loss, [11, 12, 13])).all() and (loss[11:14] == 0).all()
    # a row and a matrix of zeros: ln of the classes, and gradients that are the others' alone
    x, w, target = _inputs(40, 2000, 300, dtype, 6)
    x[4] = 0
    w[8] = 0
    _compare(x, w, target)
    _compare(np.zeros_like(x), w, target)
    _compare(x, np.zeros_like(w), target)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
def test_a_weight_past_32_bits(dtype):
    """2^20 classes of 2176 features, 4.6 GB or twice that; all but five rows are zeros, so that the sums are known."""
    vocab, width = 1 << 20, 2176
    rng = np.random.default_rng(14)
    hit = np.array([0, 1, vocab // 2, vocab - 2, vocab - 1])
    rows = (rng.standard_normal((5, width)) * width ** -0.5 * 4).astype(dtype)
    x = rng.standard_normal((3, width)).astype(dtype)
    target = np.array([vocab - 1, 0, vocab // 2])
    weight = torch.zeros((vocab, width), dtype=torch.float32 if dtype == np.float32 else torch.float16, device='cuda')
    weight[torch.from_numpy(hit).cuda()] = torch.from_numpy(rows).cuda()
    torch.cuda.synchronize()
    xt, wt = _tensor(x, True), tt.as_tensor(weight, True)
    loss = F.linear_cross_entropy(xt, wt, _tensor(target), reduction='sum')
    loss.backward()
    z = x.astype(np.float64) @ rows.astype(np.float64).T
    lse = np.log(np.exp(z).sum(1) + (vocab - 5))
    own = z[np.arange(3), [4, 0, 2]]
    assert abs(loss.data.get().item() - (lse - own).sum()) <= 2e-6 * np.abs(lse).sum()
    g = np.exp(z - lse[:, None])
    g[np.arange(3), [4, 0, 2]] -= 1.0
    # G is held to 2^-11 (2^-19: 2^-22 and what the logits are off by) of itself, and so is what is stored
    step, least = (2.0 ** -11, 2.0 ** -25) if dtype == np.float16 else (2.0 ** -19, 0.0)
    want, size = g @ rows.astype(np.float64), np.abs(g) @ np.abs(rows.astype(np.float64))
    assert (np.abs(xt.grad.get() - want) <= 3 * step * size + least).all()
    dw = torch.as_tensor(wt.grad, device='cuda')
    got = dw[torch.from_numpy(hit).cuda()].double().cpu().numpy()
    want, size = g.T @ x.astype(np.float64), np.abs(g).T @ np.abs(x.astype(np.float64))
    assert (np.abs(got - want) <= 3 * step * size + least).all()
    rest = np.exp(-lse) @ x.astype(np.float64)
    size = np.exp(-lse) @ np.abs(x.astype(np.float64))
    for v in (2, vocab // 2 - 1, vocab // 2 + 1, vocab - 3):
        assert (np.abs(dw[v].double().cpu().numpy() - rest) <= 3 * step * size + least).all()


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,width,vocab', [(1024, 96, 3500), (2100, 256, 1100), (900, 1000, 4000), (4000, 70, 777)])
def test_larger(rows, width, vocab, dtype):
    """Every size of tile, for every product."""
    x, w, target = _inputs(rows, width, vocab, dtype, 1, padded=0.1)
    _compare(x, w, target)
    g = np.random.default_rng(2).standard_normal(rows).astype(np.float32)
    _compare(x, w, target, 'none', g)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('index', [np.int64, np.int32])
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
def test_reductions(reduction, index, dtype):
    x, w, target = _inputs(70, 48, 130, dtype, 3, padded=0.2, index=index)
    rng = np.random.default_rng(4)
    if reduction == 'none':
        g = rng.standard_normal(70).astype(np.float32)
        g[5:9] = 0.0
        for factor in (1.0, 2.0 ** -40, 2.0 ** 20):
            if dtype == np.float32 or factor == 1.0:
                _compare(x, w, target, reduction, (g * factor).astype(np.float32))
    else:
        for scale in (1.0, 0.25, -3.0, 0.0, 512.0):
            _compare(x, w, target, reduction, scale=scale)
    for need in ((True, False), (False, True)):
        _compare(x, w, target, reduction, need=need)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
def test_leading_dimensions_and_other_ignored_values(dtype):
    x, w, target = _inputs(24, 40, 50, dtype, 5)
    flat = F.linear_cross_entropy(_tensor(x), _tensor(w), _tensor(target), reduction='none').data.get()
    shaped = F.linear_cross_entropy(_tensor(x.reshape(2, 3, 4, 40)), _tensor(w), _tensor(target.reshape(2, 3, 4)), reduction='none')
    assert shaped.shape == (2, 3, 4)
    np.testing.assert_array_equal(shaped.data.get().reshape(-1), flat)
    one = F.linear_cross_entropy(_tensor(x[0]), _tensor(w), _tensor(target[:1].reshape(())), reduction='none')
    assert one.shape == ()
    check(one.data.get(), *[np.asarray(v[0]) for v in products64.linear_cross_entropy(x[:1], w, target[:1], 'none')[0]], 'one position')
    _compare(x, w, target, ignore_index=int(target[0]))
    _compare(x, w, target, ignore_index=-1)
    negative = np.where(np.arange(24) % 2 == 0, target - 50, target)        # (count from the end)
    np.testing.assert_array_equal(F.linear_cross_entropy(_tensor(x), _tensor(w), _tensor(negative), reduction='none').data.get(), flat)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('reduction', ['none', 'sum', 'mean'])
def test_positions_without_a_target(reduction, dtype):
    """They may hold anything, and all positions may be such."""
    x, w, target = _inputs(140, 80, 200, dtype, 6, padded=0.3)
    clean = _compare(x, w, target, reduction).data.get()
    dirty = x.copy()
    dirty[target == -100] = np.nan
    dirty[np.flatnonzero(target == -100)[0]] = np.inf
    np.testing.assert_array_equal(_compare(dirty, w, target, reduction).data.get(), clean)
    nothing = np.full(140, -100)
    xt, wt = _tensor(dirty, True), _tensor(w, True)
    loss = F.linear_cross_entropy(xt, wt, _tensor(nothing), reduction=reduction)
    want = np.nan if reduction == 'mean' else 0.0
    np.testing.assert_array_equal(loss.data.get(), np.full(loss.shape, want))
    loss.backward(_tensor(np.ones(140, np.float32)) if reduction == 'none' else None)
    assert not xt.grad.get().any() and not wt.grad.get().any()


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('wrong', [130, 131, -131, 1 << 20, -(1 << 40)])
def test_targets_outside_the_vocabulary(wrong, dtype):
    x, w, target = _inputs(20, 24, 130, dtype, 7)
    target[3] = wrong
    for reduction in ('none', 'sum', 'mean'):
        _compare(x, w, target, reduction)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
def test_no_positions(dtype):
    w = _inputs(1, 8, 9, dtype)[1]
    for reduction, want in (('sum', 0.0), ('mean', np.nan), ('none', None)):
        xt, wt = _tensor(np.zeros((0, 8), dtype), True), _tensor(w, True)
        loss = F.linear_cross_entropy(xt, wt, _tensor(np.zeros(0, np.int64)), reduction=reduction)
        if reduction == 'none':
            assert loss.shape == (0,)
            loss.backward(_tensor(np.zeros(0, np.float32)))
        else:
            np.testing.assert_array_equal(loss.data.get(), want)
            loss.backward()
        assert xt.grad.shape == (0, 8) and not wt.grad.get().any() and wt.grad.dtype == dtype


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
def test_large_and_confident_logits(dtype):
    """Differences of hundreds, a target that has all of the probability and one that has none."""
    x, w, target = _inputs(40, 32, 90, dtype, 8)
    x, w = (x * 8).astype(dtype), (w * 8).astype(dtype)
    best = (x.astype(np.float64) @ w.astype(np.float64).T).argmax(1)
    target[:20] = best[:20]
    _compare(x, w, target)
    _compare(np.zeros_like(x), w, target)           # (all logits equal)
    _compare(x, np.zeros_like(w), target)


def test_rows_of_unlike_size():
    """Rows of x and W that differ by many powers of two, in float32: each has a scale of its own."""
    x, w, target = _inputs(90, 70, 110, np.float32, 9)
    rng = np.random.default_rng(9)
    a, b = rng.integers(-12, 1, (90, 1)), rng.integers(-12, 4, (110, 1))
    x, w = np.ldexp(x, a).astype(np.float32), np.ldexp(w, b).astype(np.float32)
    w[17] = 0.0
    x[11] = 0.0
    _compare(x, w, target)
    tiny, huge = np.ldexp(x, -60).astype(np.float32), np.ldexp(w, 60).astype(np.float32)
    _compare(tiny, huge, target, 'sum')


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
def test_nan_among_the_features(dtype):
    x, w, target = _inputs(12, 24, 130, dtype, 10)
    x[4, 7] = np.nan
    xt, wt = _tensor(x, True), _tensor(w, True)
    loss = F.linear_cross_entropy(xt, wt, _tensor(target), reduction='none')
    got = loss.data.get()
    assert np.isnan(got[4]) and np.isfinite(np.delete(got, 4)).all()
    loss.backward(_tensor(np.ones(12, np.float32)))
    dx = xt.grad.get()
    assert np.isnan(dx[4]).all() and np.isfinite(np.delete(dx, 4, 0)).all() and np.isnan(wt.grad.get()).all()


def test_gradients_against_differences():
    rng = np.random.default_rng(11)
    x, w, target = _inputs(30, 20, 40, np.float32, 11, padded=0.2)
    xt, wt = _tensor(x, True), _tensor(w, True)
    F.linear_cross_entropy(xt, wt, _tensor(target)).backward()
    for leaf, of in ((xt, 0), (wt, 1)):
        v = rng.standard_normal(leaf.shape)
        v /= np.linalg.norm(v)
        h = 1e-2
        ends = []
        for sign in (1, -1):
            moved = [x.copy(), w.copy()]
            moved[of] = (moved[of] + sign * h * v).astype(np.float32)
            ends.append(F.linear_cross_entropy(_tensor(moved[0]), _tensor(moved[1]), _tensor(target)).data.get().item())
        slope = float((leaf.grad.get() * v).sum())
        # the losses, about 3, are off by a few units of 2^-24 of it and the inputs are rounded: 2e-6 / 2 h; third derivative times h^2
        assert abs((ends[0] - ends[1]) / (2 * h) - slope) < 3e-4 + 0.01 * h * abs(slope)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
def test_chunks_of_positions(dtype):
    """More logits than are kept at once: 262144 classes, 2304 positions are a chunk of 2048 and one of 256."""
    rng = np.random.default_rng(12)
    rows, width, vocab = 2304, 8, 1 << 18
    x = rng.standard_normal((rows, width)).astype(dtype)
    w = (rng.standard_normal((vocab, width)) * 0.3).astype(dtype)
    target = rng.integers(0, vocab, rows)
    target[::7] = -100
    g = rng.random(rows).astype(np.float32)
    xt, wt = _tensor(x, True), _tensor(w, True)
    loss = F.linear_cross_entropy(xt, wt, _tensor(target), reduction='none')
    loss.backward(_tensor(g))
    losses, dx, dw = loss.data.get(), xt.grad.get(), wt.grad.get().astype(np.float64)
    kept = target != -100
    some = np.concatenate([np.arange(0, 40), np.arange(2030, 2070), np.arange(2290, 2304)])
    z = x[some].astype(np.float64) @ w.astype(np.float64).T
    lse = np.log(np.exp(z).sum(1))
    own = z[np.arange(len(some)), np.where(kept[some], target[some], 0)]
    np.testing.assert_allclose(losses[some], np.where(kept[some], lse - own, 0.0), rtol=2e-6)
    p = np.exp(z - lse[:, None])
    p[np.arange(len(some)), np.where(kept[some], target[some], 0)] -= 1.0
    want = (p * (kept * g)[some][:, None]) @ w.astype(np.float64)
    # (half a unit for the gradient of a logit, half a unit for the result; of terms that add up to about the result)
    tolerance = 2.0 ** -10 if dtype == np.float16 else 2.0 ** -18
    np.testing.assert_allclose(dx[some], want, atol=tolerance)
    # every position's gradients add up to zero over the classes: the columns of dw too
    column = dw.sum(0)
    size = np.abs(dw).sum(0)
    assert (np.abs(column) <= (2.0 ** -11 + 2.0 ** -11 if dtype == np.float16 else 2.0 ** -20) * size + 2.0 ** -24 * vocab).all()
    # a class that no position has: sum of p g x
    hit = np.flatnonzero(np.bincount(target[kept], minlength=vocab))[:8]
    for v in hit:
        zs = x[kept].astype(np.float64) @ w[v].astype(np.float64) - _lse(x[kept], w)
        gv = (np.exp(zs) - (target[kept] == v)) * g[kept]
        np.testing.assert_allclose(dw[v], gv @ x[kept].astype(np.float64), rtol=2.0 ** -9 if dtype == np.float16 else 2e-5, atol=2.0 ** -12 if dtype == np.float16 else 2.0 ** -20)
    # the scalar loss's gradients are accumulated over the chunks, too
    xt, wt = _tensor(x, True), _tensor(w, True)
    F.linear_cross_entropy(xt, wt, _tensor(target), reduction='sum').backward()
    again = wt.grad.get().astype(np.float64)
    for v in hit:
        gv = np.exp(x[kept].astype(np.float64) @ w[v].astype(np.float64) - _lse(x[kept], w)) - (target[kept] == v)
        np.testing.assert_allclose(again[v], gv @ x[kept].astype(np.float64), rtol=2.0 ** -9 if dtype == np.float16 else 2e-5, atol=2.0 ** -12 if dtype == np.float16 else 2.0 ** -20)


_kept_lse = {}


def _lse(x, w):
    key = x.dtype.str
    if key not in _kept_lse:
        out = np.empty(len(x))
        for i in range(0, len(x), 128):
            out[i:i + 128] = np.log(np.exp(x[i:i + 128].astype(np.float64) @ w.astype(np.float64).T).sum(1))
        _kept_lse[key] = out
    return _kept_lse[key]


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
def test_equal_calls_have_equal_bits(dtype):
    x, w, target = _inputs(700, 300, 3000, dtype, 13, padded=0.1)

    def once():
        xt, wt = _tensor(x, True), _tensor(w, True)
        loss = F.linear_cross_entropy(xt, wt, _tensor(target))
        loss.backward()
        return loss.data.get(), xt.grad.get(), wt.grad.get()

    first = once()
    _compare(*_inputs(50, 900, 70, dtype, 14))          # (another call's scratch memory in between)
    for a, b in zip(first, once()):
        np.testing.assert_array_equal(a, b)


def test_leaves_are_used_twice_and_accumulate():
    x, w, target = _inputs(60, 30, 80, np.float32, 15)
    once, wt = _tensor(x, True), _tensor(w, True)
    F.linear_cross_entropy(once, wt, _tensor(target)).backward()
    single = wt.grad.get()
    xt, wt = _tensor(x, True), _tensor(w, True)
    a, b = (F.linear_cross_entropy(xt, wt, _tensor(target)) for _ in range(2))
    tt.backward([a, b])
    np.testing.assert_array_equal(wt.grad.get(), single + single)
    np.testing.assert_array_equal(xt.grad.get(), once.grad.get() * 2)


def test_a_weight_written_in_between_is_noticed():
    x, w, target = _inputs(6, 5, 8, np.float32, 16)
    xt, wt = _tensor(x, True), _tensor(w, True)
    loss = F.linear_cross_entropy(xt, wt, _tensor(target), reduction='none')
    wt.requires_grad = False
    wt.copy_(w * 2)
    with pytest.raises(RuntimeError, match='modified'):
        loss.backward(_tensor(np.ones(6, np.float32)))


def test_module():
    layer = tt.nn.LinearCrossEntropy(40, 90, reduction='sum').cuda()
    x, _, target = _inputs(33, 40, 90, np.float32, 17, padded=0.2)
    xt = _tensor(x, True)
    loss = layer(xt, _tensor(target))
    want = products64.linear_cross_entropy(x, layer.weight.data.get(), target, 'sum')
    check(loss.data.get(), *want[0], 'loss')
    loss.backward()
    check(xt.grad.get(), *want[1], 'dx')
    check(layer.weight.grad.get(), *want[2], 'dw')


def test_unaligned_slices_of_others_memory():
    x, w, target = _inputs(10, 24, 30, np.float16, 18)
    want = F.linear_cross_entropy(_tensor(x), _tensor(w), _tensor(target), reduction='none').data.get()
    def shifted(a):
        block = torch.zeros(a.size + 1, dtype=torch.from_numpy(a).dtype, device='cuda')
        block[1:] = torch.from_numpy(a.reshape(-1)).cuda()
        return tt.as_tensor(block[1:].view(a.shape))
    arguments = shifted(x), shifted(w), shifted(target)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(F.linear_cross_entropy(*arguments, reduction='none').data.get(), want)


def test_refusals():
    x, w, target = (_tensor(a) for a in _inputs(6, 5, 8, np.float32))
    with pytest.raises(RuntimeError, match='linear_cross_entropy takes input'):
        F.linear_cross_entropy(x, w, _tensor(np.zeros(5, np.int64)))
    with pytest.raises(RuntimeError, match='linear_cross_entropy takes input'):
        F.linear_cross_entropy(x, _tensor(np.zeros((8, 6), np.float32)), target)
    with pytest.raises(TypeError, match='one type'):
        F.linear_cross_entropy(x, _tensor(np.zeros((8, 5), np.float16)), target)
    with pytest.raises(TypeError, match='int64 or int32'):
        F.linear_cross_entropy(x, w, _tensor(np.zeros(6, np.float32)))
    with pytest.raises(TypeError, match='float32 or float16'):
        F.linear_cross_entropy(_tensor(np.zeros((6, 5))), _tensor(np.zeros((8, 5))), target)
    with pytest.raises(ValueError, match='not a valid value for reduction'):
        F.linear_cross_entropy(x, w, target, reduction='max')
    ok = np.zeros(64, np.float32)
    a = hiparray(ok)
    for kind, half, bits, red, n, h, v in ((2, 0, 64, 2, 1, 1, 1), (0, 1, 64, 2, 1, 1, 1), (0, 0, 16, 2, 1, 1, 1), (0, 0, 64, 3, 1, 1, 1),
                                           (0, 0, 64, 2, 0, 1, 1), (0, 0, 64, 2, 1, 0, 1), (0, 0, 64, 2, 1, 1, 0),
                                           (0, 0, 64, 2, 1, 1, (1 << 20) + 1), (0, 0, 64, 2, 1, (1 << 20) + 1, 1)):
        with pytest.raises(RuntimeError, match='linear_cross_entropy'):
            _hip.call('tt_linear_cross_entropy', a.ptr, a.ptr, a.ptr, None, a.ptr, None, None, kind, half, bits, -100, red, n, h, v)
    with pytest.raises(RuntimeError, match='null'):
        _hip.call('tt_linear_cross_entropy', a.ptr, a.ptr, a.ptr, None, None, None, None, 0, 0, 64, -100, 2, 1, 1, 1)
    with pytest.raises(RuntimeError, match='aligned'):
        _hip.call('tt_linear_cross_entropy', a.ptr + 4, a.ptr, a.ptr, None, a.ptr, None, None, 0, 0, 64, -100, 2, 1, 1, 1)
