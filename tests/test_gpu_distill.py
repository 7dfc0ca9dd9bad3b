"""GPU: ``F.distill_loss`` and ``nn.DistillLoss`` against the formulas in 64 bits (``plain64``, where the bounds are
derived) and against differences of the forward pass."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu
F = tt.nn.functional


def _tensor(a, grad=False):
    return None if a is None else tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _inputs(rows, vocab, k, dtype, seed, teacher_dtype=None, index_dtype=np.int64):
    rng = np.random.default_rng(seed)
    z = (rng.standard_normal((rows, vocab)) * 2).astype(dtype)
    if k <= vocab:
        index = (rng.integers(0, vocab, (rows, 1)) + np.arange(k) * (vocab // k)) % vocab
    else:
        index = rng.integers(0, vocab, (rows, k))
    teacher = -np.sort(-(rng.standard_normal((rows, k)) * 2 + 6), axis=1)
    return z, teacher.astype(teacher_dtype or dtype), index.astype(index_dtype)


def _compare(z, teacher, index, temperature=1.0, reduction='mean', g=None, scale=None):
    (loss, off), (dz, bound) = plain64.distill(z, teacher, index, temperature, reduction, g)
    with tt.no_grad():
        plain = F.distill_loss(_tensor(z), _tensor(teacher), _tensor(index), temperature, reduction)
    xt = _tensor(z, True)
    got = F.distill_loss(xt, _tensor(teacher), _tensor(index), temperature, reduction)
    assert got.dtype == np.float32 and got.shape == loss.shape and not plain.requires_grad
    plain64.check(got.data.get(), loss, off, 'loss')
    plain64.check(plain.data.get(), loss, off, 'loss without gradients')
    if scale is not None:
        dz, bound = dz * scale, bound * abs(scale)
        got.backward(_tensor(np.asarray(scale, np.float32)))
    else:
        got.backward(_tensor(g))
    assert xt.grad.dtype == z.dtype
    plain64.check(xt.grad.get(), dz, plain64.stored(bound, dz, z.dtype), 'dx')


VOCABS = [1, 2, 5, 8, 10, 63, 64, 65, 100, 257, 511, 1000, 1024, 1025, 2049, 4097, 8200, 16385, 32768, 32771, 50021, 65537,
          131072, 200003]


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('vocab', VOCABS)
def test_sizes(vocab, dtype):
    for rows, k, t, reduction in ((1, min(4, vocab), 1.0, 'mean'), (3, min(33, vocab), 2.0, 'sum'), (6, 1, 4.0, 'mean')):
        _compare(*_inputs(rows, vocab, k, dtype, vocab + rows), t, reduction)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,vocab,k', [(5000, 10, 4), (1300, 100, 10), (700, 1000, 64), (515, 4099, 8), (300, 9001, 100),
                                          (258, 33000, 32), (513, 20001, 16), (64, 70001, 64), (300, 40001, 50),
                                          (270, 70001, 7)])
def test_many_rows(rows, vocab, k, dtype):
    z, teacher, index = _inputs(rows, vocab, k, dtype, rows)
    rng = np.random.default_rng(vocab)
    index[rng.random(rows) < 0.2] = -1                                      # no teacher
    index[rng.random(index.shape) < 0.1] = -1                               # holes
    _compare(z, teacher, index, 1.5, 'mean')
    _compare(z, teacher, index, 1.0, 'none', rng.standard_normal(rows).astype(np.float32))


@pytest.mark.parametrize('dtype,teacher_dtype,index_dtype', [(np.float32, np.float16, np.int32), (np.float16, np.float32, np.int64),
                                                             (np.float32, np.float32, np.int32), (np.float16, np.float16, np.int32)])
@pytest.mark.parametrize('vocab', [40, 3001, 60001])
def test_types(vocab, dtype, teacher_dtype, index_dtype):
    _compare(*_inputs(5, vocab, 12, dtype, 3, teacher_dtype, index_dtype), 2.0, 'mean')


@pytest.mark.parametrize('k', [1, 2, 63, 64, 65, 255, 256, 257, 700, 1024])
@pytest.mark.parametrize('vocab', [50, 2500])
def test_numbers_of_entries(k, vocab):
    """Among them more entries than classes: those of one class add up."""
    _compare(*_inputs(5, vocab, k, np.float32, k), 1.0, 'mean')


@pytest.mark.parametrize('scale', [1.0, 0.25, -3.0, 0.0, 65536.0])
@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('vocab', [30, 5003, 60001])
def test_incoming_gradients(vocab, dtype, scale):
    """One, as ``loss.backward()`` sends it, and others, as a weighted or scaled loss does."""
    z, teacher, index = _inputs(4, vocab, 9, dtype, 4)
    _compare(z, teacher, index, 1.0, 'mean', scale=scale / 65536 if dtype == np.float16 and scale > 100 else scale)
    ones_and_others = np.array([1.0, 0.5, 1.0, -2.0], np.float32)
    _compare(z, teacher, index, 1.0, 'none', ones_and_others)
    _compare(z, teacher, index, 1.0, 'none', np.ones(4, np.float32))


def test_a_second_backward_pass_through_a_new_node_and_accumulation():
    z, teacher, index = _inputs(7, 2500, 9, np.float32, 5)
    xt = _tensor(z, True)
    for _ in range(2):
        F.distill_loss(xt, _tensor(teacher), _tensor(index)).backward()
    (_, _), (dz, bound) = plain64.distill(z, teacher, index, 1.0, 'mean')
    plain64.check(xt.grad.get(), 2 * dz, 2 * bound + 2 * plain64.U * np.abs(dz), 'twice')


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows', [3, 30, 300])
@pytest.mark.parametrize('vocab', [13, 300, 5003, 40009])
def test_masks_and_poison(rows, vocab, dtype):
    """Rows without a teacher, teachers of -inf, students that a mask leaves nothing of (with -inf or the type's lowest
    value), entries where the student has -inf, NaN, infinities, indexes out of range: row by row."""
    if rows * vocab > 4e6:
        rows = 66
    k = 6
    z, teacher, index = _inputs(rows, vocab, k, dtype, vocab)
    low = np.finfo(dtype).min
    rng = np.random.default_rng(6)
    for r in range(rows):
        kind = r % 12
        if kind == 1:
            index[r] = -1
        elif kind == 2:
            teacher[r] = -np.inf
        elif kind == 3:
            teacher[r, 1:] = -np.inf
            z[r, index[r, 1]] = -np.inf                 # asked for with probability zero only
        elif kind == 4:
            z[r] = -np.inf
        elif kind == 5:
            z[r] = low
        elif kind == 6:
            z[r, index[r, 0]] = -np.inf                 # infinitely far
        elif kind == 7:
            z[r, vocab - 1] = np.nan
        elif kind == 8:
            teacher[r, 2] = np.nan
        elif kind == 9:
            index[r, 3] = vocab
        elif kind == 10:
            teacher[r], index[r, ::2] = low, -7
        elif kind == 11:
            z[r, rng.random(vocab) < 0.5] = -np.inf
            z[r, index[r]] = 1.0
    g = rng.standard_normal(rows).astype(np.float32)
    _compare(z, teacher, index, 1.0, 'none', g)
    _compare(z, teacher, index, 3.0, 'none', g)
    fine = np.isin(np.arange(rows) % 12, (0, 1, 2, 3, 5, 10, 11))
    _compare(np.ascontiguousarray(z[fine]), np.ascontiguousarray(teacher[fine]), np.ascontiguousarray(index[fine]), 1.0, 'mean')


def test_no_row_has_a_teacher():
    z, teacher, index = _inputs(3, 40, 2, np.float32, 7)
    index[:] = -1
    xt = _tensor(z, True)
    mean = F.distill_loss(xt, _tensor(teacher), _tensor(index))
    assert np.isnan(mean.item())                # nothing to average, as in nll_loss
    mean.backward()
    np.testing.assert_array_equal(xt.grad.get(), np.zeros((3, 40)))
    assert F.distill_loss(xt, _tensor(teacher), _tensor(index), reduction='sum').item() == 0.0


@pytest.mark.parametrize('temperature', [1e-3, 0.5, 1.0, 7.0, 1e3])
def test_temperatures(temperature):
    z, teacher, index = _inputs(5, 900, 8, np.float32, 8)
    _compare(z, teacher, index, temperature, 'none', np.ones(5, np.float32))


@pytest.mark.parametrize('vocab', [60, 5000])
def test_gradient_against_differences(vocab):
    """(L(z + e v) - L(z - e v)) / 2e: L is of size 5 with rounding 1e-6 and its third derivative of size 1: with
    e = 1e-2 the quotient is off by 1e-4 + 1e-4 at most, 5e-3 is asked for."""
    z, teacher, index = _inputs(4, vocab, 5, np.float32, 9)
    xt = _tensor(z, True)
    F.distill_loss(xt, _tensor(teacher), _tensor(index), 2.0).backward()
    v = np.random.default_rng(10).standard_normal(z.shape).astype(np.float32)
    ends = [F.distill_loss(_tensor((z + np.float32(e) * v).astype(np.float32)), _tensor(teacher), _tensor(index), 2.0).item()
            for e in (1e-2, -1e-2)]
    slope = (xt.grad.get().astype(np.float64) * v).sum()
    assert abs((ends[0] - ends[1]) / 2e-2 - slope) <= 5e-3 * max(1.0, abs(slope))


def test_leading_dimensions_and_the_module():
    z, teacher, index = _inputs(30, 77, 5, np.float32, 11)
    flat = F.distill_loss(_tensor(z), _tensor(teacher), _tensor(index), 2.0, 'none').data.get()
    layer = tt.nn.DistillLoss(temperature=2.0, reduction='none')
    cube = layer(_tensor(z.reshape(2, 3, 5, 77)), _tensor(teacher.reshape(2, 3, 5, 5)), _tensor(index.reshape(2, 3, 5, 5)))
    assert cube.shape == (2, 3, 5)
    np.testing.assert_array_equal(cube.data.get().ravel(), flat)
    one = layer(_tensor(z[4]), _tensor(teacher[4]), _tensor(index[4]))
    assert one.shape == ()
    np.testing.assert_allclose(one.item(), flat[4], rtol=1e-5)


def test_a_teachers_alternatives_are_what_the_student_learns_from():
    """token_log_prob's alternatives go in as they are: with all classes among them the loss of the teacher's own logits
    is zero, and its gradient."""
    rng = np.random.default_rng(12)
    z = (rng.standard_normal((6, 50)) * 2).astype(np.float32)
    _, _, top, index = F.token_log_prob(_tensor(z), _tensor(np.zeros(6, np.int64)), top=50)
    xt = _tensor(z, True)
    loss = F.distill_loss(xt, top, index, reduction='sum')
    loss.backward()
    # six rows of a sum of 50 terms q log(q / p), each within 16 u (1 + |log q|) of zero
    assert abs(loss.item()) <= 6 * 16 * plain64.U * 12 and np.abs(xt.grad.get()).max() <= 64 * plain64.U


def test_results_repeat_bit_for_bit():
    z, teacher, index = _inputs(90, 45001, 20, np.float32, 13)
    first = None
    for _ in range(3):
        xt = _tensor(z, True)
        loss = F.distill_loss(xt, _tensor(teacher), _tensor(index))
        loss.backward()
        out = [loss.data.get(), xt.grad.get()]
        first = first or out
        for a, b in zip(first, out):
            np.testing.assert_array_equal(a, b)


def test_no_rows():
    for reduction, want in (('none', np.zeros(0)), ('sum', 0.0), ('mean', np.nan)):
        xt = _tensor(np.zeros((0, 12), np.float32), True)
        loss = F.distill_loss(xt, _tensor(np.zeros((0, 3), np.float32)), _tensor(np.zeros((0, 3), np.int64)),
                              reduction=reduction)
        np.testing.assert_array_equal(loss.data.get(), want)
        loss.backward(_tensor(np.zeros(0, np.float32)) if reduction == 'none' else None)
        assert xt.grad.shape == (0, 12)


def test_a_changed_input_is_noticed():
    z, teacher, index = _inputs(3, 20, 4, np.float32, 14)
    xt = _tensor(z, True)
    y = xt + xt
    loss = F.distill_loss(y, _tensor(teacher), _tensor(index))
    F.relu_(y)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_refusals():
    x, t, i = (_tensor(a) for a in (np.zeros((4, 8), np.float32), np.zeros((4, 3), np.float32), np.zeros((4, 3), np.int64)))
    with pytest.raises(RuntimeError, match='takes logits'):
        F.distill_loss(x, t, _tensor(np.zeros((4, 2), np.int64)))
    with pytest.raises(RuntimeError, match='takes logits'):
        F.distill_loss(_tensor(np.zeros((5, 8), np.float32)), t, i)
    with pytest.raises(RuntimeError, match='same device'):
        F.distill_loss(x, tt.zeros(4, 3), i)
    with pytest.raises(ValueError, match='1 to 1024 entries'):
        F.distill_loss(x, _tensor(np.zeros((4, 0), np.float32)), _tensor(np.zeros((4, 0), np.int64)))
    with pytest.raises(ValueError, match='1 to 1024 entries'):
        F.distill_loss(x, _tensor(np.zeros((4, 1025), np.float32)), _tensor(np.zeros((4, 1025), np.int64)))
    with pytest.raises(ValueError, match='not a valid value for reduction'):
        F.distill_loss(x, t, i, reduction='batch')
    for temperature in (0.0, -1.0, float('nan'), float('inf'), 1e-9):
        with pytest.raises(ValueError, match='temperature'):
            F.distill_loss(x, t, i, temperature)
    with pytest.raises(TypeError, match='logits must be float32 or float16'):
        F.distill_loss(_tensor(np.zeros((4, 8), np.float64)), t, i)
    with pytest.raises(TypeError, match="teacher's logits must be"):
        F.distill_loss(x, _tensor(np.zeros((4, 3), np.int32)), i)
    with pytest.raises(TypeError, match="teacher's indexes must be"):
        F.distill_loss(x, t, _tensor(np.zeros((4, 3), np.int16)))
    from pytortto_amd import _hip
    p = x.data.ptr
    good = [p, p, p, p, p, p, None, 1.0, 2, 0, 0, 64, 4, 8, 3]
    for at, value, message in ((0, None, 'null pointer'), (0, p + 4, '16-byte aligned'), (7, 0.0, 'temperature must be'),
                               (8, 3, 'reduction must be'), (9, 2, 'unknown type'), (10, -1, 'unknown type'),
                               (11, 8, '32 or 64 bits'), (12, 0, 'rows must be'), (13, 0, 'vocabulary must have'),
                               (14, 0, 'entries must be'), (14, 1025, 'entries must be')):
        args = list(good)
        args[at] = value
        with pytest.raises(RuntimeError, match=message):
            _hip.call('tt_distill_fwd', *args)
