"""GPU: ``F.token_log_prob`` against the formulas in 64 bits (``plain64``, where the bounds are derived) and against
differences of the forward pass."""
import numpy as np
import pytest

import pytortto_amd as tt
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu
F = tt.nn.functional


def _tensor(a, grad=False):
    return None if a is None else tt.Tensor(hiparray(a), requires_grad=grad, dtype=a.dtype)


def _logits(rows, vocab, dtype, seed):
    rng = np.random.default_rng(seed)
    z = rng.standard_normal((rows, vocab)) * 2
    z[np.arange(rows), rng.integers(0, vocab, rows)] += 8
    return z.astype(dtype)


def _compare(z, tokens, top, ignore_index=-100, grads=True, seed=1):
    """Forward, and backward with random gradients of all outputs, against plain64."""
    rng = np.random.default_rng(seed)
    xt = _tensor(z, grads)
    got = F.token_log_prob(xt, _tensor(tokens), top=top, ignore_index=ignore_index)
    (logp, entropy, best, order), bounds = plain64.token_log_prob(z, tokens, top, ignore_index)
    assert len(got) == (4 if top else 2) and all(g.dtype == np.float32 for g in got[:3])
    plain64.check(got[0].data.get(), logp, bounds[0], 'logp')
    plain64.check(got[1].data.get(), entropy, bounds[1], 'entropy')
    if top:
        assert got[3].dtype == np.int64 and not got[3].requires_grad
        np.testing.assert_array_equal(got[3].data.get(), order)
        plain64.check(got[2].data.get(), best, bounds[2], 'top_logp')
    if not grads:
        assert not got[0].requires_grad
        return
    rows = len(tokens)
    g = [rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32),
         rng.standard_normal((rows, top)).astype(np.float32) if top else None]
    used = 3 if top else 2
    tt.backward(got[:used], [_tensor(v) for v in g[:used]])
    assert xt.grad.dtype == z.dtype
    want, bound = plain64.token_log_prob_grad(z, tokens, top, *g, ignore_index)
    plain64.check(xt.grad.get(), want, plain64.stored(bound, want, z.dtype), 'dx')


VOCABS = [1, 2, 3, 5, 7, 8, 9, 10, 31, 63, 64, 65, 100, 255, 256, 257, 511, 1000, 1023, 1024, 1025, 2047, 2049, 4095,
          4097, 8191, 8200, 12345, 16385, 32768, 32771, 50021, 65537, 131072, 200003]


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('vocab', VOCABS)
def test_sizes(vocab, dtype):
    """Few rows, odd numbers of them, rows that begin at every alignment."""
    rng = np.random.default_rng(vocab)
    for rows, top in ((1, min(5, vocab)), (2, 0), (7, min(20, vocab))):
        z = _logits(rows, vocab, dtype, vocab + rows)
        _compare(z, rng.integers(0, vocab, rows), top)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,vocab,top', [(5000, 10, 3), (1300, 100, 0), (700, 1000, 10), (600, 1537, 64), (515, 4099, 0),
                                            (300, 9001, 5), (257, 33000, 1), (258, 33000, 64), (513, 20001, 0), (64, 70001, 20),
                                            (300, 40001, 20), (270, 70001, 0)])
def test_many_rows(rows, vocab, top, dtype):
    rng = np.random.default_rng(rows)
    z = _logits(rows, vocab, dtype, rows + vocab)
    tokens = rng.integers(0, vocab, rows)
    tokens[rng.random(rows) < 0.1] = -100
    _compare(z, tokens, top)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows', [2, 40, 600])
@pytest.mark.parametrize('vocab', [11, 300, 5003, 40009])
def test_masks_and_poison(rows, vocab, dtype):
    """Rows that a mask leaves nothing of, with -inf or the type's lowest value, single survivors, NaN, infinities;
    tokens that are masked, ignored, counted from the end, out of range."""
    if rows * vocab > 4e6:
        rows = 70
    rng = np.random.default_rng(vocab)
    z = _logits(rows, vocab, dtype, vocab)
    low = np.finfo(dtype).min
    z[rng.random(z.shape) < 0.3] = -np.inf
    tokens = rng.integers(-vocab, vocab, rows)
    for r in range(rows):
        kind = r % 11
        if kind == 1:
            z[r] = -np.inf
        elif kind == 2:
            z[r] = low
        elif kind == 3:
            z[r], z[r, vocab // 2] = -np.inf, 3.0
        elif kind == 4:
            z[r, vocab - 1] = np.nan
        elif kind == 5:
            z[r, vocab // 3] = np.inf
        elif kind == 6:
            z[r], z[r, 0] = low, -5.0
        elif kind == 7:
            tokens[r] = -100
            z[r] = np.nan
        elif kind == 8:
            tokens[r] = vocab if vocab > 200 else vocab + 7
        elif kind == 9:
            tokens[r] = -vocab - 1
        elif kind == 10:
            z[r] = np.finfo(dtype).max
    tokens[tokens == -100] = np.where(np.arange(rows) % 11 == 7, -100, 0)[tokens == -100]
    _compare(z, tokens, min(7, vocab))
    _compare(z, tokens, 0)


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('vocab', [17, 64, 257, 2050, 4100, 33001, 70000])
@pytest.mark.parametrize('top', [1, 13, 64])
def test_alternatives_of_awkward_orders(vocab, top, dtype):
    """Ties, sorted rows, and rows whose largest values lie where one thread reads them: every period that divides a
    power of two, and runs.  -0 and 0 are equal."""
    top = min(top, vocab)
    j = np.arange(vocab)
    rng = np.random.default_rng(vocab)
    rows = [np.zeros(vocab), j, -j, j % 3, -(j % 7), rng.integers(0, 4, vocab), np.where(j % 2, 0.0, -0.0),
            rng.permutation(vocab) % 50, np.where(j < 1000, 5, 0), np.where(j >= vocab - 100, 5, 0) + j % 2]
    for period in (4, 8, 16, 64, 256, 512, 1024, 2048, 4096, 8192):
        rows.append(np.where(j % period == period // 3, 10 + (j // period) % 37, rng.standard_normal(vocab)))
        rows.append(np.where(j % period < 8, 10 + rng.random(vocab), 0))
    z = (np.stack(rows) / (vocab if dtype == np.float16 and vocab > 60000 else 1)).astype(dtype)
    _compare(z, rng.integers(0, vocab, len(rows)), top, grads=False)


@pytest.mark.parametrize('kept', [0, 1, 2, 5, 30])
@pytest.mark.parametrize('vocab', [40, 3001, 66000])
def test_fewer_possible_tokens_than_alternatives(vocab, kept):
    rng = np.random.default_rng(kept)
    z = np.full((9, vocab), -np.inf, np.float32)
    for r in range(9):
        z[r, rng.choice(vocab, kept, False)] = rng.standard_normal(kept)
    _compare(z, rng.integers(0, vocab, 9), 20)


@pytest.mark.parametrize('kind', [np.int64, np.int32])
def test_token_types_and_leading_dimensions(kind):
    rng = np.random.default_rng(3)
    z = _logits(30, 77, np.float32, 4)
    tokens = rng.integers(-77, 77, 30).astype(kind)
    _compare(z, tokens, 4)
    whole = F.token_log_prob(_tensor(z), _tensor(tokens), top=4)
    cube = F.token_log_prob(_tensor(z.reshape(2, 3, 5, 77)), _tensor(tokens.reshape(2, 3, 5)), top=4)
    assert [c.shape for c in cube] == [(2, 3, 5), (2, 3, 5), (2, 3, 5, 4), (2, 3, 5, 4)]
    for a, b in zip(whole, cube):
        np.testing.assert_array_equal(a.data.get().ravel(), b.data.get().ravel())
    one = F.token_log_prob(_tensor(z[3]), _tensor(np.asarray(tokens[3])), top=2)
    assert [o.shape for o in one] == [(), (), (2,), (2,)]
    np.testing.assert_allclose(one[0].item(), whole[0].data.get()[3], rtol=1e-6)


@pytest.mark.parametrize('vocab', [50, 5001, 60001])
def test_gradients_of_single_outputs(vocab):
    """Each output's gradient alone, and together in one pass."""
    rng = np.random.default_rng(5)
    z, tokens = _logits(6, vocab, np.float32, 6), rng.integers(0, vocab, 6)
    g = [rng.standard_normal(6).astype(np.float32), rng.standard_normal(6).astype(np.float32),
         rng.standard_normal((6, 3)).astype(np.float32)]
    for i in range(3):
        xt = _tensor(z, True)
        got = F.token_log_prob(xt, _tensor(tokens), top=3)
        got[i].backward(_tensor(g[i]))
        want, bound = plain64.token_log_prob_grad(z, tokens, 3, *[v if k == i else None for k, v in enumerate(g)])
        plain64.check(xt.grad.get(), want, bound, f'output {i}')


def test_an_ignored_token_that_counts_from_the_end_elsewhere():
    z = _logits(4, 200, np.float32, 7)
    tokens = np.array([-100, -1, 3, -200])
    _compare(z, tokens, 3)
    _compare(z, tokens, 3, ignore_index=3)
    _compare(z, tokens, 3, ignore_index=-1)


@pytest.mark.parametrize('vocab', [60, 3000])
def test_gradient_against_differences(vocab):
    """L = sum of outputs times constants: (L(z + e v) - L(z - e v)) / 2e.  L is of size 10 with rounding 1e-6, and its
    third derivative of size 10: with e = 1e-2 the quotient is off by 1e-4 + 1e-3 at most, 1e-2 is asked for."""
    rng = np.random.default_rng(8)
    z, tokens = _logits(3, vocab, np.float32, 9), rng.integers(0, vocab, 3)
    g = [rng.standard_normal(3).astype(np.float32), rng.standard_normal(3).astype(np.float32)]
    xt = _tensor(z, True)
    tt.backward(F.token_log_prob(xt, _tensor(tokens)), [_tensor(v) for v in g])
    v = rng.standard_normal(z.shape).astype(np.float32)
    ends = []
    for e in (1e-2, -1e-2):
        out = F.token_log_prob(_tensor((z + np.float32(e) * v).astype(np.float32)), _tensor(tokens))
        ends.append(sum((o.data.get().astype(np.float64) * c).sum() for o, c in zip(out, g)))
    slope = (xt.grad.get().astype(np.float64) * v).sum()
    assert abs((ends[0] - ends[1]) / 2e-2 - slope) <= 1e-2 * max(1.0, abs(slope))


def test_results_repeat_bit_for_bit():
    z, tokens = _logits(90, 45001, np.float16, 10), np.random.default_rng(11).integers(0, 45001, 90)
    first = None
    for _ in range(3):
        xt = _tensor(z, True)
        got = F.token_log_prob(xt, _tensor(tokens), top=10)
        tt.backward(got[:2], [_tensor(np.ones(90, np.float32))] * 2)
        out = [g.data.get() for g in got] + [xt.grad.get()]
        first = first or out
        for a, b in zip(first, out):
            np.testing.assert_array_equal(a, b)


def test_a_changed_input_is_noticed():
    xt = _tensor(_logits(3, 20, np.float32, 12), True)
    y = xt + xt
    got = F.token_log_prob(y, _tensor(np.array([1, 2, 3])))
    F.relu_(y)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        got[0].backward(_tensor(np.ones(3, np.float32)))


def test_no_rows():
    xt = _tensor(np.zeros((0, 12), np.float32), True)
    got = F.token_log_prob(xt, _tensor(np.zeros(0, np.int64)), top=2)
    assert [g.shape for g in got] == [(0,), (0,), (0, 2), (0, 2)]
    got[0].backward(_tensor(np.zeros(0, np.float32)))
    assert xt.grad.shape == (0, 12)


def test_more_than_2_to_the_31_logits():
    """Offsets past 32 bits: float16 logits of 4.4 GB, one block of rows copied over and over on the device."""
    from pytortto_amd import _hip
    vocab, block, copies = 131072, 260, 65
    z = np.tile(_logits(13, vocab, np.float16, 13), (block // 13, 1))
    tokens = np.tile(np.arange(13) * 997, block * copies // 13)
    small, big = hiparray(z), hiparray.empty((block * copies, vocab), np.float16)
    for i in range(copies):
        _hip.call('tt_memcpy_d2d', big.ptr + i * small.nbytes, small.ptr, small.nbytes)
    assert big.size > 2 ** 31
    few = F.token_log_prob(_tensor(z[:13]), _tensor(tokens[:13]), top=3)
    xt = tt.Tensor(big, requires_grad=True, dtype=big.dtype)
    many = F.token_log_prob(xt, _tensor(tokens), top=3)
    for a, b in zip(few, many):
        a, b = a.data.get(), b.data.get()
        for at in (0, block * copies - 13):
            if a.dtype == np.int64:
                np.testing.assert_array_equal(a, b[at:at + 13])
            else:
                np.testing.assert_allclose(a, b[at:at + 13], rtol=2e-5, atol=2e-5)
    ones = np.ones(block * copies, np.float32)
    many[0].backward(_tensor(ones))
    last = hiparray.empty((13, vocab), np.float16)
    _hip.call('tt_memcpy_d2d', last.ptr, xt.grad.ptr + xt.grad.nbytes - last.nbytes, last.nbytes)
    want, bound = plain64.token_log_prob_grad(z[:13], tokens[:13], 0, ones[:13], None, None)
    plain64.check(last.get(), want, plain64.stored(bound, want, np.float16), 'the last rows of dx')


def test_refusals():
    x, t = _tensor(np.zeros((4, 8), np.float32)), _tensor(np.zeros(4, np.int64))
    with pytest.raises(RuntimeError, match='takes logits'):
        F.token_log_prob(x, _tensor(np.zeros(3, np.int64)))
    with pytest.raises(RuntimeError, match='takes logits'):
        F.token_log_prob(_tensor(np.zeros((4, 0), np.float32)), t)
    with pytest.raises(RuntimeError, match='same device'):
        F.token_log_prob(x, tt.tensor(np.zeros(4, np.int64)))
    for top in (-1, 9, 2.0):
        with pytest.raises(ValueError, match='alternatives'):
            F.token_log_prob(x, t, top=top)
    with pytest.raises(ValueError, match='0 to 64 alternatives'):
        F.token_log_prob(_tensor(np.zeros((4, 100), np.float32)), t, top=65)
    with pytest.raises(TypeError, match='logits must be float32 or float16'):
        F.token_log_prob(_tensor(np.zeros((4, 8), np.float64)), t)
    with pytest.raises(TypeError, match='tokens must be int64 or int32'):
        F.token_log_prob(x, _tensor(np.zeros(4, np.int16)))
    from pytortto_amd import _hip
    p = x.data.ptr
    for args, message in (((p, p, p, p, None, None, None, 2, 64, -100, 4, 8, 0), 'unknown type'),
                          ((p, p, p, p, None, None, None, 0, 16, -100, 4, 8, 0), '32 or 64 bits'),
                          ((p, p, p, p, None, None, None, 0, 64, -100, 0, 8, 0), 'rows must be'),
                          ((p, p, p, p, None, None, None, 0, 64, -100, 4, 0, 0), 'vocabulary must have'),
                          ((p, p, p, p, None, None, None, 0, 64, -100, 4, 8, 3), 'null pointer for the alternatives'),
                          ((p, p, p, p, p, p, None, 0, 64, -100, 4, 8, 9), 'alternatives must be'),
                          ((p + 4, p, p, p, None, None, None, 0, 64, -100, 1, 4, 0), '16-byte aligned'),
                          ((p, None, p, p, None, None, None, 0, 64, -100, 4, 8, 0), 'null pointer')):
        with pytest.raises(RuntimeError, match=message):
            _hip.call('tt_token_log_prob_fwd', *args)
