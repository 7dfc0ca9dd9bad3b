"""GPU: what decides how many threads share a row of logits, from both sides of every limit, and rows laid out against
the search for the best alternatives.  (Comparisons and bounds: the operators' own tests.)"""
import numpy as np
import pytest

from tests import test_gpu_distill as distill
from tests import test_gpu_token_log_prob as logp

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize('dtype', [np.float32, np.float16])


def _packs(dtype):
    return 16 // np.dtype(dtype).itemsize


@BOTH
@pytest.mark.parametrize('packs', [2, 16, 17, 32, 33, 64, 127, 128, 129, 512, 513, 1024, 1025])
@pytest.mark.parametrize('odd', [-1, 0, 1])
def test_packs_of_a_row(packs, odd, dtype):
    vocab, rows = packs * _packs(dtype) + odd, 67
    rng = np.random.default_rng(vocab)
    z = logp._logits(rows, vocab, dtype, vocab)
    tokens = rng.integers(0, vocab, rows)
    tokens[::9] = -100
    logp._compare(z, tokens, 0)
    if odd == 1:
        logp._compare(z, tokens, min(vocab, 4))
    z, teacher, index = distill._inputs(rows, vocab, min(vocab, 9), dtype, vocab)
    index[::7] = -1
    distill._compare(z, teacher, index, 2.0, 'mean')
    distill._compare(z, teacher, index, 1.0, 'none', rng.standard_normal(rows).astype(np.float32))


@pytest.mark.parametrize('vocab,k', [(200, 64), (200, 65), (1500, 64), (1500, 256), (1500, 257), (5000, 1024)])
def test_entries_of_a_row(vocab, k):
    """Numbers of entries from which on more threads take a row; some of one class."""
    z, teacher, index = distill._inputs(50, vocab, k, np.float32, k)
    index[:, k // 2] = index[:, 0]
    index[3, :] = index[3, 0]
    distill._compare(z, teacher, index, 1.0, 'sum')


@BOTH
@pytest.mark.parametrize('top', [31, 32, 33, 64])
def test_numbers_of_alternatives(top, dtype):
    rng = np.random.default_rng(top)
    for rows, vocab in ((70, 90), (70, 3001), (9, 50000)):
        logp._compare(logp._logits(rows, vocab, dtype, top), rng.integers(0, vocab, rows), top, grads=False)


@BOTH
@pytest.mark.parametrize('top', [5, 20, 32, 64])
def test_more_candidates_than_room(top, dtype):
    """All large values lie with as many threads as there are alternatives, whichever way a row is shared; and rows of
    few values, of which many threads hold the largest."""
    n = _packs(dtype)
    for rows, vocab in ((12, 1000 * n + 3), (2100, 1163 * n + 5)):
        rng = np.random.default_rng(vocab)
        j = np.arange(vocab)
        z = rng.standard_normal((rows, vocab)) * 0.5
        for r in range(rows):
            at = (r * vocab) % n                # what a row begins with belongs to a pack in front of it
            pack = (j + at) // n - (at > 0)
            for threads in (64, 256):
                if r % 4 == (threads == 256):
                    z[r] += np.where(pack % threads < top, 6, 0)
            if r % 4 == 2:
                z[r] = rng.integers(0, 3, vocab)
            elif r % 4 == 3:
                z[r] = np.where(pack % 256 < top + 40, 2.0, z[r])
        logp._compare(z.astype(dtype), rng.integers(0, vocab, rows), top, grads=False)


@BOTH
@pytest.mark.parametrize('top', [1, 5, 20, 32, 33])
@pytest.mark.parametrize('packs', [1, 9, 64, 100, 128, 129, 200, 256, 257])
def test_equal_values_in_rows_of_a_wave(packs, top, dtype):
    """More values reach the bound than a wave has room for: equal ones, whose places decide."""
    vocab = packs * _packs(dtype) - (packs > 1)
    rng = np.random.default_rng(packs)
    j = np.arange(vocab)
    low = np.finfo(dtype).min
    rows = [np.zeros(vocab), np.full(vocab, -np.inf), np.full(vocab, low), j % 2, -(j % 3), rng.integers(0, 2, vocab),
            np.where(j < vocab // 2, -np.inf, 1.0), np.where(rng.random(vocab) < 0.1, 3.0, low), np.where(j % 64 < 40, 2.0, 0),
            np.where(j == vocab - 1, 5.0, -np.inf), rng.standard_normal(vocab)]
    z = np.stack(rows).astype(dtype)
    logp._compare(z, rng.integers(0, vocab, len(rows)), min(top, vocab), grads=False)


def test_counters_are_zero_again():
    """Launches of different numbers of blocks in turn, each of which counts its blocks."""
    for rows, vocab in ((1, 40000), (2000, 40), (3, 200000), (33, 9001), (700, 100), (31, 300), (4000, 20)):
        distill._compare(*distill._inputs(rows, vocab, 4, np.float32, rows), 1.0, 'mean')
        logp._compare(logp._logits(rows, vocab, np.float32, rows), np.arange(rows) % vocab, 3, grads=False)
