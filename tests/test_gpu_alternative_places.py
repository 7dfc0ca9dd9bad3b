"""GPU: the places of the best alternatives lie in memory that their receiver can write; a place outside the row that the
backward pass finds there is passed over, and nothing outside the gradient is written."""
import numpy as np
import pytest

from pytortto_amd import ops
from pytortto_amd.xparray import hiparray
from tests import plain64

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [np.float32, np.float16])
@pytest.mark.parametrize('rows,vocab', [(6, 7), (5, 33), (5, 300), (4, 3001), (3, 20003)])
def test_places_outside_the_row(rows, vocab, dtype):
    rng = np.random.default_rng(vocab)
    z, g = (rng.standard_normal((rows, vocab)) * 2).astype(dtype), rng.standard_normal((rows, 3)).astype(np.float32)
    zeros = np.zeros(rows, np.int64)
    x, tokens = hiparray(z), hiparray(zeros)
    _, entropy, _, places, stats = ops.token_log_prob_fwd(x, tokens, 3, -100, True)
    wrong = places.get()
    wrong[:, 1] = np.resize([vocab, 2 ** 40, -1, -2 ** 40, 2 ** 31 + 1, vocab + 1], rows)
    places.set(wrong)
    dx = ops.token_log_prob_bwd(x, tokens, stats, entropy, places, (None, None, hiparray(g)), 3, -100)
    want, bound = plain64.token_log_prob_grad(z, zeros, 3, None, None, g)
    best = plain64.token_log_prob(z, zeros, 3)[0][3]
    want[np.arange(rows), best[:, 1]] -= g[:, 1]            # all of the second alternative's but its place
    plain64.check(dx.get(), want, plain64.stored(bound, want, dtype))
