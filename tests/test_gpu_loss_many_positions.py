"""GPU: ``F.linear_cross_entropy`` over more positions than a launch has threads for, and what scratch memory it takes for them."""
import ctypes

import pytest

torch = pytest.importorskip('torch')
import pytortto_amd as tt
from pytortto_amd import _hip
from tests.test_gpu_loss_chunks import _check, _make

pytestmark = pytest.mark.gpu
F = tt.nn.functional
POSITIONS = (1 << 26) + 77


@pytest.fixture
def scratch():
    """How much scratch memory the library has taken since the test began."""
    torch.cuda.empty_cache()
    _hip.call('tt_empty_cache')
    def taken():
        sizes = [ctypes.c_size_t() for _ in range(3)]
        _hip.call('tt_mem_stats', *[ctypes.byref(n) for n in sizes])
        return sizes[2].value

    yield taken
    _hip.call('tt_empty_cache')
    torch.cuda.empty_cache()


@pytest.mark.parametrize('half,reduction', [(False, 'none'), (True, 'sum')], ids=['f32', 'f16'])
def test_more_positions_than_threads(half, reduction, scratch):
    _check(POSITIONS, 8, 12, half, reduction)
    # logits, features in the products' form once or twice, a sixteenth for all else, and the quarter that the library adds
    assert scratch() <= (4 if half else 6) * 2 ** 30 * 1.0625 * 1.25


@pytest.mark.parametrize('half', [False, True], ids=['f32', 'f16'])
@pytest.mark.parametrize('rows,width', [(POSITIONS, 6), (2_500_000, 1050)])
def test_scores_of_many_positions(rows, width, half, scratch):
    x, w, target, _ = _make(rows, width, 12, half, 3)
    want = 0.0
    for i in range(0, rows, 1 << 20):
        t = target[i:i + (1 << 20)]
        logp = torch.log_softmax(x[i:i + (1 << 20)].double() @ w.double().T.contiguous(), -1)
        want -= float((logp.gather(1, t.clamp(min=0)[:, None])[:, 0] * (t != -100)).sum())
    want /= float((target != -100).sum())
    torch.cuda.synchronize()
    with tt.no_grad():
        got = F.linear_cross_entropy(tt.as_tensor(x), tt.as_tensor(w), tt.as_tensor(target)).item()
    # (a logit's error is (44 + 6 K / 32) units of its terms, whose sizes add up to some tens)
    assert abs(got - want) <= (44 + 6 * width / 32) * 2.0 ** -24 * 100
    assert scratch() <= 2 * 2 ** 30 * 1.25 * 1.25
