"""GPU: ``F.linear_cross_entropy`` over more positions than one chunk takes, where the blocks that make the weight's gradient also
share its reduction, against the formulas in 64 bits (torch on the device)."""
import numpy as np
import pytest

torch = pytest.importorskip('torch')
import pytortto_amd as tt
from pytortto_amd import _hip

pytestmark = pytest.mark.gpu
F = tt.nn.functional
U = 2.0 ** -24


def _make(rows, width, vocab, half, seed):
    """The last positions have the first eight classes, the others all that follow them: what an earlier chunk adds to a class
    is not what a later one adds."""
    gen = torch.Generator('cuda')
    gen.manual_seed(seed)
    kind = torch.float16 if half else torch.float32
    w = (torch.randn((vocab, width), generator=gen, device='cuda') * width ** -0.5).to(kind)
    target = torch.randint(8, vocab, (rows,), generator=gen, device='cuda')
    target[-rows // 3:] %= 8
    x = torch.empty((rows, width), dtype=kind, device='cuda')
    for i in range(0, rows, 1 << 22):       # (torch's own kernels leave NaN in the middle of 2^29 float16 values)
        some = target[i:i + (1 << 22)]
        x[i:i + (1 << 22)] = torch.randn((len(some), width), generator=gen, device='cuda') + 3.0 * w[some].float()
    target[::11] = -100
    g = torch.rand((rows,), generator=gen, device='cuda') + 0.25
    return x, w, target, g


def _over_rows(p, a):
    """p.T @ a, many rows in parts side by side"""
    parts = len(p) // 16384
    if parts < 32:
        return p.T.contiguous() @ a
    n = parts * 16384
    sums = torch.bmm(p[:n].view(parts, 16384, -1).transpose(1, 2).contiguous(), a[:n].view(parts, 16384, -1)).sum(0)
    return sums + p[n:].T.contiguous() @ a[n:]


def _want(x, w, target, g, half):
    """(losses, dx, dw, bound of dx, bound of dw) with a weight g of each position, 0 for those without a target.

    The bounds, u = 2^-24: logits are off by (32 + 12 + 6 K / 32) u of their terms (K features), so e^z by that times |x| |w|, and G by that
    and twelve roundings more; G of float16 is rounded by 2^-11.  Of dw's reduction a block takes at most 32768 positions one after the
    other, 32 at a time, two roundings for each of three products; 64 blocks' sums and four chunks' are added after it.  An entry of G
    is held to 2^-37 of the largest weight of a position at worst."""
    rows, vocab = len(x), len(w)
    losses, dx, dw = torch.zeros(rows, dtype=torch.float64, device='cuda'), torch.zeros_like(x, dtype=torch.float64), 0.0
    size_x, size_w = torch.zeros_like(dx), 0.0
    w = w.double()
    step = max(1, (1 << 25) // vocab)
    most = 0.0
    for i in range(0, rows, step):
        a, t, kept = x[i:i + step].double(), target[i:i + step].clamp(min=0), target[i:i + step] != -100
        z = a @ w.T.contiguous()
        most = max(most, float((a.abs() @ w.abs().T.contiguous()).max()))
        logp = torch.log_softmax(z, -1)
        losses[i:i + step] = torch.where(kept, -logp.gather(1, t[:, None])[:, 0], 0.0)
        p = logp.exp_()
        p.scatter_add_(1, t[:, None], torch.full((len(t), 1), -1.0, dtype=torch.float64, device='cuda'))
        p *= (g[i:i + step].double() * kept)[:, None]
        dx[i:i + step] = p @ w
        dw = dw + _over_rows(p, a)
        p.abs_()
        size_x[i:i + step] = p @ w.abs()
        size_w = size_w + _over_rows(p, a.abs())
    logit = (44 + 6 * x.shape[1] / 32) * U * most
    gradient = 2 * logit + 12 * U + (2.0 ** -11 if half else 0.0)
    least = 2.0 ** -37 * float(g.max())
    off_x = (gradient + (44 + 6 * vocab / 32) * U) * size_x + least * w.abs().sum(0)
    off_w = (gradient + (44 + 6 * 32768 / 32 + 68) * U) * size_w + least * x.double().abs().sum(0)
    # (a loss is a difference of two such logits, and has a few roundings of its own)
    return losses, dx, dw, 3 * logit + 24 * U, off_x, off_w


def _near(got, want, bound, what, half=False):
    got = torch.as_tensor(got, device='cuda')
    if half:
        assert got.dtype == torch.float16
        bound = bound + 2.0 ** -11 * (want.abs() + bound) + 2.0 ** -25
    off = (got.double() - want).abs()
    worst = int((off - bound).argmax())
    fits = bool((off <= bound).all())
    assert fits, (what, worst, float(off.view(-1)[worst]), float(want.view(-1)[worst]))


def _check(rows, width, vocab, half, reduction, seed=0):
    x, w, target, g = _make(rows, width, vocab, half, seed)
    if reduction != 'none':
        g = torch.ones_like(g) * (1.0 if reduction == 'sum' else 1.0 / float((target != -100).sum()))
    losses, dx, dw, off, off_x, off_w = _want(x, w, target, g, half)
    # (float16 gradients of a scalar loss are trained with a scaled one)
    scale = 1.0 if reduction == 'none' or not half else 2.0 ** -9 if reduction == 'sum' else 1024.0
    torch.cuda.synchronize()
    xt, wt = tt.as_tensor(x, True), tt.as_tensor(w, True)
    loss = F.linear_cross_entropy(xt, wt, tt.as_tensor(target), reduction=reduction)
    loss.backward(tt.as_tensor(g) if reduction == 'none' else tt.as_tensor(torch.full((), scale, device='cuda')))
    _hip.call('tt_sync')            # (torch reads on a stream of its own)
    if reduction == 'none':
        _near(loss.data, losses, off, 'losses')
    else:
        value = float((losses * g).sum())
        assert abs(loss.item() - value) <= off * float(g.sum()) + 2 * U * value
    _near(xt.grad, dx * scale, (off_x + 4 * U * dx.abs()) * scale, 'dx', half)
    _near(wt.grad, dw * scale, (off_w + 4 * U * dw.abs()) * scale, 'dw', half)


# (chunks of 524288 positions of a thousand classes, of 762368 of 701, of 32768 of 16384, of 65536 of 8192)
@pytest.mark.parametrize('half', [False, True], ids=['f32', 'f16'])
@pytest.mark.parametrize('rows,width,vocab,reduction', [
    (1_100_000, 64, 1000, 'none'), (1_100_000, 64, 1000, 'mean'), (526_288, 64, 1000, 'sum'), (60_000, 512, 16384, 'sum'),
    (100_001, 512, 16384, 'none'), (140_000, 256, 8192, 'mean'), (65_600, 256, 8192, 'none')])
def test_shared_reductions_of_several_chunks(rows, width, vocab, reduction, half):
    """Chunks that are shared alike, and a short last one: of fewer shares, of one."""
    _check(rows, width, vocab, half, reduction, rows)


@pytest.mark.parametrize('half', [False, True], ids=['f32', 'f16'])
@pytest.mark.parametrize('width', [3, 66, 130])
def test_rows_of_the_gradient_that_are_not_aligned(width, half):
    _check(900_000, width, 701, half, 'sum', width)
