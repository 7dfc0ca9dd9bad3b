"""Layer normalisation, token log probabilities and distillation in 64 bits, written from their formulas, and how far a
float32 evaluation may be from them.

The bounds: u = 2^-24 is float32's rounding.  A sum of n terms by a kernel whose threads each add at most n / 64 of them
one after the other (n / 256 from 4096 on) and then join in a tree is off by at most u (n / 64 + 16) sum |terms|; the few
roundings around it make it ``chain(n)`` u.  A float16 result adds half a unit of its last place."""
import numpy as np

U = 2.0 ** -24


def chain(n):
    return 24 + n / (256 if n >= 4096 else 64)


def stored(bound, value, dtype):
    """``bound`` of a float32 result once it is stored as ``dtype``."""
    if np.dtype(dtype) == np.float16:
        return bound + 2.0 ** -11 * (np.abs(value) + bound) + 2.0 ** -25
    return bound


def check(got, want, bound, what=''):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    finite = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    np.testing.assert_array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)], err_msg=what)
    off = np.abs(got - want)[finite]
    most = np.broadcast_to(bound, want.shape)[finite]
    worst = np.argmax(off - most) if off.size else 0
    assert not off.size or off[worst] <= most[worst], \
        f'{what}: off by {off[worst]:.3g} where {most[worst]:.3g} is allowed (value {want[finite][worst]:.6g})'


# ---- layer normalisation ---------------------------------------------------------------------------

def layer_norm(x, w, b, eps):
    """(y, bound, n, rstd, bound of n) of rows [R, D]"""
    x = x.astype(np.float64)
    w, b = (np.full(x.shape[1], v) if a is None else a.astype(np.float64) for a, v in ((w, 1.0), (b, 0.0)))
    m = x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt(((x - m) ** 2).mean(1, keepdims=True) + eps)
    n = (x - m) * r
    y = n * w + b
    # the mean is off by chain u max|x|, which moves n by that times rstd; rstd itself is off by chain u
    off = U * chain(x.shape[1]) * (np.abs(x).max(1, keepdims=True) * r + np.abs(n))
    return y, off * np.abs(w) + 4 * U * (np.abs(y) + np.abs(b)), n, r, off


def layer_norm_grad(x, dy, w, eps):
    """((dx, dw, db), their bounds)"""
    _, _, n, r, off = layer_norm(x, w, None, eps)
    dy = dy.astype(np.float64)
    h = dy * (1.0 if w is None else w.astype(np.float64))
    rows, d = n.shape
    mh, mhn = h.mean(1, keepdims=True), (h * n).mean(1, keepdims=True)
    dx = r * (h - mh - n * mhn)
    ah = np.abs(h).mean(1, keepdims=True)
    sums = U * chain(d) * (ah + np.abs(n) * np.abs(h * n).mean(1, keepdims=True))
    bound = r * (sums + off * np.abs(mhn) + np.abs(n) * (np.abs(h) * off).mean(1, keepdims=True)
                 + 8 * U * (np.abs(h) + np.abs(mh) + np.abs(n * mhn))) + U * chain(d) * np.abs(dx)
    # a thread adds up to every eighth row before the partial sums are joined
    down = U * (24 + rows / 8)
    return ((dx, (dy * n).sum(0), dy.sum(0)),
            (bound, down * np.abs(dy * n).sum(0) + (np.abs(dy) * off).sum(0), down * np.abs(dy).sum(0)))


# ---- logits ----------------------------------------------------------------------------------------

def _softmax(z):
    """(log probabilities, probabilities, z - max, poisoned, empty) of rows; an empty row has log probabilities -inf"""
    z = z.astype(np.float64)
    poisoned = (np.isnan(z) | (z == np.inf)).any(1, keepdims=True)
    m = np.where(poisoned, 0.0, np.where(np.isnan(z), 0.0, z).max(1, keepdims=True))
    empty = m == -np.inf
    with np.errstate(invalid='ignore', divide='ignore', over='ignore'):
        d = z - np.where(empty, 0.0, m)
        s = np.exp(d).sum(1, keepdims=True)
        logp = np.where(empty, -np.inf, d - np.log(s))
        logp = np.where(poisoned, np.nan, logp)
        return logp, np.where(empty, 0.0, np.exp(logp)), d, poisoned, empty


def _finite(v):
    return np.where(np.isfinite(v), v, 0.0)


def token_log_prob(z, tokens, top, ignore_index=-100):
    """(values, bounds): logp, entropy, top_logp, top_index (the last without a bound)"""
    rows, v = z.shape
    logp, p, d, poisoned, empty = _softmax(z)
    ignored = (tokens == ignore_index)
    t = np.where(tokens < 0, tokens + v, tokens)
    bad = ((t < 0) | (t >= v)) & ~ignored
    at = np.clip(np.where(ignored, 0, t), 0, v - 1)[:, None]
    mine = np.take_along_axis(logp, at, 1)[:, 0]
    mine = np.where(ignored, 0.0, np.where(bad, np.nan, mine))
    with np.errstate(invalid='ignore'):
        entropy = -np.where(p > 0, p * logp, np.where(np.isnan(p), np.nan, 0.0)).sum(1)
    spread = np.where(p > 0, p * np.abs(_finite(d)), 0.0).sum(1)
    entropy = np.where(ignored, 0.0, entropy)
    order = np.argsort(-np.where(np.isnan(z), 0, z).astype(np.float64), axis=1, kind='stable')[:, :top]
    best = np.where(ignored[:, None], 0.0, np.take_along_axis(logp, order, 1))
    order = np.where(ignored[:, None] | poisoned, -1, order)
    c = U * chain(v)
    return ((mine, entropy, best, order),
            (c + 4 * U * np.abs(_finite(mine)), 2 * c * (1 + spread), c + 4 * U * np.abs(_finite(best))))


def token_log_prob_grad(z, tokens, top, g_logp, g_entropy, g_top, ignore_index=-100):
    rows, v = z.shape
    logp, p, d, poisoned, empty = _softmax(z)
    (_, entropy, _, order), (_, off_entropy, _) = token_log_prob(z, tokens, top, ignore_index)
    ignored = (tokens == ignore_index)[:, None]
    t = np.where(tokens < 0, tokens + v, tokens)[:, None]
    bad = ((t < 0) | (t >= v)) & ~ignored
    zero = np.zeros(rows)
    a, h = ((zero if g is None else g.astype(np.float64))[:, None] for g in (g_logp, g_entropy))
    g = np.zeros((rows, top)) if g_top is None else g_top.astype(np.float64)
    total, size = a + g.sum(1, keepdims=True), np.abs(a) + np.abs(g).sum(1, keepdims=True)
    ln, H = np.maximum(_finite(logp), -200.0), _finite(entropy)[:, None]
    dz = -p * (total + h * (ln + H))
    one = np.zeros((rows, v))
    np.add.at(one, (np.arange(rows)[:, None], np.clip(t, 0, v - 1)), np.where(bad | ignored, 0.0, a))
    np.add.at(one, (np.arange(rows)[:, None], np.clip(order, 0, v - 1)), g)
    c = U * (chain(v) + 8 + 4 * np.abs(ln))
    bound = p * (c * (size + np.abs(h) * (np.abs(ln) + np.abs(H))) + np.abs(h) * (c + off_entropy[:, None])) \
        + 4 * U * (1 + top) * (np.abs(dz) + p * size + np.abs(one)) + 1e-38
    dz = dz + one
    dz = np.where(ignored | empty, 0.0, np.where(poisoned | (bad & (g_logp is not None)), np.nan, dz))
    return dz, np.broadcast_to(_finite(bound), dz.shape)


def distill(z, teacher, index, temperature, reduction, g=None):
    """((loss, its bound), (dz, its bound)); ``g``: the gradient of a loss for each row"""
    rows, v = z.shape
    k = index.shape[1]
    t = float(temperature)
    te = np.where(index < 0, -np.inf, np.where(index >= v, np.nan, teacher.astype(np.float64) / t))
    logq, q, dq, bad, none = _softmax(te)
    none = none[:, 0]
    logp, p, d, poisoned, empty = _softmax(z.astype(np.float64) / t)
    at = np.clip(index, 0, v - 1)
    picked = np.take_along_axis(logp, at, 1)
    with np.errstate(invalid='ignore'):
        loss = t * t * np.where(q != 0, q * (logq - picked), 0.0).sum(1)
        size = t * t * np.where(q != 0, q * (np.abs(_finite(logq)) + np.abs(_finite(picked)) + 1), 0.0).sum(1)
    loss = np.where(none, 0.0, loss)
    off = 2 * U * (chain(v) + chain(k) + 8) * _finite(size)
    count = (~none).sum()
    scale = 1.0
    if reduction != 'none':
        scale = 1.0 / count if reduction == 'mean' else 1.0
        with np.errstate(invalid='ignore'):
            loss, off = np.asarray(loss.sum() * scale), np.asarray(off.sum() * scale + 4 * U * np.abs(_finite(loss)).sum() * scale)
    gain = (t * scale * (np.ones(rows) if g is None else g.astype(np.float64)))[:, None]
    taken = np.zeros((rows, v))
    np.add.at(taken, (np.arange(rows)[:, None], at), _finite(q))
    dz = gain * (p - taken)
    c = U * (chain(v) + chain(k) + 8)
    ln = np.maximum(_finite(logp), -200.0)
    offq = np.zeros((rows, v))
    np.add.at(offq, (np.arange(rows)[:, None], at), _finite(q) * 4 * U * np.abs(np.maximum(_finite(logq), -200.0)))
    bound = np.abs(gain) * (p * (c + 4 * U * np.abs(ln)) + taken * c + offq) + 4 * U * np.abs(dz) + 1e-38
    dead = none[:, None] | empty
    dz = np.where(dead, 0.0, np.where(poisoned | bad, np.nan, dz))
    return (loss, off), (dz, _finite(bound))
