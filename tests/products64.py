"""A vocabulary's loss from features and weights, and Newton-Schulz orthogonalisation, in 64 bits, written from their
formulas, and how far an evaluation by products of float16 terms with float32 sums may be from them.

Products.  u = 2^-24.  Float32 operands are two terms each: the first is off by at most 2^-11 of the value, the second by 2^-11 of
that, so the two hold the value to 2^-22 of itself, or to 2^-25 of the scaled unit where the second is subnormal; the
largest value of what is scaled together is at least 2^13 units, so that is 2^-38 of it.  Left out is lo lo, 2^-22 of a
term.  Together 3 2^-22 = 12 u of every term, and the floor of either operand.  A sum of K terms comes in chunks of 32, three times each
for two terms: 3 K / 32 additions to a running sum, off by u of it each, or 2 u where the unit truncates, and 32 u for the additions
within a chunk."""
import numpy as np

U = 2.0 ** -24


def product(a, b, terms, floor_a=0.0, floor_b=0.0):
    """(a @ b.T, how far off it may be); floors: 2^-38 of what each value of the operand is scaled with"""
    size = np.abs(a) @ np.abs(b).T
    k = a.shape[1]
    off = U * (32 + 6 * k / 32 + (12 if terms == 2 else 0)) * size
    if terms == 2:
        off = off + (np.broadcast_to(floor_a, a.shape) @ np.abs(b).T + np.abs(a) @ np.broadcast_to(floor_b, b.shape).T)
    return a @ b.T, off


def _floor(a):
    return 2.0 ** -38 * np.abs(a).max(1, keepdims=True)


def linear_cross_entropy(x, w, target, reduction, g=None, scale=1.0, ignore_index=-100):
    """((loss, bound), (dx, bound), (dw, bound)), the gradients before they are stored; g: a weight of each row's loss;
    scale: the incoming gradient of a scalar loss.  Rows without a target count as zeros, as they do in a padded batch."""
    terms = 2 if x.dtype == np.float32 else 1
    kept = target != ignore_index
    x = np.where(kept[:, None], x, 0).astype(np.float64)
    w = w.astype(np.float64)
    rows, v = len(x), len(w)
    t = np.where(target < 0, target + v, target)
    bad = kept & ((t < 0) | (t >= v))
    at = np.where(kept & ~bad, t, 0)
    z, off_z = product(x, w, terms, _floor(x), _floor(w))
    m = z.max(1, keepdims=True)
    d = z - m
    s = np.exp(d).sum(1, keepdims=True)
    logp = d - np.log(s)
    p = np.exp(logp)
    # of the exponentials (their arguments in bits are rounded twice, v_exp_f32 is good to a unit), and of sums: 16 values
    # in a row, 64 threads' blocks of 64 columns in a row, trees between them
    weight = p * (4 + 4 * np.abs(d))
    off_lse = (p * off_z).sum(1) + U * (weight.sum(1) + 40 + v / 4096)
    own = np.take_along_axis(logp, at[:, None], 1)[:, 0]
    loss = np.where(kept, -own, 0.0)
    off = np.where(kept, off_lse + np.take_along_axis(off_z, at[:, None], 1)[:, 0]
                   + 8 * U * (np.abs(own) + np.abs(np.log(s[:, 0])) + np.abs(np.take_along_axis(d, at[:, None], 1)[:, 0])), 0.0)
    loss = np.where(bad, np.nan, loss)
    count = kept.sum()
    gain = 1.0 if reduction != 'mean' else 1.0 / count if count else 0.0
    row = (np.ones(rows) if g is None else g.astype(np.float64))
    dz = p * row[:, None]
    one = np.zeros((rows, v))
    one[np.arange(rows), at] = 1.0
    off_dz = np.abs(dz) * (off_z + off_lse[:, None] + U * (8 + 4 * np.abs(d)))
    dz = dz - one * row[:, None]
    # the target's own entry is expm1(-loss)
    off_dz = np.where(one > 0, np.abs(row[:, None]) * (np.exp(np.minimum(own, 0.0)) * off + 4 * U)[:, None], off_dz)
    dz, off_dz = (np.where(kept[:, None], a, 0.0) for a in (dz, off_dz))
    # stored with W's and x's scales on top; the largest of all is at least 2^13 units when a row's largest gradient is its g
    # (each scale is a power of two within a factor of two, 2^-25 of 2^14 and two factors of two; a row of zeros has the largest)
    sw = np.abs(w).max(1) if terms == 2 else np.ones(v)
    sx = np.abs(x).max(1) if terms == 2 else kept.astype(float)
    most = max(sw.max() * (sx * np.abs(row)).max(), 1e-300)
    sw, sx = (np.where(a > 0, a, max(a.max(), 1e-150)) for a in (sw, sx))
    floor = np.where(kept[:, None], 2.0 ** -36 * most / (sx[:, None] * sw), 0.0)
    if terms == 1:
        off_dz = off_dz + 2.0 ** -11 * np.abs(dz) + floor
        floor = np.zeros_like(floor)
    kind = terms
    dx, off_x = product(dz, w.T, kind, floor, 2.0 ** -38 * np.abs(w).max(1)[None, :])
    dw, off_w = product(dz.T, x.T, kind, floor.T, 2.0 ** -38 * np.abs(x).max(1)[None, :])
    off_x, off_w = off_x + off_dz @ np.abs(w), off_w + off_dz.T @ np.abs(x)
    if reduction != 'none':
        loss, off = np.asarray(loss.sum()), np.asarray(off.sum())
        loss, off = (loss * gain, off * gain + 2 * U * np.abs(np.nan_to_num(loss)) * gain) if count or reduction == 'sum' else (np.asarray(np.nan), np.asarray(0.0))
    factor = gain * scale
    out = [(loss, off + 1e-45)]
    for value, bound in ((dx, off_x), (dw, off_w)):
        value = value * factor
        if bad.any():
            value = np.full_like(value, np.nan)
        out.append((value, bound * abs(factor) + 4 * U * np.abs(np.nan_to_num(value)) + 1e-44))
    if bad.any():       # (a row of dx is its own)
        dx = np.where(bad[:, None], np.nan, dx * factor)
        out[1] = (dx, off_x * abs(factor) + 4 * U * np.abs(np.nan_to_num(dx)) + 1e-44)
    return out


def newton_schulz(x, steps, coefficients, eps):
    """(the result, how far off it may be in the Frobenius norm, before it is stored)

    With |X| <= 1 in the spectral norm and the odd polynomial q(s) = a s + b s^3 + c s^5, a difference dX before a step is one
    of at most L |dX| behind it (Frobenius norm), L the largest of (q(s) -+ q(t)) / (s -+ t): on the spectrum's interval at most
    the largest |q'| and |q(s) / s|.  A step itself adds, with every product's terms held as ``product`` has it, and k = m or n its
    length, |X| the spectral norm s and f the Frobenius norm:
      X stored             2^-22 f + floor
      A = X X^T            c_n s f + its storing, then through b A + c A A times X:  (|b| + 2 |c| s^2) s
      A A, b A + c A A     c_m s^2 |A|_F |c| + their storing, times s
      the last product     c_m |b A + c A A| f
    (the norm of |X| |X|^T is taken for that of X X^T's terms: at most the Frobenius norms' product)."""
    a, b, c = coefficients
    x = x.astype(np.float64)
    x = x / max(np.linalg.norm(x), eps)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    m, n = x.shape
    def chunks(k):
        return U * (32 + 6 * k / 32 + 12)
    floor = 2.0 ** -39 * np.sqrt(float(m) * n)
    floor_a = 2.0 ** -37 * m
    off = (4 * U) * np.linalg.norm(x) + floor
    top = 1.0
    for _ in range(steps):
        s = np.linspace(0.0, top, 2001)
        slope = np.abs(a + 3 * b * s ** 2 + 5 * c * s ** 4).max()
        slope = max(slope, np.abs(a + b * s ** 2 + c * s ** 4).max())
        f = np.linalg.norm(x)
        gram = x @ x.T
        size = np.linalg.norm(np.abs(x) @ np.abs(x).T)
        off_gram = chunks(n) * size + 4 * U * np.linalg.norm(gram) + floor_a
        poly = b * gram + c * (gram @ gram)
        off_poly = abs(c) * chunks(m) * np.linalg.norm(np.abs(gram) @ np.abs(gram)) + 8 * U * (abs(b) + abs(c)) * np.linalg.norm(gram) + floor_a * 4
        off_poly += off_gram * (abs(b) + 2 * abs(c) * np.linalg.norm(gram, 2))
        spectral = np.linalg.norm(x, 2)
        new = a * x + poly @ x
        off = slope * off + off_poly * spectral + chunks(m) * np.linalg.norm(np.abs(poly) @ np.abs(x)) \
            + 4 * U * (abs(a) * f + np.linalg.norm(new)) + 2 * floor
        x = new
        top = max(top, spectral * slope, 1.3)
        top = min(top, 1.9)
    return (x.T if tall else x), off
