"""``SGD`` (``src/tortto/optim/sgd.py``), ``Adam`` and ``AdamW`` (``adam.py``, ``adamw.py``): argument
checks and per-parameter state of the reference; the arithmetic is one kernel launch per parameter
(``_functional.py`` here).  ``Muon`` and ``orthogonalize`` are not in the reference."""
import math
from functools import lru_cache

import numpy as np

from .. import ops
from ..tensor import Tensor
from ..xparray import hiparray
from . import _functional as F
from .optimizer import Optimizer, required


def _check(ok, text, value):
    if not ok:
        raise ValueError(text.format(value))


class SGD(Optimizer):
    def __init__(self, params, lr=required, momentum=0, dampening=0, weight_decay=0, nesterov=False):
        _check(lr is required or lr >= 0.0, 'Invalid learning rate: {}', lr)
        _check(momentum >= 0.0, 'Invalid momentum value: {}', momentum)
        _check(weight_decay >= 0.0, 'Invalid weight_decay value: {}', weight_decay)
        if nesterov and (momentum <= 0 or dampening != 0):
            raise ValueError('Nesterov momentum requires a momentum and zero dampening')
        super().__init__(params, dict(lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay,
                                      nesterov=nesterov))

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault('nesterov', False)

    def step(self):
        for group, members in self._with_grad():
            buffers = [self.state[p].get('momentum_buffer') for p in members]
            F.sgd(members, [p.grad for p in members], buffers, group['weight_decay'], group['momentum'], group['lr'],
                  group['dampening'], group['nesterov'])
            for p, buf in zip(members, buffers):        # created by the first step when momentum != 0
                self.state[p]['momentum_buffer'] = buf


class Adam(Optimizer):
    _rule = staticmethod(F.adam)

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, amsgrad=False):
        _check(lr >= 0.0, 'Invalid learning rate: {}', lr)
        _check(eps >= 0.0, 'Invalid epsilon value: {}', eps)
        for i in (0, 1):
            _check(0.0 <= betas[i] < 1.0, 'Invalid beta parameter at index %d: {}' % i, betas[i])
        _check(weight_decay >= 0.0, 'Invalid weight_decay value: {}', weight_decay)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad))

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:
            group.setdefault('amsgrad', False)

    def _moments(self, p, amsgrad):
        """The parameter's state, created on its first step (adam.py:45-54), with the step advanced."""
        state = self.state[p]
        if not state:
            state['step'] = 0
            names = ('exp_avg', 'exp_avg_sq') + (('max_exp_avg_sq',) if amsgrad else ())
            for name in names:
                state[name] = hiparray.zeros(p.data.shape)
        state['step'] += 1
        return state

    def step(self):
        for group, members in self._with_grad():
            amsgrad = group['amsgrad']
            states = [self._moments(p, amsgrad) for p in members]
            self._rule(members, [p.grad for p in members], [s['exp_avg'] for s in states],
                       [s['exp_avg_sq'] for s in states], [s['max_exp_avg_sq'] for s in states] if amsgrad else [],
                       [s['step'] for s in states], amsgrad, *group['betas'], group['lr'], group['weight_decay'],
                       group['eps'])


class AdamW(Adam):
    _rule = staticmethod(F.adamw)

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, amsgrad=False):
        super().__init__(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad)


COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def _coefficients(values):
    values = tuple(float(v) for v in values)
    if len(values) != 3 or not all(math.isfinite(v) for v in values):
        raise ValueError(f'Newton-Schulz takes three coefficients, got {values}')
    return values


@lru_cache(maxsize=64)
def _grow(a, b, c, steps):
    """Whether coefficients let a singular value out of [0, 1], or what a step multiplies it with, out of the kernels' range."""
    s = np.arange(4097) / 4096.0
    with np.errstate(all='ignore'):
        for _ in range(steps):
            p = b * (s * s) + c * (s * s) * (s * s)
            grows = not (np.abs(p) <= 15.0).all() or not (np.abs(a + p) <= 15.0).all()
            s = s * (a + p)
            if grows or not (np.abs(s) <= 1.9).all():
                return True
    return False


def orthogonalize(matrix, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """The nearest semi-orthogonal matrix, roughly: X / max(|X|, eps) (Frobenius norm), then ``steps`` times
    X <- a X + b (X X^T) X + c (X X^T)^2 X, which brings singular values to about 1 and leaves the singular vectors.  ``matrix`` [rows,
    columns] is a float32 or float16 device tensor, the result a new one of its type, without a graph.  Coefficients that let a
    singular value out of [0, 1] grow past 1.9 are refused."""
    if not isinstance(matrix, Tensor) or matrix.data.__class__ is not hiparray:
        raise RuntimeError('orthogonalize: device (HIP) path only; move the matrix with .cuda() first')
    if matrix.ndim != 2:
        raise RuntimeError(f'orthogonalize takes a matrix, got shape {matrix.shape}')
    if steps.__class__ is not int or not 1 <= steps <= 100:
        raise ValueError(f'orthogonalize takes 1 to 100 steps, got {steps}')
    _check(0.0 < eps <= 1e30, 'Invalid epsilon value: {}', eps)
    return Tensor.on(ops.orthogonalize(matrix.data, steps, _coefficients(coefficients), float(eps)))


_ADJUST = {'original': lambda rows, columns: math.sqrt(max(1.0, rows / columns)),
           'match_rms_adamw': lambda rows, columns: 0.2 * math.sqrt(max(rows, columns))}


class Muon(Optimizer):
    """Momentum, orthogonalised by Newton-Schulz products, for matrices:

        m <- m + (1 - momentum) (g - m)        u = g + momentum (m - g) with ``nesterov``, else m
        p <- p (1 - lr weight_decay) - lr scale orthogonalize(u)

    ``adjust_lr_fn`` names the scale: 'original' sqrt(max(1, rows / columns)), 'match_rms_adamw' 0.2 sqrt(max(rows, columns)).
    Parameters of more than two dimensions are matrices of their first and the others; those of one belong to another
    optimiser."""

    def __init__(self, params, lr=1e-3, weight_decay=0.1, momentum=0.95, nesterov=True, ns_coefficients=COEFFICIENTS, eps=1e-7,
                 ns_steps=5, adjust_lr_fn='original'):
        options = dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov, ns_coefficients=_coefficients(ns_coefficients),
                       eps=eps, ns_steps=ns_steps, adjust_lr_fn=adjust_lr_fn)
        self._check_options(options)
        super().__init__(params, options)

    @staticmethod
    def _check_options(group):
        _check(group['lr'] >= 0.0, 'Invalid learning rate: {}', group['lr'])
        _check(0.0 <= group['momentum'] < 1.0, 'Invalid momentum value: {}', group['momentum'])
        _check(group['weight_decay'] >= 0.0, 'Invalid weight_decay value: {}', group['weight_decay'])
        _check(0.0 < group['eps'] <= 1e30, 'Invalid epsilon value: {}', group['eps'])
        steps, coefficients = group['ns_steps'], _coefficients(group['ns_coefficients'])
        _check(steps.__class__ is int and 1 <= steps <= 100, 'Invalid number of steps: {}', steps)
        _check(group['adjust_lr_fn'] in _ADJUST, 'Invalid adjust_lr_fn: {}', group['adjust_lr_fn'])
        _check(not _grow(*coefficients, steps), 'Newton-Schulz coefficients {} let singular values grow past 1.9', coefficients)
        return coefficients

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups.pop()
        for p in group['params']:
            if p.ndim < 2:
                raise ValueError(f'Muon takes matrices, got a parameter of shape {p.shape}')
        self._check_options(group)
        self.param_groups.append(group)

    def step(self):
        work = []
        for group, members in self._with_grad():
            coefficients = self._check_options(group)       # (they may have been changed, or loaded)
            if members:
                momenta = [self.state[p].get('momentum_buffer') for p in members]
                work.append((group, members, momenta, [F.muon_matrix(p, p.grad, m) for p, m in zip(members, momenta)], coefficients))
        groups = []
        for group, members, momenta, matrices, coefficients in work:
            if None in momenta:
                for p in members:
                    if 'momentum_buffer' not in self.state[p]:
                        self.state[p]['momentum_buffer'] = hiparray.zeros(p.data.shape)
                momenta = [self.state[p]['momentum_buffer'] for p in members]
            arguments = (group['lr'], group['momentum'], group['weight_decay'], int(bool(group['nesterov'])), group['ns_steps'],
                         *coefficients, group['eps'])
            groups.append((members, [p.grad for p in members], momenta, matrices, _ADJUST[group['adjust_lr_fn']], arguments))
        F.muon(groups)
