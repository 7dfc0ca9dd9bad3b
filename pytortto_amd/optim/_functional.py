"""The update rules (``src/tortto/optim/_functional.py``) as fused kernels, a group's parameters in a few launches.
Device parameters only: host tensors belong to tortto's NumPy path and are refused."""
import ctypes
from math import prod

import numpy as np

from .. import _hip, ops
from ..xparray import hiparray

_F32 = np.dtype(np.float32)


def _device(param, *arrays):
    for a in (param.data,) + arrays:
        if a is not None and (a.__class__ is not hiparray or a._dtype != _F32):
            raise RuntimeError('the optimisers of pytortto_amd update float32 device parameters only; move the model '
                               'with .cuda() first')


def sgd(params, d_p_list, momentum_buffer_list, weight_decay, momentum, lr, dampening, nesterov):
    """_functional.py:4-22, all parameters of the group in one call (a few launches)."""
    count = len(params)
    if count == 0:
        return
    first = [0] * count
    for i, param in enumerate(params):
        _device(param, d_p_list[i], momentum_buffer_list[i])
        if momentum != 0 and momentum_buffer_list[i] is None:
            momentum_buffer_list[i] = hiparray.empty(param.data.shape)      # the kernel stores d_p into it (:12-13)
            first[i] = 1
    for param in params:            # written in place: nothing may still depend on the old values
        param.data.own()
    pointers = ctypes.c_void_p * count
    bufs = pointers(*[None if b is None else b.ptr for b in momentum_buffer_list])
    _hip.call('tt_sgd_step_multi_f32', count, pointers(*[p.data.ptr for p in params]),
              pointers(*[g.ptr for g in d_p_list]), bufs, (ctypes.c_size_t * count)(*[p.data.size for p in params]),
              (ctypes.c_int * count)(*first), lr, momentum, dampening, weight_decay, int(bool(nesterov)))


def _adam(params, grads, exp_avgs, exp_avg_sqs, max_exp_avg_sqs, state_steps, amsgrad, beta1, beta2, lr,
          weight_decay, eps, decoupled):
    count = len(params)
    if count == 0:
        return
    for i, param in enumerate(params):
        _device(param, grads[i], exp_avgs[i], exp_avg_sqs[i], max_exp_avg_sqs[i] if amsgrad else None)
    for param in params:            # written in place: nothing may still depend on the old values
        param.data.own()
    pointers = ctypes.c_void_p * count
    vmax = pointers(*[a.ptr for a in max_exp_avg_sqs]) if amsgrad else None
    _hip.call('tt_adam_step_multi_f32', count, pointers(*[p.data.ptr for p in params]),
              pointers(*[g.ptr for g in grads]), pointers(*[a.ptr for a in exp_avgs]),
              pointers(*[a.ptr for a in exp_avg_sqs]), vmax, (ctypes.c_size_t * count)(*[p.data.size for p in params]),
              (ctypes.c_int * count)(*state_steps), lr, beta1, beta2, eps, weight_decay, int(bool(amsgrad)),
              int(decoupled))


def adam(params, grads, exp_avgs, exp_avg_sqs, max_exp_avg_sqs, state_steps, amsgrad, beta1, beta2, lr,
         weight_decay, eps):
    """_functional.py:25-65."""
    _adam(params, grads, exp_avgs, exp_avg_sqs, max_exp_avg_sqs, state_steps, amsgrad, beta1, beta2, lr,
          weight_decay, eps, False)


def adamw(params, grads, exp_avgs, exp_avg_sqs, max_exp_avg_sqs, state_steps, amsgrad, beta1, beta2, lr,
          weight_decay, eps):
    """_functional.py:68-119."""
    _adam(params, grads, exp_avgs, exp_avg_sqs, max_exp_avg_sqs, state_steps, amsgrad, beta1, beta2, lr,
          weight_decay, eps, True)


def muon_matrix(param, grad, momentum):
    """(rows, columns) of a parameter, the first dimension and all others (a convolution's output channels and its taps), whose gradient
    and momentum (or None, of a first step) fit it, and that fits the kernels (the C ABI takes ints)."""
    _device(param, grad, momentum)
    shape = param.data._shape
    if grad._shape != shape or (momentum is not None and momentum._shape != shape):
        raise RuntimeError(f"a gradient and a momentum are of their parameter's shape {shape}, got {grad._shape}"
                           + ('' if momentum is None else f' and {momentum._shape}'))
    rows, columns = shape[0], prod(shape[1:])
    if rows > ops.MOST_ROWS or columns > ops.MOST_ROWS or rows * columns > 1 << 32:
        ops._check_products('muon', (rows, ops.MOST_ROWS, 'rows'), (columns, ops.MOST_ROWS, 'columns'), (rows * columns, 1 << 32, 'values'))
    return rows, columns


def muon(groups):
    """The matrices of a group share their launches.  ``groups`` holds (params, grads, momenta, matrices, adjust, arguments) of each,
    the matrices as ``muon_matrix`` has them.  What the library may refuse, and all memory, comes before the first parameter moves: a step
    that fails can be made again."""
    for params, _, momenta, _, _, _ in groups:
        for param, m in zip(params, momenta):       # written in place: nothing may still depend on the old values
            param.data.own()
            m.own()
    calls = []
    for params, grads, momenta, matrices, adjust, arguments in groups:
        rest, at = [k for k, (rows, columns) in enumerate(matrices) if rows and columns], [param.data.ptr for param in params]
        while rest:
            now, later = rest, []
            if len(set(at)) != len(at):
                # (a parameter that comes twice, or another on the same memory, is stepped again afterwards)
                seen, now = set(), []
                for k in rest:
                    (later if at[k] in seen else now).append(k)
                    seen.add(at[k])
            count = len(now)
            pointers, ints = ctypes.c_void_p * count, ctypes.c_int * count
            tables = (pointers(*[at[k] for k in now]), pointers(*[grads[k].ptr for k in now]), pointers(*[momenta[k].ptr for k in now]))
            calls.append((count, tables, (ints(*[matrices[k][0] for k in now]), ints(*[matrices[k][1] for k in now]),
                                          (ctypes.c_double * count)(*[adjust(*matrices[k]) for k in now]), *arguments)))
            rest = later
    if len(calls) > 1:
        for count, _, arguments in calls:       # (without tables: the scratch memory that the call will need)
            _hip.call('tt_muon_step_multi_f32', count, None, None, None, *arguments)
    for count, tables, arguments in calls:
        _hip.call('tt_muon_step_multi_f32', count, *tables, *arguments)
