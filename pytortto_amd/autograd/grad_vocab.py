"""Autograd functions of models over a vocabulary: ``LayerNorm`` (interface of ``src/tortto/autograd/grad_nn.py:993-1052``),
``TokenLogProb``, ``DistillLoss`` and ``LinearCrossEntropy`` (not in the reference).  Device tensors only, float32 or float16; parameters,
losses and all statistics are float32."""
import math
from math import prod

from .. import ops
from ..tensor import Tensor
from ..xparray import hiparray
from .function import Function
from .grad_mode import is_grad_enabled
from .grad_nn import _device_only
from .helper import build_links


def _same_device(name, *data):
    for d in data:
        if d is not None and d.__class__ is not hiparray:
            raise RuntimeError(f'{name}: expected all tensors to be on the same device')


class LayerNorm(Function):
    @staticmethod
    def forward(ctx, *inputs, **params):
        xt0, xt1, xt2 = inputs   # input, weight, bias
        xd0 = xt0.data
        shape, eps = tuple(params['normalized_shape']), params['eps']
        _device_only('layer_norm', xd0)
        w = None if xt1 is None else xt1.data
        b = None if xt2 is None else xt2.data
        _same_device('layer_norm', w, b)
        if not shape or xd0._shape[-len(shape):] != shape:
            raise RuntimeError(f'Given normalized_shape={list(shape)}, expected input with shape '
                               f'[*{"".join(f", {n}" for n in shape)}], but got input of size {list(xd0.shape)}')
        width = prod(shape)
        if width == 0:
            raise RuntimeError(f'layer_norm needs at least one value to normalise over, got {list(shape)}')
        if (w is not None and w._shape != shape) or (b is not None and b._shape != shape):
            name, d = ('weight', w) if w is not None and w._shape != shape else ('bias', b)
            raise RuntimeError(f'Expected {name} to be of same shape as normalized_shape, but got {name} of shape '
                               f'{list(d.shape)} and normalized_shape = {list(shape)}')
        keep = ctx.requires_grad and is_grad_enabled()
        yd0, stats = ops.layer_norm_fwd(xd0, w, b, width, eps, keep)
        yt0 = build_links(yd0, grad_fn=ctx)
        if keep:
            ctx.save_for_backward(xt0, xt1)
            ctx.params = {'stats': stats, 'shape': shape}
        return yt0

    @staticmethod
    def backward(ctx, *grad_outputs):
        gd0, = grad_outputs
        xd0, w = ctx.saved_tensors
        return ops.layer_norm_bwd(xd0, gd0, w, ctx.params['stats'], ctx.params['shape'], ctx.needs_input_grad)


class TokenLogProb(Function):
    @staticmethod
    def forward(ctx, *inputs, **params):
        xt0, = inputs
        xd0, tokens, top = xt0.data, params['tokens'], params['top']
        _device_only('token_log_prob', xd0)
        td0 = tokens.data
        _same_device('token_log_prob', td0)
        if xd0.ndim == 0 or td0.shape != xd0.shape[:-1] or xd0.shape[-1] == 0:
            raise RuntimeError(f'token_log_prob takes logits [..., V] and tokens [...], got {xd0.shape} and {td0.shape}')
        most = min(ops.MOST_ALTERNATIVES, xd0.shape[-1])
        if top.__class__ is not int or not 0 <= top <= most:
            raise ValueError(f'token_log_prob returns 0 to {most} alternatives here, got top={top}')
        keep = ctx.requires_grad and is_grad_enabled()
        logp, entropy, top_logp, top_index, stats = ops.token_log_prob_fwd(xd0, td0, top, params['ignore_index'], keep)
        values = (logp, entropy, top_logp) if top else (logp, entropy)
        outputs = tuple(build_links(y, grad_fn=ctx, _output_idx=i) for i, y in enumerate(values))
        index = Tensor.on(top_index) if top else None
        if keep:
            # (of the entropy its array alone: the output itself hangs on this node, and the two would keep each other)
            ctx.save_for_backward(xt0, tokens, Tensor.on(entropy), index)
            ctx.params['stats'] = stats
        return outputs if index is None else outputs + (index,)

    @staticmethod
    def backward(ctx, *grad_outputs):
        x, tokens, entropy, index = ctx.saved_tensors
        p = ctx.params
        gradients = (grad_outputs + (None,))[:3]
        return ops.token_log_prob_bwd(x, tokens, p['stats'], entropy, index, gradients, p['top'], p['ignore_index'])


class DistillLoss(Function):
    @staticmethod
    def forward(ctx, *inputs, **params):
        xt0, = inputs
        xd0, teacher, index = xt0.data, params['teacher'], params['index']
        _device_only('distill_loss', xd0)
        td0, id0 = teacher.data, index.data
        _same_device('distill_loss', td0, id0)
        if xd0.ndim == 0 or xd0.shape[-1] == 0 or td0.shape != id0.shape or id0.ndim != xd0.ndim \
                or id0.shape[:-1] != xd0.shape[:-1]:
            raise RuntimeError(f'distill_loss takes logits [..., V] and a teacher\'s logits and indexes [..., K], got '
                               f'{xd0.shape}, {td0.shape} and {id0.shape}')
        if not 1 <= id0.shape[-1] <= ops.MOST_TEACHER_ENTRIES:
            raise ValueError(f'distill_loss takes 1 to {ops.MOST_TEACHER_ENTRIES} entries of the teacher, got '
                             f'{id0.shape[-1]}')
        if params['reduction'] not in ('none', 'sum', 'mean'):
            raise ValueError(f'{params["reduction"]} is not a valid value for reduction')
        if not (math.isfinite(params['temperature']) and 1e-6 <= params['temperature'] <= 1e6):
            raise ValueError(f'the temperature must be in 1e-6 to 1e6, got {params["temperature"]}')
        keep = ctx.requires_grad and is_grad_enabled()
        yd0, stats, count, dx = ops.distill_fwd(xd0, td0, id0, params['temperature'], params['reduction'], keep)
        yt0 = build_links(yd0, grad_fn=ctx)
        if keep:
            ctx.save_for_backward(xt0, teacher, index)
            ctx.params.update(stats=stats, count=count, dx=dx)
        return yt0

    @staticmethod
    def backward(ctx, *grad_outputs):
        gd0, = grad_outputs
        x, teacher, index = ctx.saved_tensors
        p = ctx.params
        return ops.distill_bwd(x, teacher, index, p['stats'], p['count'], gd0, p['dx'], p['temperature'], p['reduction'])


class LinearCrossEntropy(Function):
    """The gradients of a scalar loss are made with it, while the logits are there: a backward pass would have to make those
    again, a third of its products more."""

    @staticmethod
    def forward(ctx, *inputs, **params):
        xt0, xt1 = inputs   # input, weight
        xd0, wd0, target, reduction = xt0.data, xt1.data, params['target'], params['reduction']
        _device_only('linear_cross_entropy', xd0)
        td0 = target.data
        _same_device('linear_cross_entropy', wd0, td0)
        if xd0.ndim == 0 or wd0.ndim != 2 or td0.shape != xd0.shape[:-1] or xd0.shape[-1] != wd0.shape[1] or 0 in wd0.shape:
            raise RuntimeError(f'linear_cross_entropy takes input [..., H], weight [V, H] and target [...], got {xd0.shape}, '
                               f'{wd0.shape} and {td0.shape}')
        if wd0.dtype != xd0.dtype:
            raise TypeError(f'linear_cross_entropy takes input and weight of one type, got {xd0.dtype} and {wd0.dtype}')
        if reduction not in ('none', 'sum', 'mean'):
            raise ValueError(f'{reduction} is not a valid value for reduction')
        keep = ctx.requires_grad and is_grad_enabled()
        need = ctx.needs_input_grad if keep else (False, False)
        yd0, dx, dw = ops.linear_cross_entropy_fwd(xd0, wd0, td0, params['ignore_index'], reduction, need)
        yt0 = build_links(yd0, grad_fn=ctx)
        if keep:
            ctx.save_for_backward(xt0, xt1, target)
            ctx.params.update(dx=dx, dw=dw)
        return yt0

    @staticmethod
    def backward(ctx, *grad_outputs):
        gd0, = grad_outputs
        x, w, target = ctx.saved_tensors
        p = ctx.params
        if p['reduction'] == 'none':
            return ops.linear_cross_entropy_bwd(x, w, target, gd0, p['ignore_index'], ctx.needs_input_grad)
        return tuple(None if a is None else ops.scaled_gradient(a, gd0, x.dtype) for a in (p['dx'], p['dw']))
