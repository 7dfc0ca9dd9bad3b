"""Functional wrappers in front of the hot path (``src/tortto/nn/functional.py:80-101``,
``:119-121``) plus the activations (:6-19), ``max_pool2d`` (:104-107) and the head (``nll_loss`` :38-39,
``log_softmax`` :46-47, ``linear`` :54-63): argument plumbing only."""
from ..autograd.grad_fcn import Squeeze, Unsqueeze
from ..autograd.grad_nn import (BatchNorm, Convolution, LeakyRelu, LogSoftmax, MaxPool2DWithIndices, NllLoss, Relu,
                                TransposedConvolution)
from ..autograd.grad_vocab import DistillLoss, LayerNorm, TokenLogProb


def pad(input, pad, mode='constant', value=0.0):
    raise NotImplementedError("TODO: Currently only support mode='constant'" if mode != 'constant' else
                              'F.pad is outside the convolution / BatchNorm path of this build')


def conv2d(input, weight, bias=None, stride=(1, 1), padding=(0, 0), dilation=(1, 1), groups=1):
    low_dim = input.ndim == 3
    if low_dim:
        input = Unsqueeze.apply(input, dim=0)
    result = Convolution.apply(input, weight, bias, stride=stride, padding=padding, dilation=dilation,
                               groups=groups)
    if low_dim:
        result = Squeeze.apply(result, dim=0)
    return result


def conv_transpose2d(input, weight, bias=None, stride=(1, 1), padding=(0, 0), output_padding=(0, 0), groups=1,
                     dilation=(1, 1)):
    low_dim = input.ndim == 3
    if low_dim:
        input = Unsqueeze.apply(input, dim=0)
    result = TransposedConvolution.apply(input, weight, bias, stride=stride, padding=padding,
                                         output_padding=output_padding, dilation=dilation, groups=groups)
    if low_dim:
        result = Squeeze.apply(result, dim=0)
    return result


def batch_norm(input, running_mean, running_var, weight=None, bias=None, training=False, momentum=0.1, eps=1e-5,
               _count_batch=None):
    """``_count_batch`` is not in the reference's signature (functional.py:119-121): the module hands
    its ``num_batches_tracked`` buffer over so that the training kernel increments it (the module's
    ``+= 1``, nn/modules/batchnorm.py:66) instead of a launch of its own."""
    return BatchNorm.apply(input, weight, bias, running_mean=running_mean, running_var=running_var,
                           training=training, momentum=momentum, eps=eps, count_batch=_count_batch)


def relu(input, inplace=False):
    return Relu.apply(input, inplace=inplace)


def relu_(input):
    return Relu.apply(input, inplace=True)


def leaky_relu(input, negative_slope=0.01, inplace=False):
    return LeakyRelu.apply(input, negative_slope=negative_slope, inplace=inplace)


def leaky_relu_(input, negative_slope=0.01):
    return LeakyRelu.apply(input, negative_slope=negative_slope, inplace=True)


def max_pool2d(input, kernel_size, stride=(1, 1), padding=(0, 0), dilation=(1, 1), ceil_mode=False,
               return_indices=False):
    return MaxPool2DWithIndices.apply(input, kernel_size=kernel_size, stride=stride, padding=padding,
                                      dilation=dilation, ceil_mode=ceil_mode, return_indices=return_indices)


def nll_loss(input, target, weight=None, ignore_index=-100, reduction='mean'):
    return NllLoss.apply(input, target=target, weight=weight, ignore_index=ignore_index, reduction=reduction)


def log_softmax(input, dim):
    return LogSoftmax.apply(input, dim=dim)


def linear(input, weight, bias):
    """y = X @ A.T + b (nn/functional.py:54-63)."""
    from ..VariableFunctions import matmul
    if bias is not None:
        return matmul(input, weight.T) + bias
    return matmul(input, weight.T)


def layer_norm(input, normalized_shape, weight=None, bias=None, eps=1e-5):
    """(input - mean) / sqrt(var + eps) * weight + bias over the trailing dimensions ``normalized_shape``.  The input is
    float32 or float16, weight and bias are float32."""
    if normalized_shape.__class__ is int:
        normalized_shape = (normalized_shape,)
    return LayerNorm.apply(input, weight, bias, normalized_shape=normalized_shape, eps=eps)


def token_log_prob(input, tokens, top=0, ignore_index=-100):
    """Of logits [..., V] and int64 or int32 tokens [...]: ``(logp, entropy)``, the log probability of each token and the
    entropy of its distribution, in nats and float32; with ``top`` also ``(top_logp, top_index)`` [..., top], the best
    alternatives, best first and the lowest index first among equals (at most 64).

    Negative tokens count from the end.  A position whose token is ``ignore_index`` is not looked at: zeros, and -1 for
    the indexes.  A token outside the vocabulary gives NaN, and so does a NaN or +inf among the logits (indexes -1),
    for the gradient too.
    Logits of -inf alone leave log probabilities of -inf, entropy 0 and no gradient.  ``tt.backward`` takes gradients of
    several of the outputs in one pass."""
    return TokenLogProb.apply(input, tokens=tokens, top=top, ignore_index=ignore_index)


def distill_loss(input, teacher, index, temperature=1.0, reduction='mean'):
    """Kullback-Leibler divergence, times temperature^2, of a student's distribution softmax(input / temperature) over V
    classes from a teacher's over its K best: ``teacher`` [..., K] holds their logits (log probabilities do as well),
    ``index`` [..., K] their classes, int64 or int32, and -1 where there is no entry.

    Entries of one class add up.  Positions without an entry, or with -inf alone, have loss and gradient 0 and are not
    counted by 'mean'; an index of V or more gives NaN, and so does a NaN or +inf among a position's logits, for its
    gradient too.  Logits of -inf alone have no gradient.  Gradients flow to ``input`` only."""
    return DistillLoss.apply(input, teacher=teacher, index=index, temperature=float(temperature), reduction=reduction)
