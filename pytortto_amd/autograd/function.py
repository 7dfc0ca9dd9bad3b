"""Autograd nodes with the reference's operator interface (``src/tortto/autograd/function.py``).

``class X(Function)`` with static ``forward(ctx, *inputs, **params)`` / ``backward(ctx,
*grad_outputs)``, invoked as ``X.apply(*tensors, **kwargs)``.  ``ctx`` is the freshly made
``XBackward`` node: ``params`` (the kwargs, also scratch space), ``needs_input_grad``,
``next_functions``, ``requires_grad``, ``xp``, ``save_for_backward`` / ``saved_tensors``.
``backward`` returns one raw array (not a Tensor) or ``None`` per input.
"""
import sys

import numpy as np

from .. import xparray
from . import grad_mode
from .grad_mode import is_grad_enabled


class FunctionBase:
    # a node starts with these and stores what differs (one is made for every operation)
    variable = to_save = next_functions = needs_input_grad = grad = params = xp = sources = None
    prev_function_counts = 0
    requires_grad = False

    def save_for_backward(self, *tensors):
        """Remember tensors (or None) together with their in-place version (function.py:27-28)."""
        self.to_save = tuple([None if t is None else (t, t.data._version[0]) for t in tensors])

    @property
    def saved_tensors(self):
        """The saved tensors' arrays; raises if one was modified in place since (function.py:30-32)."""
        return tuple(get_data(pair) for pair in self.to_save)

    def hang(self):
        """A tensor is about to hang on this node: where the node was made without gradients (an in-place
        operation under ``no_grad``, gradients switched on again inside a forward), make the links to what its
        inputs hang on.  (The first, which a function may have re-pointed by hand, as it was.)"""
        if self.sources is not None:
            (inputs, first), self.sources = self.sources, None
            at = [first if i == 0 or t is None else (t.grad_fn, t._output_idx) for i, t in enumerate(inputs)]
            self.next_functions = tuple(_link(t, *where) if req else (None, 0)
                                        for t, req, where in zip(inputs, self.needs_input_grad, at))

    def clear(self):
        """Drop what backward no longer needs (function.py:34-40); leaf accumulators and copy
        nodes keep an empty gradient slot so they can take part in a later backward."""
        self.to_save = None
        if self.__class__ is AccumulateGrad or getattr(self, '_forward_cls', None).__name__ == 'ToCopy':
            self.grad = [None]
        else:
            self.grad = None
            self.params = None


class BackwardFunction(FunctionBase):
    def apply(self, *args):
        out = self._forward_cls.backward(self, *args)
        if out.__class__ is not tuple and out.__class__ is not list:
            out = (out,)
        if len(out) != len(self.needs_input_grad):
            raise RuntimeError(f'function {self.__class__.__name__} returned an incorrect number of gradients'
                               f' (expected {len(self.needs_input_grad)}, got {len(out)})')
        return out


class AccumulateGrad(BackwardFunction):
    next_functions = ()
    done = False        # its gradient of this pass is where it belongs

    def apply(self, *args):
        self.accumulate(self.grad[0])
        self.done = False       # (it was visited in its turn)

    def accumulate(self, g):
        """function.py:70-93: first gradient is stored (contiguous), later ones are added."""
        var = self.variable
        if var.grad is None:
            # a leaf keeps its gradient beyond this pass: it must not stay an alias of another holder's
            if g.__class__ is not xparray.hiparray:
                g = np.ascontiguousarray(g)
            elif g._shared:
                g.own()
            var.grad = g
        else:
            var.grad += g
        self.done = True


def _node_class(cls):
    """The class of ``cls``'s graph nodes, made at its first use: one made for every call is garbage that only
    the cycle collector takes back."""
    node_class = cls.__dict__.get('_node_class')
    if node_class is None:
        node_class = cls._node_class = type(cls.__name__ + 'Backward', (BackwardFunction,), {'_forward_cls': cls})
    return node_class


def _link(t, grad_fn, output_idx):
    """What a node hangs on for an input ``t`` that requires a gradient, and had ``grad_fn``."""
    if grad_fn is None:             # leaf: gradients end in an accumulator
        acc = AccumulateGrad()
        acc.variable = t
        acc.prev_function_counts = 1
        acc.grad = [None]
        return acc, 0
    grad_fn.prev_function_counts += 1
    return grad_fn, output_idx


class Function(FunctionBase):
    def __init__(self, *args, **kwargs):
        raise RuntimeError(f'{self.__class__} should not be instantiated. Methods on autograd functions'
                           'are all static, so you should invoke them on the class itself.')

    @staticmethod
    def forward(ctx, *inputs, **params):
        raise NotImplementedError('You must implement the forward function for custom autograd.Function.')

    @staticmethod
    def backward(ctx, *grad_outputs):
        raise NotImplementedError('You must implement the backward method for your custom autograd.Function '
                                  'to use it with backward mode automatic differentiation.')

    @classmethod
    def apply(cls, *inputs, **params):
        """function.py:113-179."""
        node = (cls.__dict__.get('_node_class') or _node_class(cls))()
        node.params = params
        needs, any_grad = [], False
        if grad_mode._enabled:
            links = []
            for t in inputs:
                req = False if t is None else t.requires_grad
                needs.append(req)
                any_grad |= req
                links.append(_link(t, t.grad_fn, t._output_idx) if req else (None, 0))
            node.next_functions = tuple(links)
        else:
            # nothing hangs on this node as a rule, and then it needs no accumulators for the leaves and is not
            # waited for by its inputs' nodes; what it hangs on is noted for the exception (``hang``)
            needs = [False if t is None else t.requires_grad for t in inputs]
            any_grad = True in needs
            node.next_functions = ((None, 0),) * len(needs)
            if any_grad:
                first = inputs[0]
                node.sources = inputs, first if first is None else (first.grad_fn, first._output_idx)
        node.needs_input_grad = tuple(needs)
        node.requires_grad = any_grad
        # the array namespace of the inputs (function.py:146)
        node.xp = xparray if inputs[0].data.__class__ is xparray.hiparray else np
        results = cls.forward(node, *inputs, **params)
        node.grad = [None] * (len(results) if isinstance(results, (tuple, list)) else 1)
        if node.sources is not None and sys.getrefcount(node) > 2:
            node.hang()                 # somebody keeps it: a tensor attached by hand
        return results


# ---- what the functions' forward / backward bodies and the engine share ----------------------------


def inplace_precheck(t):
    """helper.py:5-7"""
    if is_grad_enabled() and t.requires_grad and t.grad_fn is None:
        raise RuntimeError('a leaf Variable that requires grad is being used in an in-place operation.')


def inplace_update(t, grad_fn):
    """helper.py:10-16: bump the shared version counter and re-point the tensor at ``grad_fn``."""
    t.data._version[0] += 1
    t._output_idx = 0
    t.requires_grad = grad_fn.requires_grad
    if grad_fn.requires_grad:
        grad_fn.hang()
        t.grad_fn = grad_fn
    return t


def get_data(pair):
    """helper.py:19-29: hand back the saved tensor's array unless it was modified in place."""
    if pair is None:
        return None
    t, version = pair
    if t._version != version:
        origin = '' if t.grad_fn is None else f', which is the output of {t.grad_fn.__class__.__name__},'
        raise RuntimeError(f'one of the variables needed for gradient computation has been modified '
                           f'by an inplace operation: [shape: {t.shape}]{origin} is at version '
                           f'{t._version}; expected version {version} instead.')
    return t.data


def take_arrived(ctx, i, like):
    """The gradient that other consumers have already sent to where input ``i``'s goes, taken out of its
    slot for a backward kernel that adds it to what it writes (the engine would add it afterwards, in a
    pass of its own: tensor.py:568-613); None if there is none, or none laid out as ``like``."""
    fn, idx = ctx.next_functions[i]
    arrived = None if fn is None or fn.grad is None else fn.grad[idx]
    if arrived.__class__ is not xparray.hiparray or arrived.shape != like.shape or arrived.dtype != like.dtype:
        return None
    fn.grad[idx] = None
    return arrived


_Tensor = None


def build_links(data, grad_fn, copy=False, _output_idx=0):
    """helper.py:45-50: wrap a forward result, attached to ``grad_fn`` when gradients flow."""
    global _Tensor
    if _Tensor is None:                 # tensor.py imports this module's users
        from ..tensor import Tensor as _Tensor
    if data.__class__ is xparray.hiparray:
        if grad_fn.requires_grad and grad_mode._enabled:
            if grad_fn.sources is not None:
                grad_fn.hang()
            return _Tensor.on(data, True, grad_fn, _output_idx)
        return _Tensor.on(data)
    dtype = getattr(data, 'dtype', None)
    if grad_fn.requires_grad and grad_mode._enabled:
        grad_fn.hang()
        return _Tensor(data, requires_grad=True, dtype=dtype, copy=copy, grad_fn=grad_fn, _output_idx=_output_idx)
    return _Tensor(data, dtype=dtype, copy=copy)


def _edges_from(nodes):
    """How many edges lead to each node that ``nodes`` lead to: {node: edges}."""
    edges, todo, seen = {}, list(nodes), set(nodes)
    while todo:
        for fn, _ in todo.pop().next_functions or ():
            if fn is not None:
                edges[fn] = edges.get(fn, 0) + 1
                if fn not in seen:
                    seen.add(fn)
                    todo.append(fn)
    return edges


def toposort(*end_nodes):
    """helper.py:53-82: yield nodes so that a node comes after everything that feeds gradient
    into it; nodes whose other consumers are not part of this backward pass are taken from
    those ``waiting`` once nothing else is ready.  Of several end nodes, one that others lead to waits for them.
    Where several nodes wait then, one of them may lead to another, so from there on the edges that are left in this pass
    are counted, and not those of all consumers."""
    ready, waiting, left = [], {}, None         # (``waiting``: in the order of their arrival)
    for node in end_nodes:
        if node.prev_function_counts:
            waiting[node] = None
        else:
            ready.append(node)
    while ready or waiting:
        if ready:
            node = ready.pop()
        elif len(waiting) == 1:
            node, _ = waiting.popitem()
        else:
            left = _edges_from(waiting)
            ready = [node for node in waiting if node not in left]
            waiting = {}
            continue
        yield node
        for fn, _ in node.next_functions or ():
            if fn is None:
                continue
            fn.prev_function_counts -= 1
            if fn.__class__ is AccumulateGrad and fn.done:
                fn.done = False
            elif left is not None:
                left[fn] -= 1
                if left[fn] == 0:
                    ready.append(fn)
            elif fn.prev_function_counts == 0:
                ready.append(fn)
                waiting.pop(fn, None)
            else:
                waiting[fn] = None
