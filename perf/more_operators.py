"""The work that a large vocabulary's loss and the orthogonalised updates are timed on: softmax cross entropy straight
from features and a head's weight (with both gradients), Newton-Schulz orthogonalisation of a matrix, and the
optimiser's step that uses it.

Every case is one call as a user makes it: a loss without gradients (scoring), a training step's loss with its backward
pass, one matrix, or one step of an optimiser that is kept with its momentum.  ``run`` computes it in plain torch
operations, or, where ``own`` is set, through the framework's public functions on tensors that share torch's memory.

``listed()`` are fixed cases, ``draw(rng)`` makes others of the same ranges.
"""
import math

import torch

own = False

DEVICE = 'cuda'
IGNORED = -100      # the target of a position without one (padding, a prompt)
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
RATE, DECAY, MOMENTUM = 0.02, 0.1, 0.95


# ---- the cases -------------------------------------------------------------------------------------

def _loss(rows, width, vocab, half, train, reduction, padded, **more):
    return dict(more, op='loss', rows=rows, width=width, vocab=vocab, half=half, train=train, reduction=reduction,
                padded=padded)


def _orthogonal(rows, cols, half, steps, **more):
    return dict(more, op='orthogonal', rows=rows, cols=cols, half=half, steps=steps)


def _muon(shapes, nesterov, **more):
    """``shapes``: matrices as "RxC", several of one kind as "NxRxC"."""
    return dict(more, op='muon', shapes=shapes, nesterov=nesterov)


def listed():
    return [
        # how likely one given token is: latency, and the weight read once
        _loss(1, 2048, 32768, True, False, 'mean', False, name='loss_one_token_f16'),
        # the benchmark's image classifier: 64 images, a thousand classes behind 2048 features
        _loss(64, 2048, 1000, False, True, 'mean', False, name='loss_classes_f32'),
        # scoring texts, a loss for each position
        _loss(777, 1024, 50021, False, False, 'none', True, name='loss_score_f32'),
        # a language model's training step
        _loss(4096, 1024, 32768, False, True, 'mean', True, name='loss_train_f32'),
        # the same with half precision, odd sizes and a weight for each position
        _loss(2047, 1000, 50021, True, True, 'none', True, name='loss_train_ragged_f16'),
        # a large vocabulary
        _loss(4096, 2048, 131072, True, True, 'mean', True, name='loss_train_large_f16'),
        # one small matrix: latency
        _orthogonal(64, 64, False, 5, name='orthogonal_small_f32'),
        # a square projection
        _orthogonal(2048, 2048, False, 5, name='orthogonal_square_f32'),
        # a tall matrix of odd sizes
        _orthogonal(5001, 777, True, 5, name='orthogonal_tall_f16'),
        # the convolutions of a ResNet-50's last two stages, the benchmark's network
        _muon('256x512 256x2304 1024x256 1024x512 5x256x1024 5x256x2304 5x1024x256 '
              '512x1024 512x4608 2048x512 2048x1024 2x512x2048 2x512x4608 2x2048x512', True, name='muon_convolutions_f32'),
        # the matrices of one transformer block
        _muon('4x2048x2048 8192x2048 2048x8192', True, name='muon_block_f32'),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    op = rng.choice(('loss', 'loss', 'orthogonal', 'muon'))
    if op == 'loss':
        width, vocab = _spread(rng, 16, 4096), _spread(rng, 10, 131072)
        rows = _spread(rng, 1, max(1, min(8192, (1 << 29) // vocab, (1 << 39) // (width * vocab))))
        return _loss(rows, width, vocab, rng.random() < 0.5, rng.random() < 0.7, rng.choice(('mean', 'mean', 'sum', 'none')),
                     rng.random() < 0.5)
    if op == 'orthogonal':
        return _orthogonal(_spread(rng, 1, 4096), _spread(rng, 1, 4096), rng.random() < 0.4, rng.choice((3, 5, 5, 6)))
    shapes = ['%dx%d' % (_spread(rng, 8, 2048), _spread(rng, 8, 2048)) for _ in range(_spread(rng, 1, 24))]
    return _muon(' '.join(shapes), rng.random() < 0.7)


def _matrices(case):
    out = []
    for group in case['shapes'].split():
        numbers = [int(n) for n in group.split('x')]
        out += [tuple(numbers[-2:])] * (numbers[0] if len(numbers) == 3 else 1)
    return out


# ---- inputs ----------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(DEVICE)
    gen.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device=DEVICE) * std

    state = {'case': case}
    if case['op'] == 'loss':
        rows, width, vocab = case['rows'], case['width'], case['vocab']
        kind = torch.float16 if case['half'] else torch.float32
        # normalised features that lean towards their target's row, as a model's that has learned something
        weight = normal(vocab, width, std=width ** -0.5) * (0.5 + torch.rand((vocab, 1), generator=gen, device=DEVICE))
        target = torch.randint(vocab, (rows,), generator=gen, device=DEVICE)
        x = normal(rows, width) * (1.0 + 0.5 * normal(width).abs())
        x += weight[target] * (5.0 * torch.rand((rows, 1), generator=gen, device=DEVICE))
        if case['padded']:
            target[torch.rand(rows, generator=gen, device=DEVICE) < 0.1] = IGNORED
            target[:1] = 0
        state['x'], state['weight'], state['target'] = x.to(kind), weight.to(kind), target
        if case['train']:
            if case['reduction'] == 'none':     # a weight for each position
                state['g_loss'] = torch.rand((rows,), generator=gen, device=DEVICE)
            elif case['half']:                  # small gradients of halves are trained with a scaled loss
                state['g_loss'] = torch.full((), 1024.0, device=DEVICE)
        return state
    if case['op'] == 'orthogonal':
        x = _gradient(normal, case['rows'], case['cols'])
        state['x'] = x.to(torch.float16 if case['half'] else torch.float32)
        return state
    state['parameters'] = [normal(r, c, std=c ** -0.5) for r, c in _matrices(case)]
    state['gradients'] = [_gradient(normal, r, c) for r, c in _matrices(case)]
    state['momenta'] = [_gradient(normal, r, c) for r, c in _matrices(case)]
    if own:
        import pytortto_amd as tt
        # the program's model and optimiser, in the middle of a training run
        leaves = [tt.as_tensor(p, requires_grad=True) for p in state['parameters']]
        state['optimizer'] = tt.optim.Muon(leaves, lr=RATE, weight_decay=DECAY, momentum=MOMENTUM,
                                           nesterov=case['nesterov'], ns_coefficients=COEFFICIENTS, eps=EPS, ns_steps=5)
        for leaf, g, m in zip(leaves, state['gradients'], state['momenta']):
            leaf.grad = tt.as_tensor(g).data
            state['optimizer'].state[leaf]['momentum_buffer'] = tt.as_tensor(m).data
        state['leaves'] = leaves
    return state


def _gradient(normal, rows, cols):
    """A weight's gradient: noise, and a few directions that stand out."""
    few = min(4, rows, cols)
    return normal(rows, cols, std=1e-2) + normal(rows, few) @ normal(few, cols, std=2e-2)


# ---- the plain forms -------------------------------------------------------------------------------

def _plain_loss(s):
    case, x, w = s['case'], s['x'].float(), s['weight'].float()
    kept = s['target'] != IGNORED
    target = torch.where(kept, s['target'], 0)[:, None]
    z = x @ w.T
    best = z.amax(-1, keepdim=True)
    e = torch.exp(z - best)
    total = e.sum(-1, keepdim=True)
    loss = torch.where(kept, (torch.log(total) + best - z.gather(1, target))[:, 0], 0.0)
    scale = 1.0 / kept.sum() if case['reduction'] == 'mean' else torch.ones((), device=x.device)
    out = [loss if case['reduction'] == 'none' else loss.sum() * scale]
    if case['train']:
        g = s.get('g_loss', 1.0) * scale * kept
        dz = e / total
        dz.scatter_add_(1, target, torch.full_like(best, -1.0))
        dz *= g[:, None]
        out += [(dz @ w).to(s['x'].dtype), (dz.T @ x).to(s['weight'].dtype)]
    return out


def _newton_schulz(x, steps):
    a, b, c = COEFFICIENTS
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / torch.clamp(torch.sqrt((x * x).sum()), min=EPS)
    for _ in range(steps):
        gram = x @ x.T
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.T if tall else x


def _plain_orthogonal(s):
    return [_newton_schulz(s['x'].float(), s['case']['steps']).to(s['x'].dtype).contiguous()]


def _plain_muon(s):
    for p, g, m in zip(s['parameters'], s['gradients'], s['momenta']):
        m.mul_(MOMENTUM).add_(g * (1.0 - MOMENTUM))
        u = g * (1.0 - MOMENTUM) + m * MOMENTUM if s['case']['nesterov'] else m
        u = _newton_schulz(u, 5)
        p.mul_(1.0 - RATE * DECAY).sub_(u * (RATE * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))))
    return [s['parameters'], s['momenta']]


# ---- the framework's operators ---------------------------------------------------------------------

def _theirs(tensor):
    """A result of the framework as a torch tensor on the same memory."""
    return torch.as_tensor(getattr(tensor, 'data', tensor), device=DEVICE)


def _own_loss(tt, s):
    case = s['case']
    x, w = tt.as_tensor(s['x'], case['train']), tt.as_tensor(s['weight'], case['train'])
    loss = tt.nn.functional.linear_cross_entropy(x, w, tt.as_tensor(s['target']), ignore_index=IGNORED,
                                                 reduction=case['reduction'])
    if not case['train']:
        return [_theirs(loss)]
    loss.backward(tt.as_tensor(s['g_loss']) if 'g_loss' in s else None)
    return [_theirs(loss), _theirs(x.grad), _theirs(w.grad)]


def _own_orthogonal(tt, s):
    return [_theirs(tt.optim.orthogonalize(tt.as_tensor(s['x']), steps=s['case']['steps'], coefficients=COEFFICIENTS,
                                           eps=EPS))]


def _own_muon(tt, s):
    s['optimizer'].step()
    return [s['parameters'], s['momenta']]


def run(state):
    op = state['case']['op']
    if own:
        import pytortto_amd as tt
        return {'loss': _own_loss, 'orthogonal': _own_orthogonal, 'muon': _own_muon}[op](tt, state)
    return {'loss': _plain_loss, 'orthogonal': _plain_orthogonal, 'muon': _plain_muon}[op](state)


# ---- what a pass cannot do without -----------------------------------------------------------------

def _schulz_flops(rows, cols, steps):
    """Three products a step; the two symmetric ones are half as many."""
    m, n = min(rows, cols), max(rows, cols)
    return steps * (m * m * n + m * m * m + 2.0 * m * m * n)


def work(case):
    """Inputs read once, outputs written once."""
    if case['op'] == 'loss':
        size, rows, width, vocab = 2.0 if case['half'] else 4.0, case['rows'], case['width'], case['vocab']
        passes = 2 if case['train'] else 1
        return {'bytes': passes * size * (rows * width + vocab * width) + 12.0 * rows,
                'flops': (3 if case['train'] else 1) * 2.0 * rows * width * vocab}
    if case['op'] == 'orthogonal':
        n = case['rows'] * case['cols']
        return {'bytes': 2 * n * (2.0 if case['half'] else 4.0),
                'flops': _schulz_flops(case['rows'], case['cols'], case['steps'])}
    # the parameter and its momentum read and written, the gradient read
    return {'bytes': sum(20.0 * r * c for r, c in _matrices(case)),
            'flops': sum(_schulz_flops(r, c, 5) for r, c in _matrices(case))}


# ---- the same in 64 bits ---------------------------------------------------------------------------

def _exact_loss(s):
    case = s['case']
    if 6.0 * case['rows'] * case['width'] * case['vocab'] > 9e14:
        return None
    x, w, target = s['x'].double(), s['weight'].double(), s['target']
    kept = target != IGNORED
    logp = torch.log_softmax(x @ w.T, -1)
    one = torch.zeros_like(logp)
    one[kept, target[kept]] = 1.0
    loss = -(logp * one).sum(-1)
    weight = kept.double()
    if case['reduction'] != 'none':
        weight = weight / kept.sum() if case['reduction'] == 'mean' else weight
        loss = (loss * weight).sum()
    if not case['train']:
        return [loss]
    if 'g_loss' in s:
        weight = weight * s['g_loss'].double()
    dz = logp.exp_().sub_(one).mul_(weight[:, None])
    return [loss, dz @ w, dz.T @ x]


def _exact_schulz(x, steps):
    """Each step takes a singular value s to a s + b s^3 + c s^5."""
    a, b, c = COEFFICIENTS
    x = x / max(float(torch.linalg.vector_norm(x)), EPS)
    tall = x.shape[0] >= x.shape[1]
    for _ in range(steps):
        if tall:        # from the right
            gram = x.T.contiguous() @ x
            x = x @ (a * torch.eye(x.shape[1], device=x.device, dtype=x.dtype) + (b * gram + c * gram.mm(gram)))
        else:
            gram = x @ x.T.contiguous()
            x = (a * torch.eye(x.shape[0], device=x.device, dtype=x.dtype) + (b * gram + c * gram.mm(gram))) @ x
    return x


def _exact_muon(s):
    parameters, momenta = [], []
    for p, g, m in zip(s['parameters'], s['gradients'], s['momenta']):
        p, g, m = p.double(), g.double(), m.double()
        m = m + (1.0 - MOMENTUM) * (g - m)
        u = g + MOMENTUM * (m - g) if s['case']['nesterov'] else m
        parameters.append(p - RATE * DECAY * p
                          - RATE * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * _exact_schulz(u, 5))
        momenta.append(m)
    return [parameters, momenta]


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'orthogonal':
        return [_exact_schulz(s['x'].double(), case['steps'])]
    return (_exact_loss if case['op'] == 'loss' else _exact_muon)(s)
