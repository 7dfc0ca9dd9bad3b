"""The work that the language-model operators are timed on: layer normalisation, log probabilities of
given tokens (with entropy and the best alternatives) and distillation from a teacher's top logits.

Every case is one call as a user makes it: a forward pass without gradients (scoring, serving) or a
training step, forward and backward.  ``run`` computes it in plain torch operations, or, where ``own``
is set, through the framework's public functions on tensors that share torch's memory.

``listed()`` are fixed cases, ``draw(rng)`` makes others of the same ranges.
"""
import math

import torch

own = False

DEVICE = 'cuda'
EPS = 1e-5
IGNORED = -100      # the token of a position that is not scored (padding, a prompt)


# ---- the cases -------------------------------------------------------------------------------------

def _norm(rows, cols, half, train, **more):
    return dict(more, op='norm', rows=rows, cols=cols, half=half, train=train)


def _logp(rows, vocab, half, train, top, masked, **more):
    return dict(more, op='logp', rows=rows, vocab=vocab, half=half, train=train, top=top, masked=masked)


def _distill(rows, vocab, half, train, top, temperature, reduction, **more):
    return dict(more, op='distill', rows=rows, vocab=vocab, half=half, train=train, top=top, temperature=temperature,
                reduction=reduction)


def listed():
    return [
        # one token of a model that is being served: latency
        _norm(1, 1024, False, False, name='norm_one_token_f32'),
        # a prompt's tokens in half precision, forward only
        _norm(4096, 4096, True, False, name='norm_prompt_f16'),
        # a training step's block input: forward, dx, and the two sums over all tokens
        _norm(8192, 2048, False, True, name='norm_train_f32'),
        # channels of a 56x56 image batch, channel last: many short rows
        _norm(100352, 96, False, True, name='norm_train_channels_f32'),
        # odd token count and odd width, half precision
        _norm(3001, 1537, True, True, name='norm_train_ragged_f16'),
        # one generated token with its five best alternatives
        _logp(1, 32768, False, False, 5, False, name='logp_one_token_f32'),
        # a decoding batch over a large vocabulary, some tokens banned, twenty alternatives
        _logp(48, 131072, True, False, 20, True, name='logp_decode_f16'),
        # scoring a set of texts: no alternatives
        _logp(4096, 32768, False, False, 0, False, name='logp_score_f32'),
        # policy gradient with an entropy bonus, odd vocabulary
        _logp(2047, 50021, False, True, 0, False, name='logp_train_ragged_f32'),
        # a classifier's classes at the benchmark's batch, ten of a thousand from the teacher
        _distill(64, 1000, False, True, 10, 4.0, 'mean', name='distill_classes_f32'),
        # a language model's training step
        _distill(4096, 32768, False, True, 32, 1.0, 'mean', name='distill_train_f32'),
        # the same over a large vocabulary, half precision logits, softened
        _distill(1024, 131072, True, True, 64, 2.0, 'sum', name='distill_train_f16'),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, half, train = rng.choice(('norm', 'logp', 'distill')), rng.random() < 0.4, rng.random() < 0.55
    if op == 'norm':
        cols = _spread(rng, 24, 16384)
        return _norm(_spread(rng, 1, max(1, min(1 << 17, (1 << 25) // cols))), cols, half, train)
    vocab = _spread(rng, 10, 160000)
    rows = _spread(rng, 1, min(1 << 16, (1 << 26) // vocab))
    if op == 'logp':
        return _logp(rows, vocab, half, train, rng.choice((0, 0, 1, 5, 10, 20)) if vocab >= 20 else 1, rng.random() < 0.3)
    return _distill(rows, vocab, half, train, _spread(rng, 4, max(4, min(64, vocab // 2))), rng.choice((1.0, 1.0, 2.0, 4.0)),
                    rng.choice(('mean', 'mean', 'sum', 'none')))


# ---- inputs ----------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(DEVICE)
    gen.manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(shape, generator=gen, device=DEVICE) * std + mean

    kind = torch.float16 if case['half'] else torch.float32
    state, rows = {'case': case}, case['rows']
    if case['op'] == 'norm':
        cols = case['cols']
        # a residual stream: off centre, columns of unequal size
        state['x'] = (normal(rows, cols) * (1.0 + normal(cols).abs()) + 0.5 * normal(cols)).to(kind)
        state['weight'], state['bias'] = normal(cols, std=0.2, mean=1.0), normal(cols, std=0.2)
        if case['train']:
            state['dy'] = normal(rows, cols, std=0.1).to(kind)
        return state
    vocab = case['vocab']
    z = normal(rows, vocab, std=2.0)
    if case['op'] == 'logp':
        # what a model answers: a few tokens stand out; the given ones are among them as a rule
        tokens = torch.randint(vocab, (rows,), generator=gen, device=DEVICE)
        z.scatter_add_(1, torch.randint(vocab, (rows, 4), generator=gen, device=DEVICE), normal(rows, 4, std=2.0, mean=7.0))
        z.scatter_add_(1, tokens[:, None], normal(rows, 1, std=3.0, mean=6.0))
        if case['masked']:      # tokens that must not come, a given one among them now and then
            z.masked_fill_(torch.rand((rows, vocab), generator=gen, device=DEVICE) < 0.02, -math.inf)
        if rows > 16:           # positions that are not scored
            tokens[torch.rand(rows, generator=gen, device=DEVICE) < 0.05] = IGNORED
        state['x'], state['tokens'] = z.to(kind), tokens
        if case['train']:       # advantages, and the weight of the entropy bonus
            state['g_logp'], state['g_entropy'] = normal(rows) / rows, torch.full((rows,), -0.01 / rows, device=DEVICE)
            if case['top']:
                state['g_top'] = normal(rows, case['top'], std=0.1) / rows
        return state
    # the teacher's best tokens, distinct, best first; the student has learned some of it
    k = case['top']
    start = torch.randint(vocab, (rows, 1), generator=gen, device=DEVICE)
    index = (start + torch.arange(k, device=DEVICE) * (vocab // k)) % vocab
    teacher = normal(rows, k, std=2.0, mean=8.0).sort(-1, descending=True).values
    z.scatter_add_(1, index, 0.8 * teacher + normal(rows, k))
    if rows > 16:               # a prompt's positions have no teacher, some others fewer entries
        count = torch.randint(1, k + 1, (rows, 1), generator=gen, device=DEVICE)
        luck = torch.rand((rows, 1), generator=gen, device=DEVICE)
        count = torch.where(luck < 0.05, 0, torch.where(luck < 0.2, count, k))
        index = torch.where(torch.arange(k, device=DEVICE) < count, index, -1)
    state['x'], state['teacher'], state['index'] = z.to(kind), teacher.to(kind), index
    if case['train'] and case['reduction'] == 'none':
        state['g_loss'] = torch.rand((rows,), generator=gen, device=DEVICE) / rows
    return state


# ---- the plain forms -------------------------------------------------------------------------------

def _plain_norm(s):
    x, w = s['x'].float(), s['weight']
    centred = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    n = centred * r
    y = (n * w + s['bias']).to(s['x'].dtype)
    if not s['case']['train']:
        return [y]
    dy = s['dy'].float()
    h = dy * w
    dx = r * (h - h.mean(-1, keepdim=True) - n * (h * n).mean(-1, keepdim=True))
    return [y, dx.to(s['x'].dtype), (dy * n).sum(0), dy.sum(0)]


def _softmax(x):
    """(log of the sum of exponentials, probabilities); a row of -inf alone: (-inf, zeros)"""
    best = x.amax(-1, keepdim=True)
    best = torch.where(best == -math.inf, 0.0, best)
    e = torch.exp(x - best)
    total = e.sum(-1, keepdim=True)
    return torch.log(total) + best, torch.where(total > 0, e / total, 0.0)


def _best(x, k):
    """Indexes of the k largest of each row, the lowest index first among equals: the values' order and the
    index in one whole number."""
    bits = (x + 0.0).view(torch.int32).long()
    key = ((bits ^ ((bits >> 31) & 0x7fffffff)) << 32) + ((1 << 32) - 1 - torch.arange(x.shape[-1], device=x.device))
    return (1 << 32) - 1 - (torch.topk(key, k, -1).values & 0xffffffff)


def _plain_logp(s):
    case, x = s['case'], s['x'].float()
    kept = (s['tokens'] != IGNORED)[:, None]
    tokens = torch.where(kept, s['tokens'][:, None], 0)
    lse, p = _softmax(x)
    logq = torch.where(p > 0, x - lse, 0.0)
    entropy = -(p * logq).sum(-1, keepdim=True)
    logp = x.gather(1, tokens) - lse
    out = [torch.where(kept, logp, 0.0)[:, 0], torch.where(kept, entropy, 0.0)[:, 0]]
    if case['top']:
        best = _best(x, case['top'])
        out += [torch.where(kept, x.gather(1, best) - lse, 0.0), torch.where(kept, best, -1)]
    if case['train']:
        a = s['g_logp'][:, None]
        total = a + s['g_top'].sum(-1, keepdim=True) if case['top'] else a
        dx = -p * (total + s['g_entropy'][:, None] * (logq + entropy))
        dx.scatter_add_(1, tokens, a)
        if case['top']:
            dx.scatter_add_(1, best, s['g_top'])
        out.append(torch.where(kept, dx, 0.0).to(s['x'].dtype))
    return out


def _plain_distill(s):
    case, t = s['case'], s['case']['temperature']
    x, index = s['x'].float() * (1.0 / t), s['index']
    given = index >= 0
    at = torch.where(given, index, 0)
    teacher = torch.where(given, s['teacher'].float() * (1.0 / t), -math.inf)
    log_total, q = _softmax(teacher)
    counted = q.sum(-1) > 0
    lse, p = _softmax(x)
    loss = t * t * torch.where(q > 0, q * (teacher - log_total - (x.gather(1, at) - lse)), 0.0).sum(-1)
    scale = 1.0 / counted.sum() if case['reduction'] == 'mean' else torch.ones((), device=x.device)
    out = [loss if case['reduction'] == 'none' else loss.sum() * scale]
    if case['train']:
        g = s['g_loss'] if case['reduction'] == 'none' else scale
        g = (t * torch.where(counted, g, 0.0))[:, None]
        dx = p * g
        dx.scatter_add_(1, at, -q * g)
        out.append(dx.to(s['x'].dtype))
    return out


# ---- the framework's operators ---------------------------------------------------------------------

def _theirs(tensor):
    """A result of the framework as a torch tensor on the same memory."""
    return torch.as_tensor(getattr(tensor, 'data', tensor), device=DEVICE)


def _own_norm(tt, s):
    case = s['case']
    x, w, b = tt.as_tensor(s['x']), tt.as_tensor(s['weight']), tt.as_tensor(s['bias'])
    if not case['train']:
        return [_theirs(tt.nn.functional.layer_norm(x, (case['cols'],), w, b, EPS))]
    x.requires_grad = w.requires_grad = b.requires_grad = True
    y = tt.nn.functional.layer_norm(x, (case['cols'],), w, b, EPS)
    y.backward(tt.as_tensor(s['dy']))
    return [_theirs(y), _theirs(x.grad), _theirs(w.grad), _theirs(b.grad)]


def _own_logp(tt, s):
    case = s['case']
    x, tokens = tt.as_tensor(s['x']), tt.as_tensor(s['tokens'])
    x.requires_grad = case['train']
    got = tt.nn.functional.token_log_prob(x, tokens, top=case['top'], ignore_index=IGNORED)
    out = [_theirs(v) for v in got]
    if case['train']:
        gradients = (s['g_logp'], s['g_entropy']) + ((s['g_top'],) if case['top'] else ())
        tt.backward(got[:len(gradients)], [tt.as_tensor(g) for g in gradients])
        out.append(_theirs(x.grad))
    return out


def _own_distill(tt, s):
    case = s['case']
    x = tt.as_tensor(s['x'])
    x.requires_grad = case['train']
    loss = tt.nn.functional.distill_loss(x, tt.as_tensor(s['teacher']), tt.as_tensor(s['index']),
                                         temperature=case['temperature'], reduction=case['reduction'])
    if not case['train']:
        return [_theirs(loss)]
    loss.backward(tt.as_tensor(s['g_loss']) if 'g_loss' in s else None)
    return [_theirs(loss), _theirs(x.grad)]


def run(state):
    op = state['case']['op']
    if own:
        import pytortto_amd as tt
        return {'norm': _own_norm, 'logp': _own_logp, 'distill': _own_distill}[op](tt, state)
    return {'norm': _plain_norm, 'logp': _plain_logp, 'distill': _plain_distill}[op](state)


# ---- what a pass cannot do without -----------------------------------------------------------------

def work(case):
    """Inputs read once, outputs written once; an exponential counted as one operation."""
    size, rows = 2.0 if case['half'] else 4.0, case['rows']
    if case['op'] == 'norm':
        n = rows * case['cols']
        if case['train']:
            return {'bytes': 4 * n * size + 16.0 * case['cols'], 'flops': 24.0 * n}
        return {'bytes': 2 * n * size + 8.0 * case['cols'], 'flops': 8.0 * n}
    n, k = rows * case['vocab'], case['top']
    if case['op'] == 'logp':
        if case['train']:
            return {'bytes': 2 * n * size + rows * (24.0 + 16.0 * k), 'flops': 12.0 * n}
        return {'bytes': n * size + rows * (16.0 + 12.0 * k), 'flops': 6.0 * n}
    small = rows * (k * (8.0 + size) + 4.0)
    return {'bytes': (2 if case['train'] else 1) * n * size + small, 'flops': (7.0 if case['train'] else 4.0) * n}


# ---- the same in 64 bits ---------------------------------------------------------------------------

def _exact_norm(s):
    x, w, b = (s[name].double().requires_grad_() for name in ('x', 'weight', 'bias'))
    y = w * (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + EPS) + b
    if not s['case']['train']:
        return [y.detach()]
    return [y.detach(), *torch.autograd.grad(y, (x, w, b), s['dy'].double())]


def _exact_logp(s):
    case = s['case']
    x, kept, possible = s['x'].double().requires_grad_(), s['tokens'] != IGNORED, s['x'] > -math.inf
    logq = x - torch.logsumexp(x, -1, keepdim=True)
    finite = torch.where(possible, logq, 0.0)
    logp = logq.gather(1, s['tokens'].clamp(min=0)[:, None])[:, 0]
    entropy = -(torch.where(possible, logq.exp(), 0.0) * finite).sum(-1)
    out = [torch.where(kept, logp, 0.0), torch.where(kept, entropy, 0.0)]
    weights = [s['g_logp'], s['g_entropy']] if case['train'] else []
    parts = [logp, entropy]
    if case['top']:
        # among equal logits any choice has the same values; the gradient goes to the lowest index
        first = torch.sort(s['x'].double(), dim=-1, descending=True, stable=True).indices[:, :case['top']]
        parts.append(logq.gather(1, first))
        weights += [s['g_top']] if case['train'] else []
        out += [torch.where(kept[:, None], parts[2], 0.0), None]
    if case['train']:
        given = [g.double() * (kept if g.ndim == 1 else kept[:, None]) for g in weights]
        out.append(torch.autograd.grad(parts, x, given)[0])
    return [None if v is None else v.detach() for v in out]


def _exact_distill(s):
    case, t = s['case'], s['case']['temperature']
    x, index = s['x'].double().requires_grad_(), s['index']
    teacher = torch.where(index >= 0, s['teacher'].double() / t, -1e30)
    counted = (index >= 0).any(-1)
    q = torch.softmax(teacher, -1) * counted[:, None]
    logp = torch.log_softmax(x / t, -1).gather(1, index.clamp(min=0))
    loss = t * t * (torch.special.xlogy(q, q) - q * logp).sum(-1)
    if case['reduction'] != 'none':
        loss = loss.sum() / (counted.sum() if case['reduction'] == 'mean' else 1.0)
    if not case['train']:
        return [loss.detach()]
    return [loss.detach(), torch.autograd.grad(loss, x, s['g_loss'].double() if 'g_loss' in s else None)[0]]


def exact(case, seed):
    return {'norm': _exact_norm, 'logp': _exact_logp, 'distill': _exact_distill}[case['op']](prepare(case, seed))
