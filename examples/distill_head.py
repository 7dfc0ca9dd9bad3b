"""A student's vocabulary head learns from the best alternatives of a teacher's, and answers single positions.

    python examples/distill_head.py

Both are layer normalisation and a linear layer over features of a synthetic model; the teacher's is fixed.  Every step
takes the teacher's best tokens from ``token_log_prob`` and trains the student on them with ``DistillLoss``.  In the end
the student answers one position, with its best tokens, as a server would.
"""
import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir))
import pytortto_amd as tt  # noqa: E402
from pytortto_amd import nn  # noqa: E402


class Head(nn.Module):
    def __init__(self, width, vocab):
        super().__init__()
        self.norm = nn.LayerNorm(width)
        self.out = nn.Linear(width, vocab, bias=False)

    def forward(self, x):
        return self.out(self.norm(x))


def train(steps=40, positions=384, width=96, vocab=5003, alternatives=16, temperature=2.0, lr=0.02, seed=0, show=print):
    """The losses of every step and, before and after, the student's mean log probability of the teacher's best token."""
    tt.manual_seed(seed)
    rng = np.random.default_rng(seed)
    teacher, student = Head(width, vocab), Head(width, vocab)
    teacher.out.weight.data *= 6.0          # a teacher that prefers some tokens clearly
    teacher, student = teacher.cuda(), student.cuda()
    optimizer = tt.optim.Adam(student.parameters(), lr=lr)
    criterion = nn.DistillLoss(temperature)
    score = nn.functional.token_log_prob
    x = tt.tensor(rng.standard_normal((positions, width)).astype(np.float32) * 2 + 0.5).cuda()
    given = tt.tensor(rng.integers(0, vocab, positions)).cuda()

    def agreement():
        with tt.no_grad():
            _, _, _, best = score(teacher(x), given, top=1)
            logp, _ = score(student(x), tt.tensor(best.data.get()[:, 0]).cuda())
        return float(logp.data.get().mean())

    before, losses = agreement(), []
    for step in range(steps):
        with tt.no_grad():
            _, _, top_logp, top_index = score(teacher(x), given, top=alternatives)
        loss = criterion(student(x), top_logp, top_index)
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
        if show and step % 10 == 0:
            show(f'step {step:3d}: loss {losses[-1]:.4f}')
    after = agreement()
    with tt.no_grad():          # one position, as a server asks for it
        one = x.data.get()[:1]
        logp, entropy, top_logp, top_index = score(student(tt.tensor(one).cuda()), tt.tensor(np.zeros(1, np.int64)).cuda(), top=5)
    if show:
        show(f'mean log probability of the teacher\'s best token: {before:.3f} before, {after:.3f} after')
        show(f'entropy of one position {entropy.data.get()[0]:.3f}, best tokens '
             + ', '.join(f'{i} ({p:.3f})' for i, p in zip(top_index.data.get()[0], np.exp(top_logp.data.get()[0]))))
    return losses, before, after


if __name__ == '__main__':
    parser = argparse.ArgumentParser(description=__doc__.split('\n')[0])
    parser.add_argument('--steps', type=int, default=40)
    parser.add_argument('--vocab', type=int, default=5003)
    parser.add_argument('--alternatives', type=int, default=16)
    arguments = parser.parse_args()
    train(arguments.steps, vocab=arguments.vocab, alternatives=arguments.alternatives)
