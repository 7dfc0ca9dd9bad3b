"""GPU: the example that runs layer normalisation, token log probabilities and distillation together."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
EXAMPLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), os.pardir, 'examples', 'distill_head.py')


def test_the_student_learns_from_the_teachers_alternatives():
    spec = importlib.util.spec_from_file_location('distill_head', EXAMPLE)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, before, after = example.train(steps=30, positions=128, vocab=1003, show=None)
    assert losses[-1] < 0.5 * losses[0]
    assert after > before + 1.0
