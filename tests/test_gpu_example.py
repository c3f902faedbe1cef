"""examples/hybrid_stack.py: the norm, the convolution and the scan together with the delta rule, served and trained."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def load():
    spec = importlib.util.spec_from_file_location("hybrid_stack", os.path.join(ROOT, "examples", "hybrid_stack.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_a_prompt_and_single_tokens_are_the_whole_sequence():
    # four layers of bfloat16 activations and e4m3 projections: a value that rounds the other way in one path is off by a
    # step of e4m3 (2^-3) in one of 256 terms of a projection, 2^-3 / 16 of the typical size, a few of them meet in a layer
    assert load().serve() < 0.25


def test_training_lowers_the_loss():
    losses = load().train()
    assert losses[-1] < 0.7 * losses[0]
