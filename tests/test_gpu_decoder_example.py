"""GPU: the decoder example, cache to log probabilities, end to end.

A text's log probabilities while it is decoded token by token and when it is
scored in one pass come from the same weights by different kernels and row
counts.  Bound on their difference: bf16 activations carry 2^-9 relative noise
per layer product; over 2 layers x 5 products and the head, of logits with a
standard deviation of 3, a difference of 3 * sqrt(11) * 2^-8 = 0.04 in a logit
is one standard deviation at most; 0.25 is six of them.
"""

import importlib.util
import os

import pytest
from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("code", ["float8_e4m3fn", "int8"])
def test_decoder_example(native, cuda, code):
    import torch
    spec = importlib.util.spec_from_file_location("decoder_step", os.path.join(ROOT, "examples", "decoder_step.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    decoded, scored, ranks = example.run(cuda, steps=20, dtype=getattr(torch, code))
    assert bool((ranks == 1).all())  # greedy tokens are the most likely ones
    for d, s in zip(decoded, scored):
        assert bool(torch.isfinite(d).all()) and float(d.max()) < 0
        assert float((d - s).abs().max()) <= 0.25
