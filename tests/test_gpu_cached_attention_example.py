"""The example of a decode loop over the 8-bit cache: tokens fed one at a time, from a replayed graph, against the same tokens fed at once.

The two differ in how tokens are held: a page's scale grows while its tokens come one by one, and each growth codes the earlier ones again. Keys and
values carry 8 bits, half a step of at most 1 / 254 of a page's largest value (twice that when coded again); queries, keys and outputs are
rounded to BF16 (2^-9) on both sides. A layer's attention averages its values' errors; 2% of the residual stream's norm after two layers
is several times all of these."""
import importlib.util
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
PATH = Path(__file__).resolve().parents[1] / "examples" / "cached_attention.py"


def test_tokens_one_at_a_time(wq):
    spec = importlib.util.spec_from_file_location("cached_attention", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    stepwise, at_once = example.run(prompts=(33, 4, 70, 16), tokens=9)
    assert stepwise.shape == at_once.shape == (9, 4, 512) and torch.isfinite(stepwise).all()
    off = (stepwise.float() - at_once.float()).norm(dim=-1) / at_once.float().norm(dim=-1)
    assert off.max() <= 0.02, off.max().item()
