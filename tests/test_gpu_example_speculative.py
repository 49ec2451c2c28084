"""examples/speculative.py: drafts change how many passes decoding takes, not its tokens (GPU)."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("speculative", os.path.join(ROOT, "examples", "speculative.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_drafts_do_not_change_the_tokens(cuda):
    m = example()
    model, prompts = m.Toy(), [[3, 1, 4, 1, 5, 9, 2, 6] * 9, [2, 7, 1, 8, 2, 8, 1, 8] * 9]
    one, steps, _ = m.generate(model, prompts, 60, 400, 64, False)
    many, passes, evictions = m.generate(model, prompts, 60, 400, 64, True)
    assert one == many and passes <= steps == 59 and evictions == 0


def test_a_bounded_cache_goes_on(cuda):
    m = example()
    out, _, evictions = m.generate(m.Toy(), [[3, 1, 4, 1, 5, 9, 2, 6] * 9] * 3, 200, 128, 48, True)
    assert evictions >= 2 and all(len(o) == 200 for o in out) and out[0] == out[1] == out[2]
