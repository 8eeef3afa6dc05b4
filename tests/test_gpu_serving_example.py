"""The serving operators together, as the example runs them: speculative decoding from the 8-bit cache must
give what decoding one token at a time gives when the target is deterministic."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    spec = importlib.util.spec_from_file_location("speculative_serving", os.path.join(ROOT, "examples", "speculative_serving.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("cache", ["int8", "float8_e4m3fn"])
def test_speculation_does_not_change_greedy_tokens(gpu, cache):
    import torch
    ex = _example()
    model = ex.OneLayer()
    prompt = [int(x) for x in torch.randint(0, 24, (150,), generator=torch.Generator().manual_seed(1))]
    first = [3, 9, 21, 100, 3]
    plain, _ = ex.serve(model, prompt, first, 40, 0, getattr(torch, cache), greedy=True)
    for drafts in (1, 4):
        fast, accepted = ex.serve(model, prompt, first, 40, drafts, getattr(torch, cache), greedy=True)
        for a, b in zip(plain, fast):
            n = min(len(a), len(b))
            assert n >= 41 and a[:n] == b[:n]
        assert sum(map(len, fast)) == 5 + 5 * 40 + accepted


def test_sampled_steps_run(gpu):
    ex = _example()
    model = ex.OneLayer(heads=4, heads_kv=4, head_dim=128)
    texts, accepted = ex.serve(model, [5, 6, 7] * 30, [1, 2], 20, 3)
    assert all(21 <= len(t) <= 1 + 20 * 4 for t in texts) and all(0 <= x < model.vocab for t in texts for x in t)
    assert sum(map(len, texts)) == 2 + 2 * 20 + accepted
