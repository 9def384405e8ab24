"""The example layer: what it generates token by token is what its training form computes, and it learns (CUDA).

Both forms run the same formulas in float32 on the same rows, so they differ by the order of sums alone: projections of 256 terms, scores of
64, two dozen weights, an output of 512 terms, each off by its number of terms times 2^-24 of the sum of magnitudes; together under 2000 *
2^-24 = 1.2e-4 of the largest entry."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu


def _example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "mixer_layer.py")
    spec = importlib.util.spec_from_file_location("mixer_layer", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("prompt,total", [(8, 61), (40, 75)])
def test_tokens_one_by_one_are_the_training_form(prompt, total):
    E = _example()
    torch.manual_seed(3)
    layer = E.MixerLayer().cuda()
    x = torch.randn(3, total, 256, device="cuda")
    with torch.no_grad():
        want = layer(x)
        gen = E.Generation(layer, 3, torch.float32, "cuda")
        got = [gen.prompt(x[:, :prompt])] + [gen.step(x[:, t:t + 1]) for t in range(prompt, total)]
    off = (torch.cat(got, 1) - want).abs().max()
    assert off <= 1.2e-4 * want.abs().max(), off


def test_it_learns_and_generates():
    E = _example()
    torch.manual_seed(0)
    model = E.Model().to("cuda", torch.bfloat16)
    losses = E.train(model, steps=150)
    assert losses[0] > 3.5 and losses[-1] < 0.5 * losses[0]
    tokens = E.sequences(4, 64, torch.Generator().manual_seed(1))
    assert E.generate(model, tokens[:, :64], 20).shape == (4, 20)
