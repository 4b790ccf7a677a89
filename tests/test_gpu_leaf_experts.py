"""The example that runs the expert-layer operators together: behind a trained tree, with
gradients against differences, and served from 4 bits."""

import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def example():
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "examples"))
    import leaf_experts

    return leaf_experts


def test_layer_learns_inside_the_leaves(example):
    tree, both, losses, off = example.main(rows=6000, steps=40)
    assert both < tree - 0.02      # the layer explains what the tree leaves over
    assert losses[-1] < losses[0]
    # 15 steps over a group's range: a weight moves by up to a thirtieth of it, so outputs by a
    # few percent of their spread; ten times that would be a wrong weight somewhere
    assert off < 0.5


def test_layer_gradients_by_differences(example):
    """Directional differences of the loss in f32 master weights: the forward pass rounds
    weights and activations to bf16 (2^-8), so single directions are noisy; along the
    gradient itself the slope must be its squared norm within a tenth."""
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(2000, 28, generator=g, device="cuda").bfloat16()
    leaf = torch.randint(0, 5, (2000,), generator=g, device="cuda")
    target = torch.randn(2000, generator=g, device="cuda")
    layer = example.LeafExperts(28, 5, seed=4)
    layer.master["head"] *= 10

    def loss():
        score, s = layer.forward(x, leaf)
        return ((score - target) ** 2).mean(), score, s

    _, score, s = loss()
    grads = layer.gradients(2 * (score - target) / len(target), s)
    for name in ("w1", "w2", "head"):  # the gate's steps change the choice of experts
        d = grads[name]
        h = 0.05 * float(layer.master[name].norm() / d.norm())
        values = []
        for sign in (1, -1):
            layer.master[name] += sign * h * d
            values.append(float(loss()[0]))
            layer.master[name] -= sign * h * d
        slope = (values[0] - values[1]) / (2 * h)
        assert abs(slope / float((d * d).sum()) - 1) < 0.1, name
