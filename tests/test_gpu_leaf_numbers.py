"""The leaves that the expert-layer example gives its rows to."""

import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

pytest.importorskip("torch")


def test_leaves_of_equal_value_stay_apart():
    """Any tree of an ensemble, leaves with the same value among them: rows are counted as the
    tree counted them when it was grown."""
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "examples"))
    import leaf_experts as example

    import lightgbm_rs_b200 as lgb
    from lightgbm_rs_b200 import synthetic

    X, y = synthetic.binary_c0(num_data=5000, seed=11)
    params = {"objective": "binary", "num_leaves": 13}
    model = lgb.train(params, lgb.Dataset(X, y, params), num_boost_round=3).model()
    for i, tree in enumerate(model.trees):
        tree["leaf_value"][:] = 0.25
        leaf = example.leaf_numbers(model, i, X)
        count = np.bincount(leaf, minlength=tree["num_leaves"])
        assert count.tolist() == list(tree["leaf_count"])
    leaf, _ = example.leaves_of(X, y, num_leaves=13)
    assert int(leaf.max()) == 12 and len(leaf.unique()) == 13


def test_served_rows_match_their_weights():
    """Single rows served from 4 bits against the same 4-bit weights in 64 bits. On the way h, y and
    the combined row are rounded to bf16 (2^-8 each); products are summed in f32 (2^-23 of the
    magnitudes a term, over 28, 64, 2 and 8 terms); a logit of 28 terms is off by d, a weight by 2 d
    and its own few roundings (2^-20)."""
    import torch

    from test_gpu_experts import unpacked

    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                    "examples"))
    import leaf_experts as example

    g = torch.Generator("cuda").manual_seed(5)
    layer = example.LeafExperts(28, 5, seed=4)
    served = example.Served(layer)
    gate, head = layer.master["gate"], layer.master["head"].double()
    w1 = unpacked(*served.w1, 28, served.size)
    w2 = unpacked(*served.w2, example.HIDDEN, served.size)
    u, f = 2.0 ** -8, 2.0 ** -23
    for i in range(24):
        x = torch.randn(1, 28, generator=g, device="cuda").bfloat16()
        leaf = torch.tensor([i % 5], device="cuda")
        got = float(served(x, leaf))
        logits = (x.float() @ gate).masked_fill_(layer.masked[leaf], -float("inf"))[0]
        top, e = logits.sort(descending=True, stable=True)
        weight, e = top[:example.CHOSEN].double().softmax(0), e[:example.CHOSEN]
        v = x[0].double()
        d = 28 * f * float((v.abs()[:, None] * gate.double().abs())[:, e].sum(0).max())
        h = torch.einsum("ehk,k->eh", w1[e], v).relu()
        dh = u * h + 28 * f * torch.einsum("ehk,k->eh", w1[e].abs(), v.abs())
        y = torch.einsum("enh,eh->en", w2[e], h)
        dy = u * y.abs() + torch.einsum("enh,eh->en", w2[e].abs(), dh + 64 * f * h)
        out = weight @ y
        dout = u * out.abs() + weight @ dy + (2 * d + 2.0 ** -20 + 2 * f) * (weight @ y.abs())
        want = float(out @ head)
        lim = float((dout + 8 * f * out.abs()) @ head.abs())
        assert abs(got - want) <= 1.02 * lim  # products of two roundings: 2 u
