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
