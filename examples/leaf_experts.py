"""A layer of experts behind a tree: one boosted tree splits the rows, and small networks learn
what is left inside its leaves.

Every leaf has `PER_LEAF` experts of its own and there are `SHARED` for all rows. A learned gate
picks two experts for each row among those its leaf allows (the others are masked with -inf).
The layer trains with hand-written gradients and is then laid out in 4 bits to serve single
rows:  python examples/leaf_experts.py
"""

import copy
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import lightgbm_rs_b200 as lgb  # noqa: E402
from lightgbm_rs_b200 import experts, synthetic  # noqa: E402

PER_LEAF, SHARED, HIDDEN, OUT, CHOSEN, DROP = 2, 4, 64, 8, 2, 0.1


def leaf_numbers(model, tree, X):
    """The leaf that tree number `tree` of the model sends each row to: the same tree with its
    leaves' numbers as their values, predicted."""
    t = dict(model.trees[tree])
    t["leaf_value"] = np.arange(t["num_leaves"], dtype=np.float64)
    numbered = copy.copy(model)
    numbered.trees = [t]
    return lgb.Predictor(numbered).predict(X, raw_score=True).astype(np.int64)


def leaves_of(X, y, num_leaves=16):
    """One tree on the data: the rows' leaf numbers and raw scores."""
    params = {"objective": "binary", "num_leaves": num_leaves, "learning_rate": 1.0}
    booster = lgb.train(params, lgb.Dataset(X, y, params), num_boost_round=1)
    leaf = torch.from_numpy(leaf_numbers(booster.model(), 0, X))
    return leaf.cuda(), torch.from_numpy(booster.predict(X, raw_score=True)).float().cuda()


class LeafExperts:
    """gate [K, E]; w1 [E, H, K], w2 [E, OUT, H] in bf16 with f32 copies that the steps update;
    head [OUT]."""

    def __init__(self, width, leaves, seed=0):
        g = torch.Generator("cuda").manual_seed(seed)
        E = leaves * PER_LEAF + SHARED
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.master = {"gate": rand(width, E) * 0.1, "w1": rand(E, HIDDEN, width) * width ** -0.5,
                       "w2": rand(E, OUT, HIDDEN) * HIDDEN ** -0.5, "head": rand(OUT) * 0.1}
        self.moment = {k: (torch.zeros_like(v), torch.zeros_like(v))
                       for k, v in self.master.items()}
        owner = torch.arange(leaves, device="cuda").repeat_interleave(PER_LEAF)
        owner = torch.cat([owner, torch.full((SHARED,), -1, device="cuda")])
        n = torch.arange(leaves, device="cuda")[:, None]
        self.masked = (owner >= 0) & (owner != n)  # [leaves, E]
        self.steps = 0

    def forward(self, x, leaf, seed=None):
        """Scores of the rows, and what the gradient needs. Dropout only with a seed."""
        s = {"x": x, "seed": seed}
        s["w1"], s["w2"] = (self.master[k].bfloat16() for k in ("w1", "w2"))
        s["logits"] = (x.float() @ self.master["gate"]).masked_fill_(self.masked[leaf], -math.inf)
        r = s["routing"] = experts.route(s["logits"], CHOSEN)
        s["pre"] = experts.grouped_matmul(x, s["w1"], r.offsets, rows=r.rows)
        s["act"] = s["pre"].relu()
        if seed is not None:
            s["act"] = experts.dropout(s["act"], DROP, seed, self.steps)
        s["y"] = experts.grouped_matmul(s["act"], s["w2"], r.offsets)
        s["out"] = experts.combine(s["y"], r.position, r.weights)
        return s["out"].float() @ self.master["head"], s

    def gradients(self, dscore, s):
        r = s["routing"]
        g = {"head": s["out"].float().T @ dscore}
        dout = (dscore[:, None] * self.master["head"]).bfloat16()
        dy, dweights = experts.combine_backward(dout, s["y"], r.position, r.weights)
        dact, g["w2"] = experts.grouped_matmul_backward(dy, s["act"], s["w2"], r.offsets,
                                                        grad_dtype=torch.float32)
        if s["seed"] is not None:
            dact = experts.dropout_backward(dact, DROP, s["seed"], self.steps)
        dpre = dact.masked_fill(s["pre"] <= 0, 0.0)
        _, g["w1"] = experts.grouped_matmul_backward(dpre, s["x"], s["w1"], r.offsets,
                                                     rows=r.rows, grad_dtype=torch.float32,
                                                     need_dx=False)
        dlogits = experts.route_backward(dweights, s["logits"], r)
        g["gate"] = s["x"].float().T @ dlogits
        return g

    def step(self, x, leaf, base, label, rate=3e-3, seed=1234):
        """One Adam step on the logistic loss of base + layer; returns the loss before it."""
        score, s = self.forward(x, leaf, seed)
        p = torch.sigmoid(base + score)
        g = self.gradients((p - label) / len(label), s)
        self.steps += 1
        for k, w in self.master.items():
            m, v = self.moment[k]
            m.mul_(0.9).add_(g[k], alpha=0.1)
            v.mul_(0.99).addcmul_(g[k], g[k], value=0.01)
            a, b = 1 - 0.9 ** self.steps, 1 - 0.99 ** self.steps
            w.addcdiv_(m / a, (v / b).sqrt_().add_(1e-8), value=-rate)
        return torch.nn.functional.binary_cross_entropy(p, label)


class Served:
    """The layer with 4-bit experts, for a few rows at a time."""

    def __init__(self, layer, group_size=32):
        self.layer, self.size = layer, group_size
        self.w1, self.w2 = (experts.quantize_w4(layer.master[k].bfloat16(), group_size)
                            for k in ("w1", "w2"))

    def __call__(self, x, leaf):
        m = self.layer.master
        logits = (x.float() @ m["gate"]).masked_fill_(self.layer.masked[leaf], -math.inf)
        r = experts.route(logits, CHOSEN)
        (q1, s1, z1), (q2, s2, z2) = self.w1, self.w2
        h = experts.grouped_matmul_w4(x, q1, s1, r.offsets, zeros=z1, rows=r.rows,
                                      group_size=self.size).relu_()
        y = experts.grouped_matmul_w4(h, q2, s2, r.offsets, zeros=z2, group_size=self.size)
        return experts.combine(y, r.position, r.weights).float() @ m["head"]


def main(rows=20_000, steps=60):
    X, y = synthetic.binary_c0(num_data=rows, seed=7)
    leaf, base = leaves_of(X, y)
    x = torch.from_numpy(X).cuda()
    x = ((x - x.mean(0)) / x.std(0)).bfloat16()
    label = torch.from_numpy(y).cuda()
    layer = LeafExperts(x.shape[1], int(leaf.max()) + 1)
    losses = [float(layer.step(x, leaf, base, label)) for _ in range(steps)]
    tree = float(torch.nn.functional.binary_cross_entropy_with_logits(base, label))
    score, _ = layer.forward(x, leaf)
    both = float(torch.nn.functional.binary_cross_entropy_with_logits(base + score, label))
    served = Served(layer)
    few = torch.cat([served(x[i:i + 1], leaf[i:i + 1]) for i in range(32)])
    off = float((few - score[:32]).abs().max() / score.std())
    experts.check_errors()
    print(f"logistic loss: tree {tree:.4f}, with experts {both:.4f} (step 1: {losses[0]:.4f}, "
          f"step {steps}: {losses[-1]:.4f}); 4-bit rows off by {off:.3f} standard deviations")
    return tree, both, losses, off


if __name__ == "__main__":
    main()
