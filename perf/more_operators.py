"""The layers behind the router as they are measured: cases, inputs, plain forms and exact values.

`grouped_gated` is the first half of a gated feed-forward layer in every expert: gate and up
projection, the activation of one times the other. `grouped_linear` is a product with bias,
activation and residual; its dense form is a single expert. Both have backward passes. `clip_grads`
scales a training step's gradients, tensors of any sizes and types, to a largest norm over all of
them; `grad_norm` is that norm alone. Where `own` is false, `run` computes them in elementary torch
operations in 32 bits, rounded once at the end; where it is true it calls
`lightgbm_rs_b200.experts`.
"""

import functools
import importlib
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one row asks two experts of eight: the time is the weights' way from memory
        {"name": "gated, one row served", "op": "gated", "tokens": 1, "k": 2, "experts": 8,
         "inner": 2048, "outer": 4096, "type": "bf16", "act": "silu", "train": False,
         "padded": False},
        # a small ragged batch over 2000 features: nearly every expert's weights are read
        {"name": "gated, 24 rows served", "op": "gated", "tokens": 24, "k": 2, "experts": 32,
         "inner": 2000, "outer": 1024, "type": "f16", "act": "gelu", "train": False,
         "padded": False},
        # an ordinary training step: forward, input gradient, weight gradient
        {"name": "gated, training", "op": "gated", "tokens": 4096, "k": 2, "experts": 8,
         "inner": 1024, "outer": 2048, "type": "bf16", "act": "silu", "train": True,
         "padded": False},
        # a small layer in each of 255 leaves over 700 features: odd widths, ragged and empty
        # groups, padding rows without an expert
        {"name": "gated, 255 leaves, 700 features", "op": "gated", "tokens": 40009, "k": 1,
         "experts": 255, "inner": 700, "outer": 129, "type": "f16", "act": "gelu", "train": True,
         "padded": True},
        # the largest training step
        {"name": "gated, largest", "op": "gated", "tokens": 32768, "k": 2, "experts": 16,
         "inner": 2048, "outer": 2048, "type": "bf16", "act": "silu", "train": True,
         "padded": False},
        # one row through a dense layer behind the experts
        {"name": "linear, one row served", "op": "linear", "tokens": 1, "k": 1, "experts": 1,
         "inner": 4096, "outer": 2048, "type": "bf16", "act": None, "bias": True,
         "residual": True, "train": False, "padded": False},
        # a batch predicted through a dense layer, added to the residual stream
        {"name": "linear, 16384 rows, residual", "op": "linear", "tokens": 16384, "k": 1,
         "experts": 1, "inner": 2048, "outer": 4096, "type": "f16", "act": "gelu", "bias": True,
         "residual": True, "train": False, "padded": False},
        # an ordinary training step of an experts' hidden layer, with the bias's gradient
        {"name": "linear, training", "op": "linear", "tokens": 4096, "k": 2, "experts": 8,
         "inner": 1024, "outer": 4096, "type": "bf16", "act": "relu", "bias": True,
         "residual": False, "train": True, "padded": False},
        # 255 leaves over the 28 features of the default benchmark: many rows, little to multiply
        {"name": "linear, 255 leaves, 28 features", "op": "linear", "tokens": 200003, "k": 1,
         "experts": 255, "inner": 28, "outer": 64, "type": "f16", "act": "silu", "bias": True,
         "residual": False, "train": True, "padded": True},
        # the gradients of one small layer: gate, two matrices, a bias, a head
        {"name": "clip, a small layer", "op": "clip", "tensors": 5, "total": 150001, "type": "f32",
         "flat": False, "ratio": 0.1, "scale": True},
        # a deep model: biases of a few numbers beside matrices, in one buffer without gaps
        {"name": "clip, 1021 ragged tensors", "op": "clip", "tensors": 1021, "total": 60000011,
         "type": "mixed", "flat": True, "ratio": 0.1, "scale": True},
        # the 32-bit weight gradients of the largest layer of experts, both its products
        {"name": "clip, largest", "op": "clip", "tensors": 12, "total": 201326592, "type": "f32",
         "flat": False, "ratio": 0.1, "scale": True},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step`, spread evenly over its logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(step, min(hi, max(lo, n)) // step * step)


def draw(rng):
    op = rng.choice(["gated", "gated", "linear", "linear", "clip"])
    if op == "clip":
        kind = rng.choice(["f32", "bf16", "f16", "mixed"])
        total = _log(rng, 1, 400_000_000 if kind in ("bf16", "f16") else 200_000_000)
        flat = rng.random() < 0.5
        return {"op": op, "tensors": min(total, _log(rng, 1, 1500 if flat else 50)),
                "total": total, "type": kind, "flat": flat,
                "ratio": rng.choice([0.03, 0.3, 0.9, 1.5]), "scale": rng.random() < 0.75}
    # widths: multiples of 64, of 8, or any
    step = rng.choice([64, 8, 1])
    inner, outer = _log(rng, 16, 4000, step), _log(rng, 16, 4000, step)
    width = outer * (2 if op == "gated" else 1)
    experts = 1 if op == "linear" and rng.random() < 0.3 else _log(rng, 1, 256)
    while experts * inner * width > 150_000_000:
        experts = max(1, experts // 2)
    cap = max(1, min(65536, 500_000_000 // (inner * width) * 256))
    case = {"op": op, "tokens": _log(rng, 1, cap), "k": min(experts, rng.choice([1, 2, 4])),
            "experts": experts, "inner": inner, "outer": outer, "type": rng.choice(["bf16", "f16"]),
            "act": rng.choice(["silu", "gelu", "relu"]), "train": rng.random() < 0.6,
            "padded": rng.random() < 0.4}
    if op == "linear":
        if rng.random() < 0.25:
            case["act"] = None
        case["bias"] = rng.random() < 0.75
        case["residual"] = rng.random() < 0.4
    return case


# ------------------------------------------------------------------------------- inputs


def _routing(g, tokens, experts, k, padded):
    """A router's result: distinct experts for every row, some of them favoured. Of a padded batch
    one slot in sixteen has no expert; its row stands behind the last expert's."""
    score = torch.randn(tokens, experts, generator=g, device="cuda")
    if tokens > 64 and experts > 1:  # a large batch is never balanced; one expert in eight is idle
        bias = torch.randn(experts, generator=g, device="cuda") * 0.7
        bias[torch.rand(experts, generator=g, device="cuda") < 0.125] = -100.0
        score += bias
    chosen = score.topk(k, dim=1).indices.reshape(-1)
    if padded and chosen.numel() > 16:
        chosen[torch.rand(chosen.numel(), generator=g, device="cuda") < 1 / 16] = experts
    group, order = chosen.sort(stable=True)
    offsets = torch.searchsorted(group, torch.arange(experts + 1, device="cuda"))
    most = int((offsets[1:] - offsets[:-1]).max())
    return {"rows": (order // k).int(), "offsets": offsets.int(), "most": most}


def _sizes(case):
    """Sizes of the tensors: a few large ones hold most of the elements, every one has some."""
    n, total = case["tensors"], case["total"]
    rng = random.Random(n * 1_000_003 + total)
    share = [math.exp(rng.gauss(0.0, 2.0)) for _ in range(n)]
    whole, left = sum(share), total - n
    sizes = [1 + int(left * v / whole) for v in share]
    sizes[sizes.index(max(sizes))] += total - sum(sizes)
    return sizes


def _kinds(case):
    if case["type"] != "mixed":
        return [_TYPES[case["type"]]] * case["tensors"]
    rng = random.Random(case["tensors"] * 1_000_033 + case["total"])
    return [_TYPES[rng.choice(["f32", "bf16", "bf16", "f16"])] for _ in range(case["tensors"])]


def _tensors(case):
    """Tensors of these sizes, each on its own or one behind the other in a buffer a type, and
    the memory that they lie in."""
    sizes, kinds = _sizes(case), _kinds(case)
    if not case["flat"]:
        out = [torch.empty(n, device="cuda", dtype=t) for n, t in zip(sizes, kinds)]
        return out, out
    held = {}
    for n, t in zip(sizes, kinds):
        held[t] = held.get(t, 0) + n
    buffer = {t: torch.empty(n, device="cuda", dtype=t) for t, n in held.items()}
    at, out = {t: 0 for t in held}, []
    for n, t in zip(sizes, kinds):
        out.append(buffer[t][at[t]:at[t] + n])
        at[t] += n
    return out, list(buffer.values())


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "clip":
        s["grads"], s["held"] = _tensors(case)
        size = random.Random(int(seed))
        for t in s["grads"]:  # layers differ in the size of their gradients by orders
            # (f16's are those of a scaled loss: it has no smaller ones)
            low = -1.0 if t.dtype is torch.float16 else -4.0
            t.normal_(0.0, 10.0 ** size.uniform(low, low + 3.0), generator=g)
        norm = math.sqrt(sum(float(t.double().square().sum()) for t in s["grads"]))
        s["max_norm"] = norm * case["ratio"]
        s["out"], s["memory"] = _tensors(case) if case["scale"] else (None, None)
        return s
    T, K, N, dtype = case["tokens"], case["inner"], case["outer"], _TYPES[case["type"]]
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s.update(_routing(g, T, case["experts"], case["k"], case["padded"]))
    M = T * case["k"]
    if case["experts"] == 1 and not case["padded"]:
        s["rows"] = None  # a dense layer: the rows are its own
    s["x"] = rand(T, K).to(dtype)
    width = 2 * N if case["op"] == "gated" else N
    s["w"] = torch.empty(case["experts"], width, K, device="cuda", dtype=dtype)
    s["w"].normal_(0.0, K ** -0.5, generator=g)
    s["b"] = s["r"] = None
    if case.get("bias"):
        s["b"] = (rand(case["experts"], N) * 0.5).to(dtype)
    if case.get("residual"):
        s["r"] = rand(M, N).to(dtype)
    s["dy"] = rand(M, N).to(dtype) if case["train"] else None
    return s


# -------------------------------------------------------------------------- plain forms


def _act(name, v):
    """The activation and its derivative."""
    if name is None:
        return v, torch.ones_like(v)
    if name == "relu":
        return v.clamp(min=0.0), (v > 0).to(v.dtype)
    if name == "silu":
        q = 1.0 / (1.0 + torch.exp(-v))
        return v * q, q * (1.0 + v * (1.0 - q))
    # gelu: v P(v), P the normal distribution; by erfc, which stays precise where P is small
    p = 0.5 * torch.erfc(v * -(0.5 ** 0.5))
    return v * p, p + v * torch.exp(-0.5 * v * v) * (2.0 * math.pi) ** -0.5


def _plain_layer(s):
    """The experts' rows as one padded batch [experts, most, width]."""
    dtype, E, most = s["x"].dtype, s["experts"], s["most"]
    off = s["offsets"].long()
    x = s["x"].float() if s["rows"] is None else s["x"].float()[s["rows"].long()]
    M = x.shape[0]
    r = torch.arange(M, device=off.device)
    e = torch.searchsorted(off[1:], r, right=True)
    alone = e >= E  # rows of no expert
    place = (e * most + r - off[e.clamp(max=E)]).masked_fill(alone, E * most)

    def lay(a):
        out = a.new_zeros(E * most + 1, a.shape[1])
        out[place] = a.masked_fill(alone[:, None], 0.0)
        return out[:-1].view(E, most, -1)

    def back(a):
        a = a.reshape(E * most, -1)
        return torch.cat([a, a.new_zeros(1, a.shape[1])])[place]

    xp, w = lay(x), s["w"].float()
    pre = torch.bmm(xp, w.transpose(1, 2))
    if s["b"] is not None:
        pre += s["b"].float()[:, None, :]
    N = s["outer"]
    if s["op"] == "gated":
        a, d = _act(s["act"], pre[:, :, :N])
        up = pre[:, :, N:]
        y = back(a * up)
    else:
        a, d = _act(s["act"], pre)
        y = back(a)
        if s["r"] is not None:
            y += s["r"].float()
    out = [y.to(dtype)]
    if not s["train"]:
        return out
    dyp = lay(s["dy"].float())
    dpre = torch.cat([dyp * up * d, dyp * a], 2) if s["op"] == "gated" else dyp * d
    out.append(back(torch.bmm(dpre, w)).to(dtype))
    out.append(torch.bmm(dpre.transpose(1, 2), xp).to(dtype))
    if s["b"] is not None:
        out.append(dpre.sum(1).to(dtype))
    return out


def _plain_clip(s):
    parts = [t.float().square().sum(dtype=torch.float64) for t in s["grads"]]
    norm = torch.stack(parts).sum().sqrt().float()
    if not s["scale"]:
        return [norm]
    scale = (s["max_norm"] / norm).clamp(max=1.0)
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * scale)
    return [norm] + s["memory"]


# ------------------------------------------------------------------- the framework's own


@functools.lru_cache(None)
def _experts():
    return importlib.import_module("lightgbm_rs_b200.experts")


def _own(s):
    ops, op = _experts(), s["op"]
    if op == "clip":
        if not s["scale"]:
            return [ops.grad_norm(s["grads"])]
        return [ops.clip_grads(s["grads"], s["max_norm"], out=s["out"])] + s["memory"]
    if op == "gated":
        if not s["train"]:
            return [ops.grouped_gated(s["x"], s["w"], s["offsets"], rows=s["rows"],
                                      activation=s["act"])]
        h, pre = ops.grouped_gated(s["x"], s["w"], s["offsets"], rows=s["rows"],
                                   activation=s["act"], save=True)
        dx, dw = ops.grouped_gated_backward(s["dy"], pre, s["x"], s["w"], s["offsets"],
                                            rows=s["rows"], activation=s["act"])
        return [h, dx, dw]
    if not s["train"]:
        return [ops.grouped_linear(s["x"], s["w"], s["offsets"], rows=s["rows"], bias=s["b"],
                                   activation=s["act"], residual=s["r"])]
    y, pre = ops.grouped_linear(s["x"], s["w"], s["offsets"], rows=s["rows"], bias=s["b"],
                                activation=s["act"], residual=s["r"], save=True)
    dx, dw, db = ops.grouped_linear_backward(s["dy"], pre, s["x"], s["w"], s["offsets"],
                                             rows=s["rows"], activation=s["act"],
                                             need_dbias=s["b"] is not None)
    return [y, dx, dw] if s["b"] is None else [y, dx, dw, db]


def run(state):
    if own:
        return _own(state)
    return _plain_clip(state) if state["op"] == "clip" else _plain_layer(state)


# -------------------------------------------------------------------------------- work


def _active(case):
    """Experts that see a row at all (on average, for a few rows), and the share of experts
    that a large batch never uses."""
    E, T, k = case["experts"], case["tokens"], case["k"]
    if T > 64 and E > 1:
        return max(1.0, E * 0.875 * (1 - math.exp(-T * k / E)))
    return E * (1 - (1 - k / E) ** T)


def work(case):
    if case["op"] == "clip":
        n = sum(c * t.itemsize for c, t in zip(_sizes(case), _kinds(case)))
        return {"bytes": n * (2 if case["scale"] else 1) + 4,
                "flops": case["total"] * (3 if case["scale"] else 2)}
    b, T, K, N = _BYTES[case["type"]], case["tokens"], case["inner"], case["outer"]
    M, width = T * case["k"], N * (2 if case["op"] == "gated" else 1)
    biased = bool(case.get("bias"))
    n = (T * K + M * N + _active(case) * width * (K + biased)) * b
    n += 4 * (case["experts"] + 1) + (4 * M if case["experts"] > 1 or case["padded"] else 0)
    n += M * N * b if case.get("residual") else 0
    if case["train"]:
        n += (M * N + M * K) * b
        n += case["experts"] * width * (K + biased) * b
    return {"bytes": n, "flops": 2 * M * width * K * (3 if case["train"] else 1)}


# ---------------------------------------------------------------- exact values, 64 bits


def _exact_layer(s):
    """Expert by expert in 64 bits, the gradients by torch's own differentiation."""
    F, off, N = torch.nn.functional, s["offsets"].tolist(), s["outer"]
    act = {None: lambda v: v, "relu": torch.relu, "silu": F.silu, "gelu": F.gelu}[s["act"]]
    M = s["x"].shape[0] if s["rows"] is None else s["rows"].numel()
    y = torch.zeros(M, N, device="cuda", dtype=torch.float64)
    dx = torch.zeros(M, s["inner"], device="cuda", dtype=torch.float64)
    dw, db = [], []
    for e in range(s["experts"]):
        r = slice(off[e], off[e + 1])
        x = s["x"][r] if s["rows"] is None else s["x"][s["rows"][r].long()]
        leaves = [x.double(), s["w"][e].double()]
        if s["b"] is not None:
            leaves.append(s["b"][e].double())
        with torch.enable_grad():
            for v in leaves:
                v.requires_grad_(s["train"])
            pre = F.linear(*leaves)
            out = act(pre[:, :N]) * pre[:, N:] if s["op"] == "gated" else act(pre)
        y[r] = out.detach()
        if s["train"]:
            d = torch.autograd.grad(out, leaves, s["dy"][r].double())
            dx[r] = d[0]
            dw.append(d[1])
            if s["b"] is not None:
                db.append(d[2])
    if s["r"] is not None:
        y += s["r"].double()
    if not s["train"]:
        return [y]
    return [y, dx, torch.stack(dw)] + ([torch.stack(db)] if db else [])


def _exact_clip(s):
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(t.double())) ** 2
                               for t in s["grads"]))
    out = [torch.tensor(norm, dtype=torch.float64, device="cuda")]
    if s["scale"]:
        scale = min(1.0, s["max_norm"] / norm)
        out += [t.double() * scale for t in s["held"]]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_clip(s) if case["op"] == "clip" else _exact_layer(s)
