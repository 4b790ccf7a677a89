"""The expert-layer operators as they are measured: cases, inputs, plain forms and exact values.

A layer of experts works on T rows ("tokens"). `route` picks k of E experts for each and groups
the T*k slots by expert; `grouped_matmul` multiplies each expert's ragged range of rows by its
matrix; `combine` joins the k results of a row; `dropout` regularises; `grouped_matmul_w4` is the
product with 4-bit weights that serves single rows. Where `own` is false, `run` computes them in
elementary torch operations in 32 bits, rounded once at the end; where it is true it calls
`lightgbm_rs_b200.experts`.
"""

import functools
import importlib
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # one row asks for its experts: a launch and nothing else
        {"name": "route one row", "op": "route", "tokens": 1, "experts": 8, "k": 2,
         "type": "f32", "normalize": True, "train": False},
        # a training batch over as many experts as a tree of the default benchmark has leaves,
        # with masked experts and fully masked (padding) rows
        {"name": "route 255 leaves, training", "op": "route", "tokens": 65521, "experts": 255,
         "k": 4, "type": "f32", "normalize": False, "train": True},
        # four rows being served, two experts each: the time is the weights' way from memory
        {"name": "product, 4 rows served", "op": "product", "tokens": 4, "k": 2, "experts": 8,
         "inner": 2048, "outer": 4096, "type": "bf16", "train": False, "grad": "bf16"},
        # an ordinary training step: forward, input gradient, weight gradient
        {"name": "product, training", "op": "product", "tokens": 4096, "k": 2, "experts": 8,
         "inner": 1024, "outer": 4096, "type": "bf16", "train": True, "grad": "bf16"},
        # one small matrix per leaf over 700 features: odd widths, ragged and empty groups,
        # weight gradients kept in 32 bits
        {"name": "product, 255 leaves, 700 features", "op": "product", "tokens": 40009, "k": 1,
         "experts": 255, "inner": 700, "outer": 129, "type": "f16", "train": True, "grad": "f32"},
        # the largest training step
        {"name": "product, largest", "op": "product", "tokens": 32768, "k": 2, "experts": 16,
         "inner": 2048, "outer": 4096, "type": "bf16", "train": True, "grad": "f32"},
        # three rows being served
        {"name": "combine, 3 rows", "op": "combine", "tokens": 3, "k": 2, "width": 700,
         "type": "f32", "train": False},
        # a training batch, with the gradients of the rows and of the weights
        {"name": "combine, training", "op": "combine", "tokens": 16384, "k": 4, "width": 2048,
         "type": "bf16", "train": True},
        # a small hidden layer of odd width
        {"name": "dropout, small", "op": "dropout", "rows": 33, "width": 1001, "type": "f32",
         "p": 0.5, "residual": False, "train": True},
        # the hidden activations of a large batch, added to the residual stream
        {"name": "dropout, large", "op": "dropout", "rows": 32768, "width": 4096, "type": "bf16",
         "p": 0.1, "residual": True, "train": True},
        # one row being served from 4-bit weights, two experts of eight
        {"name": "4-bit product, one row", "op": "w4", "tokens": 1, "k": 2, "experts": 8,
         "inner": 4096, "outer": 4096, "group": 128, "zeros": True, "type": "f16"},
        # a small ragged batch over 2000 features: nearly every expert's weights are read
        {"name": "4-bit product, 16 rows", "op": "w4", "tokens": 16, "k": 4, "experts": 32,
         "inner": 2000, "outer": 4096, "group": 32, "zeros": False, "type": "bf16"},
    ]


def _log(rng, lo, hi, step=1):
    """A multiple of `step`, spread evenly over its logarithm."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    n = max(step, min(hi, max(lo, n)) // step * step)
    return n + step if n == 3 * 1024 else n


def draw(rng):
    op = rng.choice(["route", "product", "product", "combine", "dropout", "w4"])
    if op == "route":
        experts = _log(rng, 2, 512)
        return {"op": op, "tokens": _log(rng, 1, 65536), "experts": experts,
                "k": min(experts, rng.choice([1, 2, 3, 4, 6, 8])),
                "type": rng.choice(["f32", "bf16", "f16"]), "normalize": rng.random() < 0.5,
                "train": rng.random() < 0.7}
    if op == "product":
        # widths: multiples of 64, of 8, or any
        step = rng.choice([64, 8, 1])
        experts = _log(rng, 1, 256)
        train = rng.random() < 0.6
        inner, outer = _log(rng, 16, 4000, step), _log(rng, 16, 4000, step)
        cap = max(1, min(32768, 500_000_000 // (inner * outer) * 256))
        while experts * inner * outer > 150_000_000:
            experts //= 2
        return {"op": op, "tokens": _log(rng, 1, cap), "k": min(experts, rng.choice([1, 2, 4])),
                "experts": experts, "inner": inner, "outer": outer,
                "type": rng.choice(["bf16", "f16"]), "train": train,
                "grad": rng.choice(["f32", "same"])}
    if op == "combine":
        return {"op": op, "tokens": _log(rng, 1, 16384), "k": rng.choice([1, 2, 3, 4, 8]),
                "width": _log(rng, 1, 2048), "type": rng.choice(["bf16", "f16", "f32"]),
                "train": rng.random() < 0.6}
    if op == "dropout":
        kind = rng.choice(["bf16", "f16", "f32"])
        return {"op": op, "rows": _log(rng, 1, 16384 if kind == "f32" else 32768),
                "width": _log(rng, 1, 4096), "type": kind,
                "p": rng.choice([0.1, 0.25, 0.5, round(rng.uniform(0.01, 0.9), 3)]),
                "residual": rng.random() < 0.5, "train": rng.random() < 0.6}
    experts = _log(rng, 1, 64)
    inner, outer = _log(rng, 32, 8192), _log(rng, 16, 8192)
    while experts * inner * outer > 270_000_000:
        experts //= 2
    return {"op": op, "tokens": _log(rng, 1, 32), "k": min(experts, rng.choice([1, 2, 4])),
            "experts": experts, "inner": inner, "outer": outer,
            "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
            "type": rng.choice(["bf16", "f16"])}


# ------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator("cuda").manual_seed(int(seed))


def _logits(g, tokens, experts, dtype):
    """Logits of a gate that favours some experts, some experts masked (-inf) or set to the
    type's lowest value, and one row in sixteen masked whole (padding)."""
    x = torch.randn(tokens, experts, generator=g, device="cuda")
    x += torch.randn(experts, generator=g, device="cuda")
    u = torch.rand(tokens, experts, generator=g, device="cuda")
    x = x.to(dtype)
    x.masked_fill_(u < 0.02, torch.finfo(dtype).min)
    masked = u > 0.9
    masked |= torch.rand(tokens, 1, generator=g, device="cuda") < (1 / 16 if tokens > 16 else 0)
    if tokens == 1:
        masked.zero_()
    return x.masked_fill_(masked, -math.inf)


def _routing(g, tokens, experts, k):
    """A router's result: distinct experts for every row, some of them favoured."""
    score = torch.randn(tokens, experts, generator=g, device="cuda")
    if tokens > 64:  # a large batch is never balanced; one expert in eight sees nothing at all
        bias = torch.randn(experts, generator=g, device="cuda") * 0.7
        bias[torch.rand(experts, generator=g, device="cuda") < 0.125] = -100.0
        score += bias
    chosen = score.topk(k, dim=1).indices.reshape(-1)
    group, order = chosen.sort(stable=True)
    offsets = torch.searchsorted(group, torch.arange(experts + 1, device="cuda"))
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device="cuda")
    most = int((offsets[1:] - offsets[:-1]).max())
    return {"rows": (order // k).int(), "offsets": offsets.int(), "most": most,
            "position": position.view(tokens, k).int()}


def prepare(case, seed):
    g = _generator(seed)
    op, dtype = case["op"], _TYPES[case["type"]]
    rand = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = dict(case)
    if op == "route":
        s["logits"] = _logits(g, case["tokens"], case["experts"], dtype)
        s["dweights"] = rand(case["tokens"], case["k"])
    elif op == "product":
        s.update(_routing(g, case["tokens"], case["experts"], case["k"]))
        K, N = case["inner"], case["outer"]
        s["x"] = rand(case["tokens"], K).to(dtype)
        s["w"] = torch.empty(case["experts"], N, K, device="cuda", dtype=dtype)
        s["w"].normal_(0.0, K ** -0.5, generator=g)
        s["dy"] = rand(case["tokens"] * case["k"], N).to(dtype) if case["train"] else None
        s["grad"] = torch.float32 if case["grad"] == "f32" else dtype
    elif op == "combine":
        T, k, N = case["tokens"], case["k"], case["width"]
        s["position"] = torch.randperm(T * k, generator=g, device="cuda").view(T, k).int()
        s["weights"] = rand(T, k).softmax(1)
        s["y"] = rand(T * k, N).to(dtype)
        s["dout"] = rand(T, N).to(dtype) if case["train"] else None
    elif op == "dropout":
        shape = (case["rows"], case["width"])
        s["x"] = rand(*shape).to(dtype)
        s["residual"] = rand(*shape).to(dtype) if case["residual"] else None
        s["dout"] = rand(*shape).to(dtype) if case["train"] else None
        s["seed"], s["offset"] = (int(seed) * 0x9E3779B97F4A7C15) % (1 << 64), int(seed) % 1000
    elif op == "w4":
        s.update(_routing(g, case["tokens"], case["experts"], case["k"]))
        E, K, N = case["experts"], case["inner"], case["outer"]
        groups = -(-K // case["group"])
        # two weights a byte, the even one in the low half; rows padded to 16 bytes with zeros
        pitch = (K + 31) // 32 * 16
        s["q"] = torch.randint(0, 256, (E, N, pitch), generator=g, device="cuda",
                               dtype=torch.uint8)
        s["q"][:, :, (K + 1) // 2:] = 0
        if K % 2:
            s["q"][:, :, K // 2] &= 15
        s["scales"] = ((torch.rand(E, N, groups, generator=g, device="cuda") + 0.5)
                       * (0.2 * K ** -0.5)).to(dtype)
        s["z"] = torch.randint(4, 12, (E, N, groups), generator=g, device="cuda",
                               dtype=torch.uint8) if case["zeros"] else None
        s["x"] = rand(case["tokens"], K).to(dtype)
    return s


# -------------------------------------------------------------------------- plain forms


def _plain_route(s):
    k, l = s["k"], s["logits"].float()
    top, experts = l.sort(dim=1, descending=True, stable=True)
    top, experts = top[:, :k], experts[:, :k]
    empty = top == -math.inf
    m = top[:, :1].masked_fill(empty[:, :1], 0.0)
    ex = torch.exp(top - m)
    total = (ex if s["normalize"] else torch.exp(l - m)).sum(1, keepdim=True)
    weights = torch.where(empty, torch.zeros_like(ex), ex / total)
    experts = experts.masked_fill(empty, -1)
    flat = experts.reshape(-1)
    key = torch.where(flat < 0, torch.full_like(flat, s["experts"]), flat)
    group, order = key.sort(stable=True)
    offsets = torch.searchsorted(group, torch.arange(s["experts"] + 1, device=l.device))
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=l.device)
    out = [weights, experts.int(), position.view(-1, k).int(), (order // k).int(), offsets.int()]
    if s["train"]:
        g = s["dweights"].masked_fill(empty, 0.0)
        inner = (weights * g).sum(1, keepdim=True)
        d = torch.zeros_like(l) if s["normalize"] else -inner * torch.where(
            total > 0, torch.exp(l - m) / total, torch.zeros_like(l))
        at = experts.clamp(min=0).long()
        d.scatter_add_(1, at, weights * (g - inner) if s["normalize"] else weights * g)
        out.append(d.to(s["logits"].dtype))
    return out


def _padded(s, rows):
    """Each expert's rows as one padded batch: the row of every place (`rows` where there is
    none) and the place of every row."""
    off = s["offsets"].long()
    c = torch.arange(s["most"], device=off.device)
    at = off[:-1, None] + c
    at = torch.where(at < off[1:, None], at, torch.full_like(at, rows))
    r = torch.arange(rows, device=off.device)
    e = torch.searchsorted(off[1:], r, right=True)
    return at, e * s["most"] + (r - off[e])


def _lay(a, at):
    """Rows of `a` laid into the padded batch, zeros where there is none."""
    a = torch.cat([a, a.new_zeros(1, a.shape[1])])
    return a[at]


def _plain_product(s):
    x, w = s["x"].float()[s["rows"].long()], s["w"].float()
    at, place = _padded(s, x.shape[0])
    xp = _lay(x, at)
    y = torch.bmm(xp, w.transpose(1, 2)).flatten(0, 1)[place].to(s["x"].dtype)
    if not s["train"]:
        return [y]
    dyp = _lay(s["dy"].float(), at)
    dx = torch.bmm(dyp, w).flatten(0, 1)[place].to(s["x"].dtype)
    return [y, dx, torch.bmm(dyp.transpose(1, 2), xp).to(s["grad"])]


def _plain_combine(s):
    at, w = s["position"].long(), s["weights"]
    y = s["y"].float()[at]
    out = [(w[:, :, None] * y).sum(1).to(s["y"].dtype)]
    if s["train"]:
        d = s["dout"].float()
        dy = torch.empty_like(s["y"])
        dy[at] = (w[:, :, None] * d[:, None, :]).to(dy.dtype)
        out += [dy, (y * d[:, None, :]).sum(2)]
    return out


def _philox(blocks, seed, offset):
    """Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): counter (block, offset), key = seed;
    four words of 32 bits for every block, in int64."""
    low = 0xFFFFFFFF
    i = torch.arange(blocks, device="cuda")
    c0, c1 = i & low, i >> 32
    c2, c3 = torch.full_like(i, offset & low), torch.full_like(i, offset >> 32)
    k0, k1 = seed & low, seed >> 32

    def mul(m, c):  # high and low word of m * c, by halves: the product does not fit int64
        a, b = m * (c & 0xFFFF), m * (c >> 16)
        return ((b + (a >> 16)) >> 16) & low, (a + ((b & 0xFFFF) << 16)) & low

    for _ in range(10):
        h0, l0 = mul(0xD2511F53, c0)
        h1, l1 = mul(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([c0, c1, c2, c3], 1)


def _plain_dropout(s):
    x, n = s["x"].float(), s["x"].numel()
    words = _philox(-(-n // 8), s["seed"], s["offset"])
    halves = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n].view(x.shape)
    drop = int(math.floor(s["p"] * 65536 + 0.5))
    keep, scale = halves >= drop, 65536.0 / (65536 - drop) if drop < 65536 else 0.0
    zero = torch.zeros_like(x)
    out = torch.where(keep, x * scale, zero)
    out = [(out if s["residual"] is None else out + s["residual"].float()).to(s["x"].dtype)]
    if s["train"]:
        out.append(torch.where(keep, s["dout"].float() * scale, zero).to(s["x"].dtype))
    return out


def _plain_w4(s):
    K, G = s["inner"], s["group"]
    q = torch.stack([s["q"] & 15, s["q"] >> 4], 3).flatten(2)[:, :, :K].float()
    spread = lambda a: a.float().repeat_interleave(G, 2)[:, :, :K]  # noqa: E731
    w = spread(s["scales"]) * (q - (8.0 if s["z"] is None else spread(s["z"])))
    x = s["x"].float()[s["rows"].long()]
    at, place = _padded(s, x.shape[0])
    y = torch.bmm(_lay(x, at), w.transpose(1, 2))
    return [y.flatten(0, 1)[place].to(s["x"].dtype)]


_PLAIN = {"route": _plain_route, "product": _plain_product, "combine": _plain_combine,
          "dropout": _plain_dropout, "w4": _plain_w4}


# ------------------------------------------------------------------- the framework's own


@functools.lru_cache(None)
def _experts():
    return importlib.import_module("lightgbm_rs_b200.experts")


def _own(s):
    ops, op = _experts(), s["op"]
    if op == "route":
        r = ops.route(s["logits"], s["k"], normalize=s["normalize"])
        out = [r.weights, r.experts, r.position, r.rows, r.offsets]
        if s["train"]:
            out.append(ops.route_backward(s["dweights"], s["logits"], r,
                                          normalize=s["normalize"]))
        return out
    if op == "product":
        out = [ops.grouped_matmul(s["x"], s["w"], s["offsets"], rows=s["rows"])]
        if s["train"]:
            out += ops.grouped_matmul_backward(s["dy"], s["x"], s["w"], s["offsets"],
                                               rows=s["rows"], grad_dtype=s["grad"])
        return out
    if op == "combine":
        out = [ops.combine(s["y"], s["position"], s["weights"])]
        if s["train"]:
            out += ops.combine_backward(s["dout"], s["y"], s["position"], s["weights"])
        return out
    if op == "dropout":
        out = [ops.dropout(s["x"], s["p"], s["seed"], s["offset"], residual=s["residual"])]
        if s["train"]:
            out.append(ops.dropout_backward(s["dout"], s["p"], s["seed"], s["offset"]))
        return out
    return [ops.grouped_matmul_w4(s["x"], s["q"], s["scales"], s["offsets"], zeros=s["z"],
                                  rows=s["rows"], group_size=s["group"])]


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# -------------------------------------------------------------------------------- work


def _active(case):
    """Experts that see a row at all (on average, for a few rows), and the share of experts
    that a large batch never uses."""
    E, T, k = case["experts"], case["tokens"], case["k"]
    if T > 64:
        return max(1.0, E * 0.875 * (1 - math.exp(-T * k / E)))
    return E * (1 - (1 - k / E) ** T)


def work(case):
    op, b = case["op"], _BYTES[case["type"]]
    if op == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        n, f = T * E * b + T * k * 16 + 4 * (E + 1), T * E
        if case["train"]:
            n += T * k * 4 + T * E * b
            f += 2 * T * E
        return {"bytes": n, "flops": f}
    if op == "product":
        T, M, K, N = case["tokens"], case["tokens"] * case["k"], case["inner"], case["outer"]
        weights = _active(case) * N * K
        n = (T * K + M * N + weights) * b + 4 * M
        if case["train"]:
            n += (M * N + M * K) * b
            n += case["experts"] * N * K * (4 if case["grad"] == "f32" else b)
        return {"bytes": n, "flops": 2 * M * N * K * (3 if case["train"] else 1)}
    if op == "combine":
        T, M, N = case["tokens"], case["tokens"] * case["k"], case["width"]
        n, f = (M + T) * N * b + 8 * M, 2 * M * N
        if case["train"]:
            n += (M + T) * N * b + 4 * M
            f += 3 * M * N
        return {"bytes": n, "flops": f}
    if op == "dropout":
        n = case["rows"] * case["width"]
        passes = 2 + bool(case["residual"]) + (2 if case["train"] else 0)
        return {"bytes": n * b * passes, "flops": 2 * n * (2 if case["train"] else 1)}
    T, M, K, N = case["tokens"], case["tokens"] * case["k"], case["inner"], case["outer"]
    groups = -(-K // case["group"])
    n = _active(case) * N * (K / 2 + groups * (b + bool(case["zeros"])))
    return {"bytes": n + (T * K + M * N) * b, "flops": 2 * M * N * K}


# ---------------------------------------------------------------- exact values, 64 bits


def _exact_route(s):
    l, k = s["logits"].double().cpu().numpy(), s["k"]
    import numpy as np

    T, E = l.shape
    order = np.argsort(-l, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(l, order, 1)
    taken = top > -np.inf
    m = np.where(taken[:, :1], top[:, :1], 0.0)
    ex, full = np.exp(top - m), np.exp(l - m)
    total = (ex if s["normalize"] else full).sum(1, keepdims=True)
    w = np.divide(ex, total, out=np.zeros_like(ex), where=taken)
    out = [w, None, None, None, None]
    if s["train"]:
        g = np.where(taken, s["dweights"].double().cpu().numpy(), 0.0)
        chosen = np.zeros((T, E))
        np.put_along_axis(chosen, order, np.where(taken, 1.0, 0.0), 1)
        grad = np.zeros((T, E))
        np.put_along_axis(grad, order, g, 1)
        p = np.divide(full * (chosen if s["normalize"] else 1.0), total,
                      out=np.zeros_like(full), where=total > 0)
        out.append(p * (grad - (p * grad).sum(1, keepdims=True)))
    return out


def _exact_product(s, w=None):
    off = s["offsets"].tolist()
    x = s["x"].double()[s["rows"].long()]
    dy = s["dy"].double() if s.get("train") else None
    y, dx, dw = [], [], []
    for e in range(s["experts"]):
        r = slice(off[e], off[e + 1])
        m = s["w"][e].double() if w is None else w(e)
        y.append(x[r] @ m.T)
        if dy is not None:
            dx.append(dy[r] @ m)
            dw.append((dy[r].T @ x[r])[None])
    return [torch.cat(y)] if dy is None else [torch.cat(y), torch.cat(dx), torch.cat(dw)]


def _exact_combine(s):
    T, k = s["position"].shape
    inverse = torch.argsort(s["position"].reshape(-1).long())
    token = inverse // k
    y, w = s["y"].double(), s["weights"].double().reshape(-1)[inverse]
    out = [torch.zeros(T, y.shape[1], device="cuda", dtype=torch.float64).index_add_(
        0, token, w[:, None] * y)]
    if s["train"]:
        d = s["dout"].double()[token]
        dots = torch.empty(T * k, device="cuda", dtype=torch.float64)
        dots[inverse] = torch.einsum("mn,mn->m", d, y)
        out += [w[:, None] * d, dots.view(T, k)]
    return out


def _exact_dropout(s):
    import numpy as np

    n = s["x"].numel()
    u = np.uint64
    low, half = u(0xFFFFFFFF), u(32)
    block = np.arange(-(-n // 8), dtype=np.uint64)
    c = [block & low, block >> half, np.full_like(block, s["offset"] & 0xFFFFFFFF),
         np.full_like(block, s["offset"] >> 32)]
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for _ in range(10):
        p, q = c[0] * u(0xD2511F53), c[2] * u(0xCD9E8D57)
        c = [(q >> half) ^ c[1] ^ u(key[0]), q & low, (p >> half) ^ c[3] ^ u(key[1]), p & low]
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    bits = np.stack(c, 1).astype(np.uint32).view(np.uint16).reshape(-1)[:n]
    drop = int(math.floor(s["p"] * 65536 + 0.5))
    scale = 65536.0 / (65536 - drop) if drop < 65536 else 0.0
    keep = torch.from_numpy((bits >= drop).astype(np.float64) * scale).cuda().view(s["x"].shape)
    out = [s["x"].double() * keep]
    if s["residual"] is not None:
        out[0] += s["residual"].double()
    return out + [s["dout"].double() * keep] if s["train"] else out


def _exact_w4(s):
    K, G = s["inner"], s["group"]
    group = torch.arange(K, device="cuda") // G

    def matrix(e):
        byte = s["q"][e].long()[:, torch.arange(K, device="cuda") // 2]
        q = (byte >> (4 * (torch.arange(K, device="cuda") % 2))) % 16
        z = 8 if s["z"] is None else s["z"][e].long()[:, group]
        return (q - z).double() * s["scales"][e].double()[:, group]

    return _exact_product(s, matrix)


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "product": _exact_product, "combine": _exact_combine,
            "dropout": _exact_dropout, "w4": _exact_w4}[case["op"]](s)
