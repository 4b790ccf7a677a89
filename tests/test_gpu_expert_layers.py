"""Gated and linear expert layers on the GPU against plain implementations in 64 bits.

Tolerances are bounds, not fits. A product of n terms in f32 is off by at most 1.1 n 2^-23 times
the sum of the terms' magnitudes (every addition rounds or cuts off once). The activations' values
are good to VALUE of themselves and their slopes to SLOPE (derived at `activation64`). Every result
is rounded once to its type, and so is the gradient of what the activation was given, on its way
into the products.
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_experts import DTYPES, UNIT, close, gen, offsets_of  # noqa: E402

# exp in f32 is off by 2 + 1.16 |v| units of 2^-23 at v: 3.3e-6 at the 22 that arguments stay
# below here; a quotient adds 2 units. silu's value has that error, its slope
# s (1 + v (1 - s)) twice that plus v times the 2^-22 of 1 - s: 1.2e-5. gelu's tail is fitted to
# 5.4e-6 and takes an exp of at most 20 (6.6e-6 with its argument's rounding): 1.2e-5 and half a
# unit for each of eight operations; its slope adds 0.25 of the same.
VALUE, SLOPE = 2e-5, 2e-5


@pytest.fixture(scope="module")
def ops():
    from lightgbm_rs_b200 import experts

    yield experts
    experts.check_errors()


def activation64(name, v):
    """Value and slope in f64."""
    if name is None:
        return v, torch.ones_like(v)
    if name == "relu":
        return v.clamp(min=0), (v > 0).double()
    if name == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    p = 0.5 * torch.special.erfc(-v / math.sqrt(2))
    return v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)


def ranges(off, experts):
    o = off.tolist()
    return [slice(o[e], o[e + 1]) for e in range(experts)]


def grouped64(x, w, off):
    """Products and the sums of their terms' magnitudes; 0 for rows of no expert."""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(y)
    for e, s in enumerate(ranges(off, w.shape[0])):
        y[s] = x[s].double() @ w[e].double().T
        mag[s] = x[s].double().abs() @ w[e].double().abs().T
    return y, mag


def owned(off, experts, m):
    """Which of m rows belong to an expert."""
    own = torch.zeros(m, 1, dtype=torch.bool, device="cuda")
    for s in ranges(off, experts):
        own[s] = True
    return own


def gradients64(dpre, err, x, w, off):
    """dx and dw of products whose gradient dpre is off by err, with bounds for both."""
    dx, dw = torch.zeros(x.shape, dtype=torch.float64, device="cuda"), []
    xb, wb = torch.zeros_like(dx), []
    far = dpre.abs() + err
    n, f = w.shape[1], 1.1 * 2.0 ** -23
    for e, s in enumerate(ranges(off, w.shape[0])):
        we, xs = w[e].double(), x[s].double()
        dx[s] = dpre[s] @ we
        xb[s] = err[s] @ we.abs() + n * f * (far[s] @ we.abs())
        dw.append(dpre[s].T @ xs)
        wb.append(err[s].T @ xs.abs() + max(1, xs.shape[0]) * f * (far[s].T @ xs.abs()))
    return dx, xb, torch.stack(dw), torch.stack(wb)


LAYERS = [  # counts, tail rows, inner, outer
    ([1], 0, 16, 8),                   # streamed: one row
    ([1, 0, 2], 1, 40, 24),
    ([0, 3, 1], 0, 700, 129),          # rows at 8 bytes
    ([5, 9], 2, 2000, 200),            # a split inner axis
    ([2, 2], 0, 1027, 65),             # rows at 2 bytes
    ([30] * 4, 3, 130, 33),            # rows at 4 bytes, items of 32 rows
    ([200, 0, 77], 3, 72, 20),         # tiles of 64 columns
    ([200, 77], 0, 72, 50),            # of 128
    ([150, 0, 90, 3], 5, 264, 136),    # of 256
    ([90, 0, 100, 0], 0, 64, 128),
    ([300, 129, 1000], 0, 200, 264),   # pairs
    ([257, 31, 400], 200, 129, 700),
    ([700], 0, 1000, 257),
    ([600], 0, 4200, 136),             # a reduction in two runs, by pairs
    ([100, 60], 4, 8300, 40),          # in three
    ([130], 0, 4112, 24),              # two runs in tiles of 64 columns
    ([33] * 200, 9, 28, 64),           # many groups, little to multiply
    ([0, 0], 5, 48, 40),               # no expert has rows
    ([3, 0, 40], 2, 40, 1100),         # input gradients summed in parts of the reduction
    ([70, 9], 0, 130, 2050),
    ([64], 1, 300, 1037),
    ([4000, 1, 0, 900], 3, 56, 40),    # narrow weight gradients in parts of the rows
    ([9000], 0, 30, 24),
    ([5], 0, 24, 4099),                # few long rows, divided among blocks
]


def layer(counts, tail, inner, outer, dt, seed, halves=1):
    g = gen(seed + inner * 7 + outer)
    m, E = sum(counts) + tail, len(counts)
    x = torch.randn(m, inner, generator=g, device="cuda").to(dt)
    w = (torch.randn(E, halves * outer, inner, generator=g, device="cuda") * inner ** -0.5).to(dt)
    dy = torch.randn(m, outer, generator=g, device="cuda").to(dt)
    if tail:  # rows of no expert hold what they like
        x[-1], dy[-1] = math.nan, math.inf
    return g, m, E, x, w, dy, offsets_of(counts)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
@pytest.mark.parametrize("counts,tail,inner,outer", LAYERS)
def test_gated(ops, counts, tail, inner, outer, act, dtype):
    dt = DTYPES[dtype]
    g, m, E, x, w, dh, off = layer(counts, tail, inner, outer, dt, 1, halves=2)
    p64, mag = grouped64(x, w, off)
    eps = 1.1 * inner * 2.0 ** -23 * mag
    gate, up, eg, eu = p64[:, :outer], p64[:, outer:], eps[:, :outer], eps[:, outer:]
    a, _ = activation64(act, gate)
    slack = 1.2 * eg * (up.abs() + eu) + a.abs() * eu + (VALUE + 2.0 ** -22) * (a * up).abs()
    h, pre = ops.grouped_gated(x, w, off, activation=act, save=True)
    close(h, a * up, slack)
    assert pre.shape == (m, 2, outer) and pre.dtype == dt
    close(pre[:, 0], gate, eg)
    close(pre[:, 1], up, eu)
    assert torch.equal(ops.grouped_gated(x, w, off, activation=act), h)

    dx, dw = ops.grouped_gated_backward(dh, pre, x, w, off, activation=act)
    own = owned(off, E, m)
    d = torch.where(own, dh.double(), 0.0)
    gate, up = pre[:, 0].double(), pre[:, 1].double()
    a, s = activation64(act, gate)
    dpre = torch.cat([d * up * s, d * a], 1)
    err = torch.cat([(d * up).abs() * (SLOPE + 2.0 ** -22), (d * a).abs() * (VALUE + 2.0 ** -22)], 1)
    err += UNIT[dt] * (dpre.abs() + err) + (dpre != 0) * 2.0 ** -25
    dx64, xb, dw64, wb = gradients64(dpre, err, x, w, off)
    close(dx, dx64, xb)
    close(dw, dw64, wb)
    wide = ops.grouped_gated_backward(dh, pre, x, w, off, activation=act, need_dx=False,
                                      grad_dtype=torch.float32)
    assert wide[0] is None
    close(wide[1], dw64, wb)


@pytest.mark.parametrize("with_bias,with_residual", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", None])
@pytest.mark.parametrize("counts,tail,inner,outer", LAYERS)
def test_linear(ops, counts, tail, inner, outer, act, dtype, with_bias, with_residual):
    dt = DTYPES[dtype]
    g, m, E, x, w, dy, off = layer(counts, tail, inner, outer, dt, 2)
    bias = torch.randn(E, outer, generator=g, device="cuda").to(dt) if with_bias else None
    res = torch.randn(m, outer, generator=g, device="cuda").to(dt) if with_residual else None
    p64, mag = grouped64(x, w, off)
    eps = 1.1 * inner * 2.0 ** -23 * mag
    if with_bias:
        for e, s in enumerate(ranges(off, E)):
            p64[s] += bias[e].double()
        eps += 2.0 ** -23 * p64.abs()
    a, _ = activation64(act, p64)
    r64 = res.double() if with_residual else torch.zeros_like(a)
    slack = 1.2 * eps + VALUE * a.abs() + 2.0 ** -22 * (a.abs() + r64.abs())
    y, pre = ops.grouped_linear(x, w, off, bias=bias, activation=act, residual=res, save=True)
    close(y, a + r64, slack)
    assert torch.equal(ops.grouped_linear(x, w, off, bias=bias, activation=act, residual=res), y)
    if act is None:
        assert pre is None
    else:
        assert pre.shape == (m, outer) and pre.dtype == dt
        close(pre, p64, eps)

    dx, dw, db = ops.grouped_linear_backward(dy, pre, x, w, off, activation=act)
    own = owned(off, E, m)
    d = torch.where(own, dy.double(), 0.0)
    if act is None:
        dpre, exact, err = d, torch.zeros_like(d), torch.zeros_like(d)
    else:
        dpre = d * activation64(act, pre.double())[1]
        exact = d.abs() * (SLOPE + 2.0 ** -22)
        err = exact + UNIT[dt] * (dpre.abs() + exact) + (dpre != 0) * 2.0 ** -25
    dx64, xb, dw64, wb = gradients64(dpre, err, x, w, off)
    close(dx, dx64, xb)
    close(dw, dw64, wb)
    wide = ops.grouped_linear_backward(dy, pre, x, w, off, activation=act, need_dx=False,
                                       grad_dtype=torch.float32)
    close(wide[1], dw64, wb)
    for e, s in enumerate(ranges(off, E)):
        n = max(1, counts[e])
        lim = exact[s].sum(0) + n * 2.0 ** -23 * (dpre[s].abs() + exact[s]).sum(0)
        close(db[e], dpre[s].sum(0), lim)
        close(wide[2][e], dpre[s].sum(0), lim)
    only = ops.grouped_linear_backward(dy, pre, x, w, off, activation=act, need_dx=False,
                                       need_dw=False)
    assert only[0] is None and only[1] is None and torch.equal(only[2], db)
    none = ops.grouped_linear_backward(dy, pre, x, w, off, activation=act, need_dbias=False)
    assert none[2] is None and torch.equal(none[0], dx) and torch.equal(none[1], dw)
