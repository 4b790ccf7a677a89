"""Gated and linear expert layers where values leave f16's range or come near to nothing.

Bounds as in test_gpu_expert_layers.py."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_experts import DTYPES, UNIT, close, gen, offsets_of  # noqa: E402
from test_gpu_expert_layers import (SLOPE, VALUE, activation64, gradients64,  # noqa: E402
                                    grouped64, ranges)


@pytest.fixture(scope="module")
def ops():
    from lightgbm_rs_b200 import experts

    yield experts
    experts.check_errors()


COUNTS = [[2, 0, 3], [150, 90], [1000, 24]]  # streamed, tiles of 64 columns, of 128 and more


def overflowing(counts, inner, outer, halves, signs, seed):
    """f16 inputs whose products are +-84000 in every fourth column `signs` ({column: sign}), in
    every third row, and ordinary elsewhere."""
    g = gen(seed)
    m, E = sum(counts), len(counts)
    x = torch.randn(m, inner, generator=g, device="cuda")
    w = torch.randn(E, halves * outer, inner, generator=g, device="cuda") * inner ** -0.5
    x[:, 0] = 0
    x[::3, 0] = 300
    w[:, :, 0] = 0
    for column, sign in signs.items():
        w[:, column:outer:4, 0] = 280 * sign
    dy = torch.randn(m, outer, generator=g, device="cuda")
    big = torch.zeros(m, dtype=torch.bool, device="cuda")
    big[::3] = True
    return x.half(), w.half(), dy.half(), offsets_of(counts), big


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("outer", [24, 140])
@pytest.mark.parametrize("counts", COUNTS)
def test_linear_beyond_the_saved_type(ops, counts, outer, act):
    """A product of +-84000 is saved as an infinity of f16: the activation's slope there is 1 or 0,
    and all gradients are those of 64 bits."""
    x, w, dy, off, big = overflowing(counts, 40, outer, 1, {0: 1, 1: -1}, 61)
    p64, mag = grouped64(x, w, off)
    y, pre = ops.grouped_linear(x, w, off, activation=act, save=True)
    infinite = torch.isinf(pre)
    assert torch.equal(infinite, p64.abs() > 65504) and infinite.any()
    assert (pre[infinite].double().sign() == p64[infinite].sign()).all()
    a, _ = activation64(act, p64)
    close(y, a, 1.3 * 40 * 2.0 ** -23 * mag + (VALUE + 2.0 ** -22) * a.abs())
    assert (y[infinite & (p64 > 0)] == math.inf).all() and not y[infinite & (p64 < 0)].any()
    v = torch.where(infinite, p64, pre.double())
    d = dy.double()
    dpre = d * activation64(act, v)[1]
    exact = d.abs() * (SLOPE + 2.0 ** -22)
    err = exact + UNIT[x.dtype] * (dpre.abs() + exact) + (dpre != 0) * 2.0 ** -25
    dx64, xb, dw64, wb = gradients64(dpre, err, x, w, off)
    dx, dw, db = ops.grouped_linear_backward(dy, pre, x, w, off, activation=act)
    close(dx, dx64, xb)
    close(dw, dw64, wb)
    for e, s in enumerate(ranges(off, len(counts))):
        n = max(1, counts[e])
        close(db[e], dpre[s].sum(0),
              exact[s].sum(0) + n * 2.0 ** -23 * (dpre[s].abs() + exact[s]).sum(0))
        # (close compares NaN's places; nothing here is infinite)
        assert torch.isfinite(dx[s]).all() and torch.isfinite(dw[e]).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("outer", [24, 140])
@pytest.mark.parametrize("counts", COUNTS)
def test_gated_far_below_zero(ops, counts, outer, act):
    """A gate of -84000 is saved as -infinity: h is 0 there, and nothing passes it backwards."""
    x, w, dh, off, big = overflowing(counts, 40, outer, 2, {1: -1}, 62)
    p64, mag = grouped64(x, w, off)
    eps = 1.1 * 40 * 2.0 ** -23 * mag
    h, pre = ops.grouped_gated(x, w, off, activation=act, save=True)
    gate, up = p64[:, :outer], p64[:, outer:]
    infinite = torch.isinf(pre[:, 0])
    assert torch.equal(infinite, gate < -65504) and infinite.any()
    a, _ = activation64(act, gate)
    close(h, a * up, 1.2 * eps[:, :outer] * (up.abs() + eps[:, outer:]) * ~infinite +
          a.abs() * eps[:, outer:] + (VALUE + 2.0 ** -22) * (a * up).abs())
    assert not h[infinite].any()
    gate, up = torch.where(infinite, gate, pre[:, 0].double()), pre[:, 1].double()
    a, s = activation64(act, gate)
    d = dh.double()
    dpre = torch.cat([d * up * s, d * a], 1)
    err = torch.cat([(d * up).abs() * (SLOPE + 2.0 ** -22), (d * a).abs() * (VALUE + 2.0 ** -22)],
                    1)
    err += UNIT[x.dtype] * (dpre.abs() + err) + (dpre != 0) * 2.0 ** -25
    dx64, xb, dw64, wb = gradients64(dpre, err, x, w, off)
    dx, dw = ops.grouped_gated_backward(dh, pre, x, w, off, activation=act)
    close(dx, dx64, xb)
    close(dw, dw64, wb)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("counts", COUNTS)
def test_gated_far_above_zero(ops, counts, act):
    """A gate of 84000 is saved as infinity: its own gradient is that of 64 bits, and what act(gate)
    is a factor of, up's, is infinite. Rows and weights that this does not enter keep theirs."""
    outer = 24
    x, w, dh, off, big = overflowing(counts, 40, outer, 2, {0: 1}, 63)
    dh[dh == 0] = 1
    p64, _ = grouped64(x, w, off)
    _, pre = ops.grouped_gated(x, w, off, activation=act, save=True)
    infinite = torch.isinf(pre[:, 0])
    assert torch.equal(infinite, p64[:, :outer] > 65504) and infinite.any()
    gate = torch.where(infinite, p64[:, :outer], pre[:, 0].double())
    up = pre[:, 1].double()
    a, s = activation64(act, gate)
    d = dh.double()
    dpre = torch.cat([d * up * s, torch.where(infinite, 0.0, d * a)], 1)
    err = torch.cat([(d * up).abs() * (SLOPE + 2.0 ** -22),
                     torch.where(infinite, 0.0, d * a).abs() * (VALUE + 2.0 ** -22)], 1)
    err += UNIT[x.dtype] * (dpre.abs() + err) + (dpre != 0) * 2.0 ** -25
    dx64, xb, dw64, wb = gradients64(dpre, err, x, w, off)
    dx, dw = ops.grouped_gated_backward(dh, pre, x, w, off, activation=act)
    assert not torch.isfinite(dx[big]).any()
    close(dx[~big], dx64[~big], xb[~big])
    for e, rows in enumerate(ranges(off, len(counts))):
        enters = torch.zeros(2 * outer, dtype=torch.bool, device="cuda")
        enters[outer:] = infinite[rows].any(0)
        close(dw[e][~enters], dw64[e][~enters], wb[e][~enters])
        assert not torch.isfinite(dw[e][enters][:, 0]).any()


@pytest.mark.parametrize("wide", [False, True])
def test_gradients_at_the_range_of_f16(ops, wide):
    """dh up act'(gate) of 60000 is exact, of 72000 an infinity, in f32 weight gradients too: in
    its own row of dx and of dw and nowhere else."""
    H, K = 8, 16
    x = torch.eye(2, K, device="cuda").half()
    w = torch.zeros(1, 2 * H, K, device="cuda").half()
    w[0, :H, :2] = 2.0 ** -6                      # gate, slope 1
    w[0, H:, 0], w[0, H:, 1] = 100.0, 120.0       # up
    off = offsets_of([2])
    _, pre = ops.grouped_gated(x, w, off, activation="relu", save=True)
    dh = torch.zeros(2, H, device="cuda").half()
    dh[0, 0], dh[1, 0], dh[1, 1] = 600.0, 600.0, 1.0
    dx, dw = ops.grouped_gated_backward(dh, pre, x, w, off, activation="relu",
                                        grad_dtype=torch.float32 if wide else None)
    want = torch.tensor([60000.0 + 600.0 * 100.0, 60000.0 + 600.0 * 120.0], device="cuda") / 64
    assert torch.equal(dx[0, :2], want.half()) and not dx[0, 2:].any()
    assert not torch.isfinite(dx[1]).any()
    assert not torch.isfinite(dw[0, 0]).any()
    rest = dw[0, 1:].double()
    exact = torch.zeros_like(rest)
    exact[0, 1] = 120.0                           # dh up of the second hidden column
    exact[H - 1, :2] = 600.0 * 2.0 ** -6          # dh act(gate)
    exact[H, 1] = 2.0 ** -6
    assert torch.equal(rest, exact)


U = 2.0 ** -23


def relative(act, v):
    """How far values and slopes (below -2) may be off, relative to themselves, before they are
    rounded to 16 bits. e^v by one instruction (2 units of U) on an argument rounded twice (0.62 |v|).
    silu: a sum (0.5), a reciprocal (1) and a product (0.5) follow; above 0 the exp's part of 1 + e^-v
    falls faster than its error grows. gelu: a tail fitted to 5.4e-6, e^(-v^2 / 2) with two more
    roundings of its argument (0.5 v^2 / 2), and seven operations of the polynomial.
    Slopes: s (1 + v (1 - s)) adds at most 4.5 units below -2; v phi(v) + P(v) is, there, a
    difference of terms whose sum is 1.53 times as large."""
    if act == "silu":
        a = torch.where(v < 0, 4 + 0.62 * v.abs(), 5.0) * U
        return a, a + 4.5 * U
    a = torch.where(v < 0, 5.4e-6 + (9 + 0.56 * v * v) * U, 1.2e-5)
    return a, 1.53 * (5.4e-6 + (10 + 0.56 * v * v) * U)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("streamed", [False, True])
def test_small_values_keep_their_digits(ops, act, dtype, streamed):
    """The activation itself (one input column, weights of 1), relative to its own size down to
    where e^v leaves f32's normal numbers: silu to -87, gelu to -13; below that nearly nothing."""
    dt = DTYPES[dtype]
    end = -87.0 if act == "silu" else -13.1
    x = torch.cat([torch.linspace(end, 0, 6001), torch.linspace(0, 12, 500),
                   -torch.logspace(-6, 2, 1600)]).to("cuda").to(dt)[:, None].contiguous()
    m, E = x.shape[0], 512 if streamed else 1
    off = offsets_of([m // E + (e < m % E) for e in range(E)])
    w = torch.ones(E, 1, 1, device="cuda", dtype=dt)
    y, pre = ops.grouped_linear(x, w, off, activation=act, save=True)
    v = x.double()
    a, s = activation64(act, v)
    rel, slope = relative(act, v)
    least = 2.0 ** -25 if dt is torch.float16 else 2.0 ** -134
    usual = v >= end
    lim = a.abs() * (UNIT[dt] + 1.01 * rel) + least
    assert ((y.double() - a).abs() <= lim)[usual].all()
    assert (y.double().abs() <= 1.1e-36 + least)[~usual].all() and (~usual).any()
    d = ops.grouped_linear_backward(torch.ones_like(x), pre, x, w, off, activation=act,
                                    need_dw=False, need_dbias=False)[0]
    lim = s.abs() * (UNIT[dt] + 1.01 * slope) + least
    assert ((d.double() - s).abs() <= lim)[usual & (v < -2)].all()
    assert (d.double().abs() <= 1.1e-36 + least)[~usual].all()
    assert bool(y[(v > -5) & (v < -4.9)].any()) and bool(d[(v > -5) & (v < -4.9)].any())
