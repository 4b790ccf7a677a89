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
    err = torch.cat([(d * up).abs() * (SLOPE + 2.0 ** -22),
                     (d * a).abs() * (VALUE + 2.0 ** -22)], 1)
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


def small(seed, rows=90, inner=40, outer=24, experts=3, halves=1, dt=torch.bfloat16):
    g = gen(seed)
    counts = [rows // 2, 0, rows - rows // 2][:experts]
    x = torch.randn(rows, inner, generator=g, device="cuda").to(dt)
    w = (torch.randn(experts, halves * outer, inner, generator=g, device="cuda") *
         inner ** -0.5).to(dt)
    dy = torch.randn(rows, outer, generator=g, device="cuda").to(dt)
    return g, x, w, dy, offsets_of(counts)


SIZES = [(90, 40, 24), (60, 700, 129), (700, 264, 136), (3000, 72, 40), (10, 96, 1)]


@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_through_rows_is_the_gathered_call(ops, rows, inner, outer):
    """Rows read through an index, one of them outside, shared and in any order: the same bits as
    from gathered rows, forward and in the gradients."""
    g, x, w, dy, off = small(5, rows, inner, outer)
    _, _, w2, _, _ = small(6, rows, inner, outer, halves=2)
    index = torch.randint(0, rows, (rows,), generator=g, device="cuda", dtype=torch.int32)
    index[3] = -1
    index[5] = rows
    inside = (index >= 0) & (index < rows)
    xg = torch.where(inside[:, None], x[index.clamp(0, rows - 1).long()], 0)
    b = torch.randn(3, outer, generator=g, device="cuda").to(x.dtype)

    def both(x, rows):
        y, p = ops.grouped_linear(x, w, off, rows=rows, bias=b, activation="gelu", save=True)
        h, q = ops.grouped_gated(x, w2, off, rows=rows, save=True)
        return [y, p, h, q, *ops.grouped_linear_backward(dy, p, x, w, off, rows=rows,
                                                         activation="gelu"),
                *ops.grouped_gated_backward(dy, q, x, w2, off, rows=rows)]

    for got, want in zip(both(x, index), both(xg, None)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("shift", [0, 1, 2, 4, 8])
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_operands_at_any_address(ops, rows, inner, outer, shift):
    """x, w, bias, residual, dy and pre somewhere inside larger memory, with row pitches of their
    own and NaN around them: the same results as from memory of their own."""
    g, x, w, dy, off = small(8, rows, inner, outer)
    b = torch.randn(3, outer, generator=g, device="cuda").to(x.dtype)
    res = torch.randn(rows, outer, generator=g, device="cuda").to(x.dtype)

    def moved(t, pitch=None):
        pitch = pitch or t.shape[-1]
        n = t.numel() // t.shape[-1]
        buf = torch.full((n * pitch + 64,), math.nan, device="cuda", dtype=t.dtype)
        v = buf[shift:shift + n * pitch].view(n, pitch)[:, :t.shape[-1]]
        v = v if t.dim() == 2 else v.view(t.shape)
        return v.copy_(t)

    y, pre = ops.grouped_linear(x, w, off, bias=b, activation="silu", residual=res, save=True)
    xm, rm, dm = moved(x, inner + 3), moved(res, outer + 5), moved(dy, outer + 7)
    wm, bm = moved(w), moved(b)
    ym, pm = ops.grouped_linear(xm, wm, off, bias=bm, activation="silu", residual=rm, save=True)
    # an operand's place decides how it is read, and how a reduction is split, but not what it says
    _, mag = grouped64(x, w, off)
    close(ym, y.double(), 2.2 * inner * 2.0 ** -23 * mag + UNIT[x.dtype] * y.double().abs())
    close(pm, pre.double(), 2.2 * inner * 2.0 ** -23 * mag + UNIT[x.dtype] * pre.double().abs())
    want = ops.grouped_linear_backward(dy, pre, x, w, off, activation="silu")
    got = ops.grouped_linear_backward(dm, moved(pre), xm, wm, off, activation="silu")
    for a, e in zip(got, want):
        assert torch.equal(a, e)


def test_saved_values_in_other_layouts(ops):
    """pre as it came, without its padding, and transposed in memory."""
    for rows, inner, outer in SIZES:
        _, x, w, dy, off = small(9, rows, inner, outer, halves=2)
        _, pre = ops.grouped_gated(x, w, off, save=True)
        want = ops.grouped_gated_backward(dy, pre, x, w, off)
        for p in (pre.contiguous(), pre.clone(), pre.transpose(0, 2).contiguous().transpose(0, 2)):
            for a, b in zip(ops.grouped_gated_backward(dy, p, x, w, off), want):
                assert torch.equal(a, b)


def test_rows_before_the_first_offset(ops):
    """A shard's offsets do not start at 0; the rows before hold NaN."""
    for rows, inner, outer in SIZES:
        g, x, w, dy, off = small(10, rows, inner, outer)
        _, _, w2, _, _ = small(11, rows, inner, outer, halves=2)
        res = torch.randn(rows + 7, outer, generator=g, device="cuda").to(x.dtype)
        pad = lambda t: torch.cat([torch.full((7, t.shape[1]), math.nan, device="cuda",  # noqa
                                              dtype=t.dtype), t])
        xp, dp, op = pad(x), pad(dy), off + 7
        y, pre = ops.grouped_linear(xp, w, op, activation="gelu", residual=res, save=True)
        h, pre2 = ops.grouped_gated(xp, w2, op, save=True)
        assert torch.equal(y[:7], res[:7]) and not h[:7].any()
        assert not pre[:7].any() and not pre2[:7].any()
        dx, dw, db = ops.grouped_linear_backward(dp, pre, xp, w, op, activation="gelu")
        dx2, dw2 = ops.grouped_gated_backward(dp, pre2, xp, w2, op)
        assert not dx[:7].any() and not dx2[:7].any()
        for t in (dx, dw, db, dx2, dw2):
            assert torch.isfinite(t).all()


def test_bad_offsets_and_rows_stay_inside(ops):
    """Index data that are not what they should be: results mean nothing, the calls and the device
    stay usable."""
    _, x, w, dy, off = small(12, 3000, 64, 40)
    _, _, w2, _, _ = small(13, 3000, 64, 40, halves=2)
    y = ops.grouped_linear(x, w, off, bias=w[:, :, 0].contiguous(), activation="relu")
    rows = torch.randint(-5000, 5000, (3000,), device="cuda", dtype=torch.int32)
    big = (1 << 31) - 1
    for bad in ([0, 10, 5, 50], [-7, 20, 4000, big], [40, 30, 20, 10], [big] * 4, [-big] * 4,
                [0, 2900, 100, 3000], [3000, 0, 3000, 0]):
        for xs, dys, m in ((x, dy, 3000), (x[:50], dy[:50], 50)):
            o = torch.tensor(bad, dtype=torch.int32, device="cuda")
            for r in (None, rows[:m]):
                _, p = ops.grouped_linear(xs, w, o, rows=r, activation="silu", residual=dys,
                                          save=True)
                ops.grouped_linear_backward(dys, p, xs, w, o, rows=r, activation="silu")
                _, p = ops.grouped_gated(xs, w2, o, rows=r, save=True)
                ops.grouped_gated_backward(dys, p, xs, w2, o, rows=r)
    ops.check_errors()
    assert torch.equal(ops.grouped_linear(x, w, off, bias=w[:, :, 0].contiguous(),
                                          activation="relu"), y)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_activations_over_their_range(ops, act, dtype):
    """One input column and weights of 1: the activation itself, from the type's lowest value to its
    highest, with zeros, infinities and NaN, and its slope times a gradient of 1."""
    dt = DTYPES[dtype]
    top = math.log10(float(torch.finfo(dt).max))
    v = torch.logspace(-7, top - 1e-3, 4001, device="cuda", dtype=torch.float64)
    near = torch.linspace(-22, 22, 20_001, device="cuda", dtype=torch.float64)
    special = torch.tensor([0.0, math.inf, math.nan, torch.finfo(dt).max, torch.finfo(dt).min],
                           device="cuda", dtype=torch.float64)
    x = torch.cat([v, -v, near, special]).to(dt)[:, None].contiguous()
    m = x.shape[0]
    w = torch.ones(1, 1, 1, device="cuda", dtype=dt)
    off = offsets_of([m])
    y, pre = ops.grouped_linear(x, w, off, activation=act, save=True)
    assert torch.equal(pre.nan_to_num(7.0), x.nan_to_num(7.0))
    a, s = activation64(act, x.double())
    a = torch.where(x == 0, 0.0, a)
    usual = torch.isfinite(x)
    lim = VALUE * a.abs() + UNIT[dt] * a.abs() + 2.0 ** -25
    # beyond 22 a value is an argument's, or vanishes: exp's error grows with its argument, but
    # what it is a factor of is below 2^-25 (bf16: below its least normal number 2^-126 at 88)
    small_a = (x.double() < -22) & (a.abs() < 1e-6)
    assert ((y.double() - a).abs() <= torch.where(small_a, lim + a.abs(), lim))[usual].all()
    assert torch.isnan(y[torch.isnan(x)]).all()
    assert (y[x == math.inf] == math.inf).all()
    d = ops.grouped_linear_backward(torch.ones_like(x), pre, x, w, off, activation=act,
                                    need_dw=False, need_dbias=False)[0]
    lim = SLOPE + 2 * UNIT[dt] * (s.abs() + SLOPE) + 2.0 ** -24
    assert ((d.double() - s).abs() <= lim)[usual].all()


def test_neighbours_do_not_leak(ops):
    """An expert's infinities and NaN, in rows, weights and bias, stay in its own results."""
    for counts, inner, outer in (([37, 50, 41], 96, 72), ([200, 77, 300], 264, 272),
                                 ([3, 2, 4], 40, 24)):
        g = gen(14)
        m = sum(counts)
        bf = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa
        x, w, w2 = bf(m, inner), bf(3, outer, inner), bf(3, 2 * outer, inner)
        b, dy = bf(3, outer), bf(m, outer)
        off = offsets_of(counts)
        s = slice(counts[0], counts[0] + counts[1])

        def calls():
            y, p = ops.grouped_linear(x, w, off, bias=b, activation="silu", save=True)
            h, q = ops.grouped_gated(x, w2, off, save=True)
            return [y, h, *ops.grouped_linear_backward(dy, p, x, w, off, activation="silu"),
                    *ops.grouped_gated_backward(dy, q, x, w2, off)]

        clean = calls()
        x[s.start], x[s.stop - 1], dy[s.start + 1] = math.nan, math.inf, math.nan
        w[1, 0], w2[1, 1], b[1, 2] = math.inf, math.nan, -math.inf
        for got, want in zip(calls(), clean):
            keep = torch.ones(got.shape[0], dtype=torch.bool, device="cuda")
            keep[1 if got.shape[0] == 3 else s] = False
            assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("kind", ["gated", "linear"])
def test_gradients_by_differences(ops, kind):
    """Directional differences of <dy, layer> in f64, whose error is h^2 / 6 of a third derivative
    (below 1e-4 of the slope at h = 1e-3), against the gradients; these hold at most three
    roundings to 16 bits a factor (pre, dpre, the result): 3 * 2^-11 of the terms' 2-norms in
    f16."""
    halves = 2 if kind == "gated" else 1
    g, x, w, dy, off = small(15, 90, 40, 24, halves=halves, dt=torch.float16)
    b = torch.randn(3, 24, generator=g, device="cuda").to(torch.float16)
    F = torch.nn.functional

    def value(x, w, b):
        out = []
        for e, s in enumerate(ranges(off, 3)):
            p = x[s] @ w[e].T
            out.append(F.silu(p[:, :24]) * p[:, 24:] if kind == "gated" else F.gelu(p + b[e]))
        return (torch.cat(out) * dy.double()).sum()

    if kind == "gated":
        _, pre = ops.grouped_gated(x, w, off, save=True)
        grads = ops.grouped_gated_backward(dy, pre, x, w, off, grad_dtype=torch.float32)
    else:
        _, pre = ops.grouped_linear(x, w, off, bias=b, activation="gelu", save=True)
        grads = ops.grouped_linear_backward(dy, pre, x, w, off, activation="gelu",
                                            grad_dtype=torch.float32)
    at = [x.double(), w.double(), b.double()]
    for i, grad in enumerate(grads):
        d = torch.randn(at[i].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-3
        moved = lambda s: value(*[t + s * h * d if j == i else t for j, t in enumerate(at)])  # noqa
        slope = (moved(1) - moved(-1)) / (2 * h)
        bound = 3 * 2.0 ** -11 * float(grad.double().norm() * d.norm()) + 1e-4 * abs(float(slope))
        assert abs(float((grad.double() * d).sum() - slope)) <= bound


def block(ops, x, w1, w2, b2, logits, dout, base, most):
    """A layer as it is trained: route, gated experts, projection with bias, combination; all
    gradients, clipped together."""
    r = ops.route(logits, 2)
    h, pre = ops.grouped_gated(x, w1, r.offsets, rows=r.rows, save=True)
    y = ops.grouped_linear(h, w2, r.offsets, bias=b2, residual=base)
    out = ops.combine(y, r.position, r.weights)
    dy, dwt = ops.combine_backward(dout, y, r.position, r.weights)
    dh, dw2, db2 = ops.grouped_linear_backward(dy, None, h, w2, r.offsets,
                                               grad_dtype=torch.float32)
    dxs, dw1 = ops.grouped_gated_backward(dh, pre, x, w1, r.offsets, rows=r.rows,
                                          grad_dtype=torch.float32)
    grads = [ops.combine(dxs, r.position), dw1, dw2, db2, ops.route_backward(dwt, logits, r)]
    norm = ops.clip_grads(grads, most)
    return [out, norm, dy, *grads]


def block_inputs(seed, T=150, E=6, K=24, H=40, N=16):
    g = gen(seed)
    bf = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa
    return [bf(T, K), bf(E, 2 * H, K) * 0.2, bf(E, N, H) * 0.2, bf(E, N),
            torch.randn(T, E, generator=g, device="cuda"), bf(T, N), bf(2 * T, N)]


@pytest.mark.parametrize("sizes", [(150, 6, 24, 40, 16), (3000, 8, 72, 129, 40),
                                   (7, 9, 130, 33, 20)])
def test_block_against_autograd(ops, sizes):
    """The operators together, tokens shared by two experts each, against torch's autograd in f64
    on the same bf16 weights. On the way to a gradient at most seven results are rounded to bf16
    (h, y, dy, dh, pre, dpre, dx), each by 2^-8 of itself at most: 7 * 2^-8 in the 2-norm. The norm
    is theirs, and the clipped gradients have the wanted one."""
    x, w1, w2, b2, logits, dout, base = block_inputs(44, *sizes)
    E = w1.shape[0]
    out, norm, _, *grads = block(ops, x, w1, w2, b2, logits, dout, base, 1.0)
    r = ops.route(logits, 2)
    p = [t.double().requires_grad_() for t in (x, w1, w2, b2, logits)]
    e = r.experts.long()
    wt = p[4].gather(1, e).softmax(1)
    ref = 0
    H = w2.shape[2]
    for j in range(2):
        both = torch.zeros(x.shape[0], 2 * H, device="cuda", dtype=torch.float64)
        y = base[r.position[:, j].long()].double()
        parts = []
        for k in range(E):
            at = (e[:, j] == k).nonzero()[:, 0]
            q = p[0][at] @ p[1][k].T
            h = torch.nn.functional.silu(q[:, :H]) * q[:, H:]
            parts.append((at, h @ p[2][k].T + p[3][k]))
        order = torch.cat([a for a, _ in parts])
        y = y + torch.cat([v for _, v in parts])[order.argsort()]
        ref = ref + wt[:, j:j + 1] * y
    want = torch.autograd.grad(ref, p, dout.double())
    total = math.sqrt(sum(float(g.square().sum()) for g in want))
    ref = ref.detach()
    assert float((out.double() - ref).norm() / ref.norm()) < 7 * 2.0 ** -8
    assert abs(float(norm) / total - 1) < 7 * 2.0 ** -8
    for a, b in zip(grads, want):
        assert float((a.double() * float(norm) - b).norm() / b.norm()) < 7.5 * 2.0 ** -8
    clipped = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert abs(clipped - 1.0) < 2.0 ** -8


def test_block_in_a_graph(ops):
    """Captured once, replayed on other inputs, other routing among them; two graphs of one step."""
    inputs = block_inputs(45)
    block(ops, *inputs, 1.0)
    graphs, outs = [], []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(block(ops, *inputs, 1.0))
    for seed in (46, 47):
        for t, v in zip(inputs, block_inputs(seed)):
            t.copy_(v)
        want = block(ops, *inputs, 1.0)
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_same_bits_on_streams_and_threads(ops):
    """The same step twice, on another stream, and from threads that run at the same time."""
    import threading

    inputs = block_inputs(48, 4000, 12, 136, 200, 72)
    first = block(ops, *inputs, 1.0)
    torch.cuda.synchronize()
    results, errors = {}, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream), torch.no_grad():
                for _ in range(5):
                    results[i] = block(ops, *inputs, 1.0)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for r in results.values():
        assert all(torch.equal(a, b) for a, b in zip(r, first))


def test_no_rows_and_single_columns(ops):
    e = lambda *s: torch.empty(*s, device="cuda", dtype=torch.float16)  # noqa: E731
    w = torch.ones(2, 24, 32, device="cuda", dtype=torch.float16)
    off = offsets_of([0, 0])
    y, pre = ops.grouped_linear(e(0, 32), w, off, activation="relu", save=True)
    assert y.shape == pre.shape == (0, 24)
    dx, dw, db = ops.grouped_linear_backward(e(0, 24), pre, e(0, 32), w, off, activation="relu")
    assert dx.shape == (0, 32) and not dw.any() and not db.any()
    h, pre = ops.grouped_gated(e(0, 32), w, off, save=True)
    assert h.shape == (0, 12) and pre.shape == (0, 2, 12)
    dx, dw = ops.grouped_gated_backward(e(0, 12), pre, e(0, 32), w, off)
    assert dx.shape == (0, 32) and not dw.any()
    x = torch.tensor([[2.0], [-3.0]], device="cuda", dtype=torch.float16)
    w = torch.tensor([[[1.5], [4.0]]], device="cuda", dtype=torch.float16)
    h, pre = ops.grouped_gated(x, w, offsets_of([2]), activation="relu", save=True)
    assert h.tolist() == [[24.0], [0.0]] and pre.tolist() == [[[3.0], [8.0]], [[-4.5], [-12.0]]]
    dx, dw = ops.grouped_gated_backward(torch.ones_like(h), pre, x, w, offsets_of([2]),
                                        activation="relu")
    assert dx.tolist() == [[24.0], [0.0]] and dw.tolist() == [[[16.0], [6.0]]]


def test_offsets_pass_32_bits(ops):
    """Results, saved values, residual and gradients of more than 2^32 elements: the last rows, and
    a bias's gradient over all of them."""
    g = gen(49)
    m, n = 70_000, 64_000  # 4.48e9
    x = torch.zeros(m, 16, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, 16, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(1, n, 16, generator=g, device="cuda").to(torch.bfloat16)
    off = offsets_of([m])
    dy = torch.zeros(m, n, device="cuda", dtype=torch.bfloat16)
    dy[-3:] = torch.randn(3, n, generator=g, device="cuda").to(torch.bfloat16)
    y, pre = ops.grouped_linear(x, w, off, activation="relu", residual=dy, save=True)
    p64 = x[-3:].double() @ w[0].double().T
    eps = 1.1 * 16 * 2.0 ** -23 * (x[-3:].double().abs() @ w[0].double().abs().T)
    close(pre[-3:], p64, eps)
    close(y[-3:], p64.clamp(min=0) + dy[-3:].double(), eps + 2.0 ** -22 * (p64.abs() + 5))
    assert not y[-70:-3].any() and not y[:70].any()
    del y
    dx, _, db = ops.grouped_linear_backward(dy, pre, x, w, off, activation="relu", need_dw=False)
    d = dy[-3:].double() * (pre[-3:] > 0)
    close(db[0], d.sum(0), 8 * 2.0 ** -23 * d.abs().sum(0))
    # n terms, the sums of long reductions kept in runs
    close(dx[-3:], d @ w[0].double(), 1.1 * 4200 * 2.0 ** -23 * (d.abs() @ w[0].double().abs()))
    assert not dx[:-3].any()
    del pre, dy, dx
    w = torch.randn(1, n, 16, generator=g, device="cuda").to(torch.bfloat16)
    m2 = 2 * m
    x = torch.zeros(m2, 16, device="cuda", dtype=torch.bfloat16)
    x[-2:] = torch.randn(2, 16, generator=g, device="cuda").to(torch.bfloat16)
    h, pre = ops.grouped_gated(x, w, offsets_of([m2]), save=True)  # pre 8.96e9, h 4.48e9
    p64 = x[-2:].double() @ w[0].double().T
    eps = 1.1 * 16 * 2.0 ** -23 * (x[-2:].double().abs() @ w[0].double().abs().T)
    close(pre[-2:].flatten(1), p64, eps)
    a, up = activation64("silu", p64[:, :n // 2])[0], p64[:, n // 2:]
    close(h[-2:], a * up, 1.2 * eps[:, :n // 2] * (up.abs() + eps[:, n // 2:]) +
          a.abs() * eps[:, n // 2:] + (VALUE + 2.0 ** -22) * (a * up).abs())


def refusals():
    bf, f16, i32 = torch.bfloat16, torch.float16, torch.int32
    c = lambda *s, dtype=bf: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa
    off = lambda n: c(n, dtype=i32)  # noqa
    x, w, wg, y = c(4, 8), c(2, 6, 8), c(2, 12, 8), c(4, 6)
    lin = lambda o, **k: o.grouped_linear(**{"x": x, "w": w, "offsets": off(3), **k})  # noqa
    gat = lambda o, **k: o.grouped_gated(**{"x": x, "w": wg, "offsets": off(3), **k})  # noqa
    lb = lambda o, **k: o.grouped_linear_backward(**{  # noqa
        "dy": y, "pre": y, "x": x, "w": w, "offsets": off(3), "activation": "relu", **k})
    gb = lambda o, **k: o.grouped_gated_backward(**{  # noqa
        "dh": y, "pre": c(4, 2, 6), "x": x, "w": wg, "offsets": off(3), **k})
    grad = c(4, 8).requires_grad_()
    return [
        lambda o: lin(o, activation="tanh"),
        lambda o: lin(o, activation=2),
        lambda o: lin(o, bias=c(2, 7)),
        lambda o: lin(o, bias=c(6)),
        lambda o: lin(o, bias=c(2, 6, dtype=torch.float32)),
        lambda o: lin(o, residual=c(4, 7)),
        lambda o: lin(o, residual=c(5, 6)),
        lambda o: lin(o, residual=c(4, 6, dtype=f16)),
        lambda o: lin(o, residual=c(4, 6).cpu()),
        lambda o: lin(o, x=c(4, 8, dtype=torch.float32)),
        lambda o: lin(o, x=c(4, 7)),
        lambda o: lin(o, w=c(2, 6, 8, dtype=f16)),
        lambda o: lin(o, offsets=off(4)),
        lambda o: lin(o, offsets=off(3).long()),
        lambda o: lin(o, rows=off(4).long()),
        lambda o: lin(o, w=c(600, 6, 8), offsets=off(601)),
        lambda o: lin(o, x=grad),
        lambda o: gat(o, w=c(2, 7, 8)),
        lambda o: gat(o, activation="swish"),
        lambda o: gat(o, x=c(4, 9)),
        lambda o: lb(o, dy=c(4, 7)),
        lambda o: lb(o, dy=c(5, 6)),
        lambda o: lb(o, dy=c(4, 6, dtype=f16)),
        lambda o: lb(o, pre=None),
        lambda o: lb(o, pre=c(4, 7)),
        lambda o: lb(o, pre=c(4, 6, dtype=f16)),
        lambda o: lb(o, activation=None),
        lambda o: lb(o, grad_dtype=f16),
        lambda o: gb(o, pre=c(4, 6)),
        lambda o: gb(o, pre=c(4, 2, 7)),
        lambda o: gb(o, dh=c(4, 12)),
        lambda o: gb(o, w=c(2, 13, 8)),
        lambda o: gb(o, grad_dtype=torch.float64),
    ]


@pytest.mark.parametrize("i", range(33))
def test_refusals(ops, i):
    from lightgbm_rs_b200 import LightGBMError

    calls = refusals()
    assert len(calls) == 33
    with pytest.raises(LightGBMError):
        calls[i](ops)
