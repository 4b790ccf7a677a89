"""Expert-layer operators on the GPU against plain implementations in 64 bits.

Tolerances are bounds, not fits. A sum of n products in f32 is off by at most n * 2^-23 times
the sum of the products' magnitudes (each of n additions rounds or truncates once: 2^-23
relative), plus one rounding to the result's type: 2^-8 of a bf16, 2^-11 of an f16, 2^-24 of an
f32 (and half the least subnormal of f16, 2^-25). exp in f32 is good to 2 units in the last
place and its argument to half of one.
"""

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(scope="module")
def ops():
    from lightgbm_rs_b200 import experts

    yield experts
    experts.check_errors()


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def close(got, want, slack, dtype=None):
    """|got - want| <= slack + one rounding to got's type; NaN and infinities in the same
    places."""
    u = UNIT[dtype or got.dtype]
    g = got.double()
    fin = torch.isfinite(want) & (want.abs() <= torch.finfo(got.dtype).max)
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    lim = slack + u * want.abs() + 2.0 ** -25
    bad = ((g - want).abs() > lim) & fin
    assert not bad.any(), (int(bad.sum()), float((g - want).abs()[fin].max()))


# ----------------------------------------------------------------------------- route


def route64(logits, k, normalize):
    """Definition of the router in numpy f64: weights, experts, position, rows, offsets."""
    l = logits.double().cpu().numpy()
    T, E = l.shape
    # descending, NaN before everything, the lower expert first among equals
    key = -np.where(np.isnan(l), np.inf, np.where(l == np.inf, 1e300, l))
    ids = np.argsort(key, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(l, ids, 1)
    empty = top == -np.inf
    with np.errstate(invalid="ignore"):
        m = np.where(empty[:, :1], 0.0, top[:, :1])
        ex = np.exp(top - m)
        z = (ex if normalize else np.exp(l - m)).sum(1, keepdims=True)
        w = np.where(empty, 0.0, ex / z)
    ids = np.where(empty, -1, ids)
    flat = ids.reshape(-1)
    key = np.where(flat < 0, E, flat)
    order = np.argsort(key, kind="stable")
    position = np.empty(T * k, dtype=np.int64)
    position[order] = np.arange(T * k)
    offsets = np.searchsorted(key[order], np.arange(E + 1))
    return w, ids, position.reshape(T, k), order // k, offsets


ROUTE = [  # tokens, experts, k
    (1, 1, 1), (1, 8, 2), (3, 5, 5), (64, 255, 4), (65, 255, 4), (16, 512, 16), (200, 2, 1),
    (1000, 63, 3), (4097, 31, 8), (16384, 64, 2), (16500, 65, 6), (300, 512, 16), (17000, 100, 16),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("tokens,experts,k", ROUTE)
def test_route(ops, tokens, experts, k, normalize, dtype):
    g = gen(tokens + experts)
    dt = DTYPES[dtype]
    # multiples of 1/8 in a small range: many ties
    x = (torch.randn(tokens, experts, generator=g, device="cuda") * 16).round() / 8
    x = x.to(dt)
    u = torch.rand(tokens, experts, generator=g, device="cuda")
    x.masked_fill_(u < 0.1, torch.finfo(dt).min)
    x.masked_fill_(u > 0.7, -math.inf)
    if tokens > 2:
        x[1] = -math.inf               # nothing left
        x[2] = torch.finfo(dt).min     # everything at the type's lowest value
        x[0, 0], x[0, -1] = -0.0, 0.0  # one value
    w, ids, pos, rows, off = route64(x, k, normalize)
    r = ops.route(x, k, normalize=normalize)
    assert np.array_equal(r.experts.cpu().numpy(), ids)
    assert np.array_equal(r.position.cpu().numpy(), pos)
    assert np.array_equal(r.rows.cpu().numpy(), rows)
    assert np.array_equal(r.offsets.cpu().numpy(), off)
    # exp: 2.5 ulp of 2^-24 relative each side of the quotient, the arguments (up to 16 here,
    # rounded at 2^-21) and a sum of up to 512 terms; all relative to the weight
    close(r.weights, torch.from_numpy(w).cuda(), torch.from_numpy(w).cuda() * (512 + 32) * 2 ** -24)

    dw = torch.randn(tokens, k, generator=g, device="cuda")
    d = ops.route_backward(dw, x, r, normalize=normalize)
    l, dwn = x.double().cpu().numpy(), dw.double().cpu().numpy()
    at, taken = np.maximum(ids, 0), (ids >= 0).astype(np.float64)
    chosen, gr = np.zeros((tokens, experts)), np.zeros((tokens, experts))
    np.add.at(chosen, (np.arange(tokens)[:, None], at), taken)
    np.add.at(gr, (np.arange(tokens)[:, None], at), taken * dwn)
    top = np.where(ids[:, :1] >= 0, np.take_along_axis(l, at[:, :1], 1), 0.0)
    p = np.exp(l - top) * (chosen if normalize else 1.0)
    p = np.where(ids[:, :1] >= 0, p / np.maximum(p.sum(1, keepdims=True), 1e-300), 0.0)
    want = p * (gr - (p * gr).sum(1, keepdims=True))
    scale = p * (np.abs(gr) + (p * np.abs(gr)).sum(1, keepdims=True))
    close(d, torch.from_numpy(want).cuda(), torch.from_numpy(scale).cuda() * 1024 * 2 ** -24)


@pytest.mark.parametrize("tokens", [66, 109, 2047, 2049, 4096, 9001, 33000])
def test_route_blocks(ops, tokens):
    """Numbers of tokens at which a block takes another share of them."""
    test_route(ops, tokens, 37, 3, False, "f32")


def test_route_nan_and_infinity(ops):
    x = torch.zeros(4, 6, device="cuda")
    x[0, 3] = math.nan
    x[1, 2] = math.inf
    x[2] = torch.tensor([1.0, math.nan, 2.0, math.nan, -math.inf, 3.0])
    r = ops.route(x, 2)
    assert r.experts.tolist() == [[3, 0], [2, 0], [1, 3], [0, 1]]
    assert torch.isnan(r.weights[:3]).all()
    assert r.weights[3].tolist() == [0.5, 0.5]


@pytest.mark.parametrize("normalize", [True, False])
def test_route_gradient_by_differences(ops, normalize):
    """Central differences with h = 2^-6: error h^2 / 6 times a third derivative of the
    softmax (below 1) times |dw| plus weights' rounding 2^-22 |dw| / h, per term of k."""
    g = gen(5)
    x = torch.randn(7, 9, generator=g, device="cuda")
    dw = torch.randn(7, 3, generator=g, device="cuda")
    h = 2.0 ** -6
    # distinct logits, so that a step of h does not change the choice
    x = x.argsort(1).argsort(1).float() * 0.25
    d = ops.route_backward(dw, x, ops.route(x, 3, normalize=normalize), normalize=normalize)
    for e in range(9):
        step = torch.zeros(9, device="cuda")
        step[e] = h
        up, down = (ops.route(x + s, 3, normalize=normalize).weights for s in (step, -step))
        diff = ((up - down).double() * dw.double()).sum(1) / (2 * h)
        lim = dw.double().abs().sum(1) * (h * h / 6 + 2.0 ** -22 / h)
        assert ((diff - d[:, e].double()).abs() <= lim).all()


def test_route_strided_logits(ops):
    g = gen(1)
    big = torch.randn(500, 40, generator=g, device="cuda")
    for view in (big[:, 3:20], big[::2, 1:18], big.t()[:17, :300].t()):
        a, b = ops.route(view, 3), ops.route(view.contiguous(), 3)
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_route_no_tokens(ops):
    r = ops.route(torch.empty(0, 5, device="cuda"), 2)
    assert r.weights.shape == (0, 2) and r.rows.numel() == 0
    assert r.offsets.tolist() == [0] * 6


# --------------------------------------------------------------------------- products


def offsets_of(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32,
                        device="cuda")


def product64(x, w, off, rows):
    x, off = x.double(), off.tolist()
    if rows is not None:
        r = rows.long()
        inside = (r >= 0) & (r < x.shape[0])
        x = torch.where(inside[:, None], x[r.clamp(0, max(0, x.shape[0] - 1))],
                        torch.zeros((), dtype=torch.float64, device="cuda"))
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(y)
    for e in range(w.shape[0]):
        s = slice(off[e], off[e + 1])
        y[s] = x[s] @ w[e].double().T
        mag[s] = x[s].abs() @ w[e].double().abs().T
    return x, y, mag


PRODUCT = [  # counts, tail rows, inner, outer
    ([1], 0, 1, 1),
    ([1, 0, 1], 2, 64, 64),
    ([5], 0, 16, 8),
    ([0, 0], 3, 40, 24),
    ([63, 64, 65, 1], 0, 128, 256),
    ([127, 0, 129, 300], 7, 200, 264),
    ([2000], 0, 72, 520),
    ([17] * 40, 5, 700, 129),
    ([0, 3, 0, 0, 200, 1, 0], 1, 257, 33),
    ([31, 1100, 2], 0, 1000, 700),
    ([8] * 512, 0, 48, 40),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("counts,tail,inner,outer", PRODUCT)
def test_products(ops, counts, tail, inner, outer, dtype):
    dt = DTYPES[dtype]
    g = gen(inner * 7 + outer)
    m, E = sum(counts) + tail, len(counts)
    x = torch.randn(m, inner, generator=g, device="cuda").to(dt)
    w = (torch.randn(E, outer, inner, generator=g, device="cuda") * inner ** -0.5).to(dt)
    dy = torch.randn(m, outer, generator=g, device="cuda").to(dt)
    off = offsets_of(counts)
    if tail:  # rows of no expert hold what they like
        x[-1], dy[-1] = math.nan, math.inf
    _, y64, mag = product64(x, w, off, None)
    y = ops.grouped_matmul(x, w, off)
    close(y, y64, inner * 2.0 ** -23 * mag)
    dx, dw = ops.grouped_matmul_backward(dy, x, w, off)
    _, dx64, mag = product64(dy, w.transpose(1, 2), off, None)
    close(dx, dx64, outer * 2.0 ** -23 * mag)
    dwf = ops.grouped_matmul_backward(dy, x, w, off, need_dx=False, grad_dtype=torch.float32)[1]
    o = off.tolist()
    for e in range(E):
        s = slice(o[e], o[e + 1])
        want = dy[s].double().T @ x[s].double()
        mag = dy[s].double().abs().T @ x[s].double().abs()
        close(dw[e], want, counts[e] * 2.0 ** -23 * mag)
        close(dwf[e], want, counts[e] * 2.0 ** -23 * mag)


@pytest.mark.parametrize("inner,outer", [(264, 200), (64, 64), (130, 129)])
def test_weight_gradient_in_32_bits_stays_precise(ops, inner, outer):
    """n rows summed in runs of 768, each in 48 steps that cut off at most 2^-23 of the sum,
    the runs added with a rounding of 2^-24 each: for random signs, in the 2-norm, at most
    (48 + n / 1536) 2^-23 of the result. One sum of n / 16 steps would be off by more."""
    g = gen(31)
    n = 9000
    x = torch.randn(n, inner, generator=g, device="cuda").to(torch.bfloat16)
    dy = torch.randn(n, outer, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.zeros(2, outer, inner, device="cuda", dtype=torch.bfloat16)
    off = offsets_of([0, n])
    dw = ops.grouped_matmul_backward(dy, x, w, off, need_dx=False, grad_dtype=torch.float32)[1]
    want = dy.double().T @ x.double()
    assert float((dw[1].double() - want).norm() / want.norm()) < (48 + n / 1536) * 2.0 ** -23
    assert not dw[0].any()


@pytest.mark.parametrize("inner", [1, 7, 9, 24, 31, 37, 127, 129, 260, 517])
@pytest.mark.parametrize("start", range(8))
def test_operands_at_any_address(ops, inner, start):
    """x and dy start `start` elements into rows of their own pitch, NaN around them; values are
    small integers, so that every sum is exact."""
    g = gen(inner)
    m, E, outer = 150, 2, inner + start
    off = offsets_of([90, 60])

    def view(rows, width, pitch):
        t = torch.full((rows * pitch + start + 8,), math.nan, device="cuda", dtype=torch.float16)
        v = t[start:start + rows * pitch].view(rows, pitch)[:, :width]
        return v.copy_(torch.randint(-2, 3, (rows, width), generator=g, device="cuda"))

    x = view(m, inner, inner + start % 3)
    dy = view(m, outer, outer + start % 5)
    w = torch.randint(-1, 2, (E, outer, inner), generator=g, device="cuda").half()
    _, y, _ = product64(x, w, off, None)
    _, dx, _ = product64(dy, w.transpose(1, 2), off, None)
    assert torch.equal(ops.grouped_matmul(x, w, off).double(), y)
    got, dw = ops.grouped_matmul_backward(dy, x, w, off)
    assert torch.equal(got.double(), dx)
    for e, s in enumerate((slice(0, 90), slice(90, 150))):
        assert torch.equal(dw[e].double(), dy[s].double().T @ x[s].double())


@pytest.mark.parametrize("counts,tail", [([3000, 0], 5), ([1, 0, 1500, 700], 0),
                                         ([64, 63, 2049], 1), ([600], 0), ([0, 0, 4000, 1], 3)])
@pytest.mark.parametrize("inner,outer", [(80, 56), (129, 300), (264, 200), (1, 1), (130, 3)])
def test_weight_gradient_in_parts(ops, counts, tail, inner, outer):
    """Few outputs and many rows: an expert's rows are summed in parts and the parts joined."""
    g = gen(inner + len(counts))
    m, E = sum(counts) + tail, len(counts)
    x = torch.randn(m, inner, generator=g, device="cuda").to(torch.bfloat16)
    dy = torch.randn(m, outer, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.zeros(E, outer, inner, device="cuda", dtype=torch.bfloat16)
    if tail:
        x[-1], dy[-1] = math.nan, math.inf
    off = offsets_of(counts)
    o = off.tolist()
    for grad in (torch.float32, torch.bfloat16):
        dw = ops.grouped_matmul_backward(dy, x, w, off, need_dx=False, grad_dtype=grad)[1]
        again = ops.grouped_matmul_backward(dy, x, w, off, need_dx=False, grad_dtype=grad)[1]
        assert torch.equal(dw, again)
        for e in range(E):
            s = slice(o[e], o[e + 1])
            want = dy[s].double().T @ x[s].double()
            close(dw[e], want, counts[e] * 2.0 ** -23 * (dy[s].double().abs().T @ x[s].double().abs()))


@pytest.mark.parametrize("counts", [[70, 0, 9, 130], [700, 0, 70, 333]])
@pytest.mark.parametrize("inner,outer", [(96, 80), (75, 50), (264, 392), (130, 300)])
def test_products_through_rows(ops, inner, outer, counts):
    """Tokens gathered through `rows`: repeated, unused and out of range (a row of zeros)."""
    g = gen(3)
    tokens = 60
    m = sum(counts)
    x = torch.randn(tokens, inner, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(4, outer, inner, generator=g, device="cuda").to(torch.bfloat16)
    dy = torch.randn(m, outer, generator=g, device="cuda").to(torch.bfloat16)
    rows = torch.randint(0, tokens - 5, (m,), generator=g, device="cuda").int()
    rows[3], rows[75], rows[-1] = -1, tokens, 1 << 30
    off = offsets_of(counts)
    x64, y64, mag = product64(x, w, off, rows)
    close(ops.grouped_matmul(x, w, off, rows=rows), y64, inner * 2.0 ** -23 * mag)
    dw = ops.grouped_matmul_backward(dy, x, w, off, rows=rows, need_dx=False,
                                     grad_dtype=torch.float32)[1]
    o = off.tolist()
    for e in range(4):
        s = slice(o[e], o[e + 1])
        close(dw[e], dy[s].double().T @ x64[s],
              counts[e] * 2.0 ** -23 * (dy[s].double().abs().T @ x64[s].abs()))


@pytest.mark.parametrize("counts,inner,outer", [([37, 50, 41], 96, 72), ([200, 77, 300], 264, 272)])
def test_products_neighbours_do_not_leak(ops, counts, inner, outer):
    """Infinities and NaN in one expert's rows and weights stay in its results."""
    g = gen(8)
    m, lo, hi = sum(counts), counts[0], counts[0] + counts[1]
    x = torch.randn(m, inner, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(3, outer, inner, generator=g, device="cuda").to(torch.bfloat16)
    dy = torch.randn(m, outer, generator=g, device="cuda").to(torch.bfloat16)
    off = offsets_of(counts)
    clean = [ops.grouped_matmul(x, w, off), *ops.grouped_matmul_backward(dy, x, w, off)]
    x[lo:hi], dy[lo:hi], w[1] = math.nan, math.inf, math.nan
    dirty = [ops.grouped_matmul(x, w, off), *ops.grouped_matmul_backward(dy, x, w, off)]
    for a, b, groups in zip(clean, dirty, (False, False, True)):
        for s in ((0, 2) if groups else (slice(0, lo), slice(hi, m))):
            assert torch.equal(a[s], b[s])
        assert torch.isnan(b[1] if groups else b[lo:hi]).all()


def test_products_read_strides_in_place(ops):
    g = gen(4)
    counts = [33, 100, 0, 29]
    m, off = sum(counts), offsets_of(counts)
    bx = torch.randn(m, 200, generator=g, device="cuda").to(torch.float16)
    bd = torch.randn(m, 150, generator=g, device="cuda").to(torch.float16)
    bw = torch.randn(4, 72, 64, generator=g, device="cuda").to(torch.float16)
    w2 = torch.randn(4, 64, 72, generator=g, device="cuda").to(torch.float16).transpose(1, 2)
    for x in (bx[:, 64:128], bx[:, 3:67], bx[:, ::2][:, :64]):
        for dy in (bd[:, 8:80], bd[:, 1:73]):
            for w in (bw, w2):
                a = [ops.grouped_matmul(x, w, off),
                     *ops.grouped_matmul_backward(dy, x, w, off)]
                b = [ops.grouped_matmul(x.contiguous(), w.contiguous(), off),
                     *ops.grouped_matmul_backward(dy.contiguous(), x.contiguous(),
                                                  w.contiguous(), off)]
                assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_product_gradients_by_differences(ops):
    """Small whole numbers: every product, sum and rounding is exact, so a step of one in any
    input changes <dy, y> by exactly the gradient."""
    g = gen(9)
    counts, inner, outer = [3, 0, 4], 16, 8
    m, off = 7, offsets_of(counts)
    ints = lambda *s: torch.randint(-2, 3, s, generator=g, device="cuda").to(torch.bfloat16)  # noqa
    x, w, dy = ints(m, inner), ints(3, outer, inner), ints(m, outer)
    dx, dw = ops.grouped_matmul_backward(dy, x, w, off)
    loss = lambda a, b: (ops.grouped_matmul(a, b, off).double() * dy.double()).sum()  # noqa
    base = loss(x, w)
    for r, c in [(0, 0), (2, 15), (3, 7), (6, 1)]:
        x2 = x.clone()
        x2[r, c] += 1
        assert float(loss(x2, w) - base) == float(dx[r, c])
    for e, n, c in [(0, 0, 0), (1, 3, 3), (2, 7, 15), (2, 1, 0)]:
        w2 = w.clone()
        w2[e, n, c] += 1
        assert float(loss(x, w2) - base) == float(dw[e, n, c])


def test_products_bad_offsets_stay_inside(ops):
    """Offsets that are not monotone or pass the rows are clamped: results are defined to be
    wrong, the call and the device stay usable."""
    x = torch.randn(50, 64, device="cuda").to(torch.bfloat16)
    w = torch.randn(3, 64, 64, device="cuda").to(torch.bfloat16)
    for off in ([0, 10, 5, 50], [-7, 20, 90, 1 << 30], [40, 30, 20, 10]):
        o = torch.tensor(off, dtype=torch.int32, device="cuda")
        ops.grouped_matmul(x, w, o)
        ops.grouped_matmul_backward(x, x, w, o)
    off = offsets_of([20, 0, 30])
    _, y64, mag = product64(x, w, off, None)
    close(ops.grouped_matmul(x, w, off), y64, 64 * 2.0 ** -23 * mag)


def test_products_without_rows(ops):
    x = torch.empty(0, 32, device="cuda", dtype=torch.float16)
    w = torch.ones(2, 24, 32, device="cuda", dtype=torch.float16)
    off = offsets_of([0, 0])
    assert ops.grouped_matmul(x, w, off).shape == (0, 24)
    dx, dw = ops.grouped_matmul_backward(torch.empty(0, 24, device="cuda", dtype=torch.float16),
                                         x, w, off)
    assert dx.shape == (0, 32) and not dw.any()


# ------------------------------------------------------------------------- few rows, 4 bits


FEW = [  # counts, tail rows, inner, outer
    ([1], 0, 1, 1), ([0, 1, 0, 1], 0, 4096, 300), ([3, 0, 9], 2, 700, 129), ([8, 8, 8, 8], 0, 512, 128),
    ([33, 0, 0, 1], 3, 513, 1000), ([65], 0, 2000, 72), ([2] * 40, 1, 75, 50), ([1] * 300, 0, 64, 40),
    ([0, 0, 0], 4, 100, 20), ([7, 1, 30, 2, 0, 5], 0, 1028, 260),
]


@pytest.mark.parametrize("through_rows", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("counts,tail,inner,outer", FEW)
def test_product_of_few_rows(ops, counts, tail, inner, outer, dtype, through_rows):
    dt, g = DTYPES[dtype], gen(inner + outer)
    m, E = sum(counts) + tail, len(counts)
    tokens = m // 2 + 3 if through_rows else m
    x = torch.randn(tokens, inner, generator=g, device="cuda").to(dt)
    w = (torch.randn(E, outer, inner, generator=g, device="cuda") * inner ** -0.5).to(dt)
    rows = None
    if through_rows:
        rows = torch.randint(-1, tokens + 1, (m,), generator=g, device="cuda").int()
    off = offsets_of(counts)
    _, y64, mag = product64(x, w, off, rows)
    close(ops.grouped_matmul(x, w, off, rows=rows), y64, inner * 2.0 ** -23 * mag)


def unpacked(q, scales, zeros, inner, group):
    v = torch.stack([q & 15, q >> 4], 3).flatten(2)[:, :, :inner].double()
    at = torch.arange(inner, device="cuda") // group
    z = 8.0 if zeros is None else zeros.double()[:, :, at]
    return (v - z) * scales.double()[:, :, at]


@pytest.mark.parametrize("with_zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("counts,tail,inner,outer", FEW)
def test_product_w4(ops, counts, tail, inner, outer, dtype, group, with_zeros):
    """Every weight is scale * (q - z) exactly; n products and n / group scalings in f32."""
    dt, g = DTYPES[dtype], gen(inner * 3 + group)
    m, E = sum(counts) + tail, len(counts)
    x = torch.randn(m, inner, generator=g, device="cuda").to(dt)
    q = torch.randint(0, 256, (E, outer, (inner + 31) // 32 * 16), generator=g, device="cuda",
                      dtype=torch.uint8)  # what the padding holds does not matter
    groups = -(-inner // group)
    scales = torch.randn(E, outer, groups, generator=g, device="cuda").to(dt)
    zeros = None
    if with_zeros:
        zeros = torch.randint(0, 16, (E, outer, groups), generator=g, device="cuda",
                              dtype=torch.uint8)
    off = offsets_of(counts)
    w = unpacked(q, scales, zeros, inner, group)
    _, y64, _ = product64(x, w, off, None)
    # inside a group the sum runs over |x| |q - z|, whatever cancels there
    _, _, mag = product64(x, w.abs(), off, None)
    got = ops.grouped_matmul_w4(x, q, scales, off, zeros=zeros, group_size=group)
    close(got, y64, (inner + groups) * 2.0 ** -23 * mag)


def test_w4_through_rows_and_strides(ops):
    g = gen(21)
    big = torch.randn(9, 400, generator=g, device="cuda").to(torch.float16)
    q = torch.randint(0, 256, (3, 60, 112), generator=g, device="cuda", dtype=torch.uint8)
    scales = torch.rand(3, 60, 4, generator=g, device="cuda").half()
    rows = torch.tensor([8, 0, -1, 5, 5, 9, 2], device="cuda", dtype=torch.int32)
    off = offsets_of([2, 4, 1])
    for x in (big[:, 5:205], big[:, 8:208], big[:, ::2]):
        w = unpacked(q, scales, None, 200, 64)
        _, y64, mag = product64(x, w, off, rows)
        got = ops.grouped_matmul_w4(x, q, scales, off, rows=rows, group_size=64)
        close(got, y64, 204 * 2.0 ** -23 * mag)


@pytest.mark.parametrize("inner,group", [(256, 128), (75, 32), (700, 64)])
def test_quantize_w4_error(ops, inner, group):
    """Rounding to the nearest of the group's steps: half a step, where the step (the scale) is
    first rounded to bf16 (2^-8 of up to 15 steps, and the zero point moves by half a step)."""
    w = torch.randn(3, 40, inner, generator=gen(2), device="cuda").to(torch.bfloat16)
    for symmetric in (False, True):
        q, s, z = ops.quantize_w4(w, group, symmetric=symmetric)
        step = s.double()[:, :, torch.arange(inner, device="cuda") // group]
        off = (unpacked(q, s, z, inner, group) - w.double()).abs()
        assert (off <= step * (1.0 + 15 * 2.0 ** -8)).all()


# ---------------------------------------------------------------------------- combine


COMBINE = [  # tokens, k, width
    (1, 1, 1), (3, 2, 700), (100, 5, 33), (1000, 4, 256), (37, 3, 2048), (5, 16, 4100), (2049, 2, 8),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,k,width", COMBINE)
def test_combine(ops, tokens, k, width, dtype):
    dt = DTYPES[dtype]
    g = gen(tokens * k + width)
    m = tokens * k
    y = torch.randn(m, width, generator=g, device="cuda").to(dt)
    pos = torch.randperm(m, generator=g, device="cuda").view(tokens, k).int()
    w = torch.randn(tokens, k, generator=g, device="cuda")
    dout = torch.randn(tokens, width, generator=g, device="cuda").to(dt)
    ys = y.double()[pos.long()]
    close(ops.combine(y, pos, w), (w.double()[:, :, None] * ys).sum(1),
          k * 2.0 ** -23 * (w.double()[:, :, None] * ys).abs().sum(1))
    close(ops.combine(y, pos), ys.sum(1), k * 2.0 ** -23 * ys.abs().sum(1))
    dy, dw = ops.combine_backward(dout, y, pos, w)
    want = torch.empty(m, width, dtype=torch.float64, device="cuda")
    want[pos.long()] = w.double()[:, :, None] * dout.double()[:, None, :]
    close(dy, want, 2.0 ** -24 * want.abs())
    prod = dout.double()[:, None, :] * ys
    close(dw, prod.sum(2), width * 2.0 ** -23 * prod.abs().sum(2))
    dy1, none = ops.combine_backward(dout, y, pos)
    want[pos.long()] = dout.double()[:, None, :].expand(tokens, k, width)
    assert none is None and torch.equal(dy1.double(), want)


def test_combine_strides_and_positions_outside(ops):
    g = gen(2)
    big = torch.randn(40, 300, generator=g, device="cuda")
    y = big[:, 5:205]
    pos = torch.randint(0, 40, (9, 3), generator=g, device="cuda").int()
    pos[0, 0], pos[1] = 40, -1
    w = torch.randn(9, 3, generator=g, device="cuda")
    ys = y.double()[pos.long().clamp(0, 39)]
    ys[((pos < 0) | (pos > 39)).nonzero(as_tuple=True)] = 0
    close(ops.combine(y, pos, w), (w.double()[:, :, None] * ys).sum(1),
          3 * 2.0 ** -23 * (w.double()[:, :, None] * ys).abs().sum(1))


def test_combine_gradient_by_differences(ops):
    """Whole numbers: exact, as for the products."""
    g = gen(6)
    ints = lambda *s: torch.randint(-3, 4, s, generator=g, device="cuda").float()  # noqa
    y, w, dout = ints(12, 40), ints(4, 3), ints(4, 40)
    pos = torch.randperm(12, generator=g, device="cuda").view(4, 3).int()
    dy, dw = ops.combine_backward(dout, y, pos, w)
    loss = lambda a, b: (ops.combine(a, pos, b).double() * dout.double()).sum()  # noqa
    base = loss(y, w)
    for r, c in [(0, 0), (5, 39), (11, 7)]:
        y2 = y.clone()
        y2[r, c] += 1
        assert float(loss(y2, w) - base) == float(dy[r, c])
    for t, j in [(0, 0), (3, 2)]:
        w2 = w.clone()
        w2[t, j] += 1
        assert float(loss(y, w2) - base) == float(dw[t, j])


# ---------------------------------------------------------------------------- dropout


def philox(counter, key):
    """Philox4x32-10 of one counter (four words) and key (two), in Python integers."""
    c, (k0, k1) = list(counter), key
    for _ in range(10):
        p, q = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(q >> 32) ^ c[1] ^ k0, q & 0xFFFFFFFF, (p >> 32) ^ c[3] ^ k1, p & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def test_philox_published_vectors():
    """Known answers of Philox4x32-10 from its authors' published test vectors."""
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    f = 0xFFFFFFFF
    assert philox((f, f, f, f), (f, f)) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


def kept(n, p, seed, offset, first=0):
    drop = int(math.floor(p * 65536 + 0.5))
    bits = []
    for b in range(first // 8, (first + n + 7) // 8):
        for w in philox((b & 0xFFFFFFFF, b >> 32, offset & 0xFFFFFFFF, offset >> 32),
                        (seed & 0xFFFFFFFF, seed >> 32)):
            bits += [w & 0xFFFF, w >> 16]
    keep = torch.tensor(bits, device="cuda")[first % 8:first % 8 + n] >= drop
    return keep, 65536.0 / (65536 - drop) if drop < 65536 else 0.0


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape,p", [((1,), 0.5), ((7, 3), 0.1), ((33, 101), 0.25), ((4, 5, 6), 0.9),
                                     ((16, 128), 0.0), ((3, 8), 1.0), ((1000,), 1e-9),
                                     ((257, 16), 0.37)])
def test_dropout(ops, shape, p, dtype):
    dt, seed, offset = DTYPES[dtype], 0xFEDCBA9876543210, (7 << 32) + 5
    g = gen(3)
    x = torch.randn(shape, generator=g, device="cuda").to(dt)
    res = torch.randn(shape, generator=g, device="cuda").to(dt)
    keep, scale = kept(x.numel(), p, seed, offset)
    keep = keep.view(shape)
    want = torch.where(keep, x.double() * scale, 0.0)
    close(ops.dropout(x, p, seed, offset), want, 2.0 ** -23 * want.abs())
    both = want + res.double()
    close(ops.dropout(x, p, seed, offset, residual=res), both,
          2.0 ** -22 * (want.abs() + res.double().abs()))
    assert torch.equal(ops.dropout_backward(x, p, seed, offset), ops.dropout(x, p, seed, offset))
    # dropped places give 0 whatever they hold, kept ones what they hold
    bad = ops.dropout(torch.full_like(x, math.nan), p, seed, offset)
    assert torch.equal(torch.isnan(bad), keep) and not bad[~keep].any()


def test_dropout_gradient_by_differences(ops):
    """Linear in x: with p = 1/2 the scale is 2 and whole numbers stay exact."""
    x = torch.randint(-8, 9, (12, 19), device="cuda").float()
    dout = torch.randint(-8, 9, (12, 19), device="cuda").float()
    d = ops.dropout_backward(dout, 0.5, 11, 3)
    loss = lambda a: (ops.dropout(a, 0.5, 11, 3).double() * dout.double()).sum()  # noqa
    base = loss(x)
    for r, c in [(0, 0), (5, 18), (11, 7), (3, 3)]:
        x2 = x.clone()
        x2[r, c] += 1
        assert float(loss(x2) - base) == float(d[r, c])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_dropout_strides(ops, dtype):
    big = torch.randn(50, 96, device="cuda").to(DTYPES[dtype])
    flat = torch.randn(50 * 32 + 1, device="cuda").to(DTYPES[dtype])
    for x in (big[:, 8:40], big[:, 3:35], big[::2, 8:40], big.t()[8:40], flat[1:].view(50, 32)):
        want = ops.dropout(x.contiguous().clone(), 0.3, 1)
        assert torch.equal(ops.dropout(x, 0.3, 1), want)
        for res in (x, x.contiguous()):
            assert torch.equal(ops.dropout(x, 0.3, 1, residual=res),
                               ops.dropout(x.contiguous().clone(), 0.3, 1,
                                           residual=x.contiguous()))


def test_dropout_counter_passes_32_bits(ops):
    """Elements from 2^35 on take block numbers past 32 bits: walked as a row pitch, a view of
    one row repeated would need that much memory, so the high word is tested by an offset."""
    x = torch.ones(4096, device="cuda")
    a, b = ops.dropout(x, 0.5, 1, 1), ops.dropout(x, 0.5, 1, (1 << 32) + 1)
    assert not torch.equal(a, b)
    k, scale = kept(4096, 0.5, 1, (1 << 32) + 1)
    assert torch.equal(b, k.float() * scale)


def test_dropout_rate(ops):
    """Of n = 2^22 independent draws the kept share is within 6 standard deviations."""
    n, p = 1 << 22, 0.3
    got = float((ops.dropout(torch.ones(n, device="cuda"), p, 99) != 0).double().mean())
    q = 1 - int(p * 65536 + 0.5) / 65536
    assert abs(got - q) < 6 * math.sqrt(q * (1 - q) / n)


# ------------------------------------------------------------------- all of them together


def test_same_bits_every_time_and_on_another_stream(ops):
    g = gen(12)
    x = torch.randn(3000, 136, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn(3000, 40, generator=g, device="cuda")
    w = torch.randn(40, 72, 136, generator=g, device="cuda").to(torch.bfloat16)
    dout = torch.randn(3000, 72, generator=g, device="cuda").to(torch.bfloat16)

    def step():
        r = ops.route(logits, 3)
        y = ops.grouped_matmul(x, w, r.offsets, rows=r.rows)
        h = ops.dropout(y, 0.2, 5)
        out = ops.combine(h, r.position, r.weights)
        dh, dwt = ops.combine_backward(dout, h, r.position, r.weights)
        dy = ops.dropout_backward(dh, 0.2, 5)
        dx, dw = ops.grouped_matmul_backward(dy, x, w, r.offsets, rows=r.rows)
        return [out, ops.combine(dx, r.position), dw, ops.route_backward(dwt, logits, r)]

    first = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = step()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_layer_against_autograd(ops):
    """A whole layer, tokens shared by two experts each, against torch's autograd in f64 on the
    same bf16 weights. On the way to a gradient at most five results are rounded to bf16 (h, y,
    dy, dh, dx), each by 2^-8 of itself at most: 5 * 2^-8 in the 2-norm."""
    g = gen(44)
    T, E, k, K, H, N = 150, 6, 2, 24, 40, 16
    bf = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa
    x, w1, w2, dout = bf(T, K), bf(E, H, K) * 0.2, bf(E, N, H) * 0.2, bf(T, N)
    logits = torch.randn(T, E, generator=g, device="cuda")
    for normalize in (True, False):
        r = ops.route(logits, k, normalize=normalize)
        h = ops.grouped_matmul(x, w1, r.offsets, rows=r.rows)
        y = ops.grouped_matmul(h, w2, r.offsets)
        out = ops.combine(y, r.position, r.weights)
        dy, dwt = ops.combine_backward(dout, y, r.position, r.weights)
        dh, dw2 = ops.grouped_matmul_backward(dy, h, w2, r.offsets, grad_dtype=torch.float32)
        dxs, dw1 = ops.grouped_matmul_backward(dh, x, w1, r.offsets, rows=r.rows,
                                               grad_dtype=torch.float32)
        got = [out, ops.combine(dxs, r.position), dw1, dw2,
               ops.route_backward(dwt, logits, r, normalize=normalize)]
        p = [t.double().requires_grad_() for t in (x, w1, w2, logits)]
        e = r.experts.long()
        soft = (p[3].gather(1, e) if normalize else p[3]).softmax(1)
        wt = soft if normalize else soft.gather(1, e)
        each = torch.einsum("tknh,tkh->tkn", p[2][e], torch.einsum("tkhc,tc->tkh", p[1][e], p[0]))
        ref = (wt[:, :, None] * each).sum(1)
        want = [ref.detach(), *torch.autograd.grad(ref, p, dout.double())]
        for a, b in zip(got, want):
            assert float((a.double() - b).norm() / b.norm()) < 5 * 2.0 ** -8


def test_graph_capture(ops):
    """Routing and products read their offsets on the device: a step replays on new inputs."""
    g = gen(45)
    x = torch.randn(300, 64, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(5, 72, 64, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn(300, 5, generator=g, device="cuda")

    def step():
        r = ops.route(logits, 2)
        y = ops.dropout(ops.grouped_matmul(x, w, r.offsets, rows=r.rows), 0.25, 3)
        return ops.combine(y, r.position, r.weights)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    logits.copy_(torch.randn(300, 5, generator=g, device="cuda"))
    x.copy_(torch.randn(300, 64, generator=g, device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, step())


def test_offsets_pass_32_bits(ops):
    """Tensors of more than 2^32 elements: the last rows, weights and elements."""
    g = gen(46)
    n = (1 << 32) + 4099
    x = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    x[-4099:] = 1
    got = ops.dropout(x, 0.5, 17, 2)[-4099:]
    keep, scale = kept(4099, 0.5, 17, 2, first=1 << 32)
    assert torch.equal(got.double(), keep.double() * scale)
    del x, got

    y = torch.empty(70_000, 64_000, device="cuda", dtype=torch.bfloat16)  # 4.48e9
    y[-2:] = torch.randn(2, 64_000, generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.tensor([[69_999, 69_998]], dtype=torch.int32, device="cuda")
    wt = torch.tensor([[0.5, -2.0]], device="cuda")
    want = 0.5 * y[-1:].double() - 2.0 * y[-2:-1].double()
    close(ops.combine(y, pos, wt), want, 2.0 ** -22 * (y[-1:].double().abs() + 2 * y[-2:-1].abs()))
    del y

    w = torch.zeros(70, 8192, 8192, device="cuda", dtype=torch.bfloat16)  # 4.7e9
    w[-1] = torch.randn(8192, 8192, generator=g, device="cuda").to(torch.bfloat16)
    for m in (3, 70 * 40):  # streamed, and in tiles
        xs = torch.randn(m, 8192, generator=g, device="cuda").to(torch.bfloat16)
        off = offsets_of([0] * 69 + [m])
        want = xs.double() @ w[-1].double().T
        mag = xs.double().abs() @ w[-1].double().abs().T
        close(ops.grouped_matmul(xs, w, off), want, 8192 * 2.0 ** -23 * mag)


def refusals():
    bf, i32 = torch.bfloat16, torch.int32
    c = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa
    off = lambda n: c(n, dtype=i32)  # noqa
    u8 = lambda *s: c(*s, dtype=torch.uint8)  # noqa
    return [
        lambda o: o.route(c(4, 5), 0),
        lambda o: o.route(c(4, 5), 6),
        lambda o: o.route(c(4, 5).double(), 2),
        lambda o: o.route(c(4, 600), 2),
        lambda o: o.route(c(4, 100), 17),
        lambda o: o.route(c(4, 5).cpu(), 2),
        lambda o: o.route(c(4, 5, 6), 2),
        lambda o: o.route_backward(c(4, 3), c(4, 5), o.route(c(4, 5), 2)),
        lambda o: o.grouped_matmul(c(4, 8), c(2, 8, 8), off(3)),
        lambda o: o.grouped_matmul(c(4, 8, dtype=bf), c(2, 8, 9, dtype=bf), off(3)),
        lambda o: o.grouped_matmul(c(4, 8, dtype=bf), c(2, 8, 8, dtype=bf), off(2)),
        lambda o: o.grouped_matmul(c(4, 8, dtype=bf), c(2, 8, 8, dtype=bf), off(3).long()),
        lambda o: o.grouped_matmul(c(4, 8, dtype=bf), c(2, 8, 8, dtype=torch.float16), off(3)),
        lambda o: o.grouped_matmul(c(4, 8, dtype=bf), c(2, 8, 8, dtype=bf), off(3),
                                   rows=off(4).long()),
        lambda o: o.grouped_matmul(c(4, 8, dtype=bf), c(600, 8, 8, dtype=bf), off(601)),
        lambda o: o.grouped_matmul_backward(c(5, 8, dtype=bf), c(4, 8, dtype=bf),
                                            c(2, 8, 8, dtype=bf), off(3)),
        lambda o: o.grouped_matmul_backward(c(4, 8, dtype=bf), c(4, 8, dtype=bf),
                                            c(2, 8, 8, dtype=bf), off(3), grad_dtype=torch.float16),
        lambda o: o.grouped_matmul_w4(c(4, 64, dtype=bf), u8(2, 8, 32), c(2, 8, 2, dtype=bf), off(3),
                                      group_size=48),
        lambda o: o.grouped_matmul_w4(c(4, 64, dtype=bf), u8(2, 8, 31), c(2, 8, 2, dtype=bf), off(3),
                                      group_size=32),
        lambda o: o.grouped_matmul_w4(c(4, 64, dtype=bf), u8(2, 8, 32), c(2, 8, 1, dtype=bf), off(3),
                                      group_size=32),
        lambda o: o.grouped_matmul_w4(c(4, 64, dtype=bf), u8(2, 8, 32), c(2, 8, 2), off(3),
                                      group_size=32),
        lambda o: o.grouped_matmul_w4(c(4, 64), u8(2, 8, 32), c(2, 8, 2), off(3), group_size=32),
        lambda o: o.combine(c(4, 8), c(2, 2).long()),
        lambda o: o.combine(c(4, 8), off(4)),
        lambda o: o.combine(c(4, 8), c(2, 2, dtype=i32), c(2, 3)),
        lambda o: o.combine_backward(c(2, 8), c(5, 8), c(2, 2, dtype=i32)),
        lambda o: o.combine_backward(c(3, 8), c(4, 8), c(2, 2, dtype=i32)),
        lambda o: o.dropout(c(4, 8), 1.5, 0),
        lambda o: o.dropout(c(4, 8), float("nan"), 0),
        lambda o: o.dropout(c(4, 8), 0.5, -1),
        lambda o: o.dropout(c(4, 8), 0.5, 1 << 64),
        lambda o: o.dropout(c(4, 8).double(), 0.5, 0),
        lambda o: o.dropout(c(4, 8), 0.5, 0, residual=c(4, 9)),
    ]


@pytest.mark.parametrize("i", range(33))
def test_refusals(ops, i):
    from lightgbm_rs_b200 import LightGBMError

    calls = refusals()
    assert len(calls) == 33
    with pytest.raises(LightGBMError):
        calls[i](ops)
