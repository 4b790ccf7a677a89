"""Expert-layer operators on the GPU where they could go wrong.

Tolerances are bounds derived from the arithmetic, given at each test.
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_experts import DTYPES, UNIT, gen, offsets_of, product64, unpacked  # noqa: E402


@pytest.fixture(scope="module")
def ops():
    from lightgbm_rs_b200 import experts

    yield experts
    experts.check_errors()


# --------------------------------------------------------- rows before the first offset


LEAD = [  # rows before the first offset, counts, tail rows, inner, outer
    (1, [2], 0, 64, 64), (3, [0, 1], 1, 40, 24), (9, [1, 0, 5], 0, 700, 129), (70, [1] * 40, 2, 96, 72),
    (40, [200, 0, 77], 3, 72, 520), (300, [129, 1000], 0, 200, 264), (257, [31, 400], 200, 129, 700),
    (5, [0, 0], 0, 48, 40),
]


@pytest.mark.parametrize("lead,counts,tail,inner,outer", LEAD)
def test_rows_before_the_first_offset_are_zero(ops, lead, counts, tail, inner, outer):
    """A shard of the experts has offsets that do not start at 0. Results go to memory that holds
    NaN: what is not written stays NaN."""
    from lightgbm_rs_b200 import _lib as C

    g, L = gen(lead + inner), C.lib()
    m, E = lead + sum(counts) + tail, len(counts)
    x = torch.randn(m, inner, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(E, outer, inner, generator=g, device="cuda") * inner ** -0.5).to(torch.bfloat16)
    dy = torch.randn(m, outer, generator=g, device="cuda").to(torch.bfloat16)
    off = offsets_of(counts) + lead
    x[:lead], dy[:lead] = math.inf, math.nan  # rows of no expert hold what they like
    st = torch.cuda.current_stream().cuda_stream
    p = lambda t: t.data_ptr()  # noqa: E731
    nan = lambda *s: torch.full(s, math.nan, device="cuda", dtype=torch.bfloat16)  # noqa: E731

    y = nan(m, outer)
    n = L.lgbm_b200_experts_matmul_workspace(p(x), inner, None, p(w), m, E, inner, outer)
    ws = torch.empty(max(n, 16), device="cuda", dtype=torch.uint8)
    C.check(L.lgbm_b200_experts_matmul(p(x), m, inner, None, p(w), p(off), 1, m, E, inner, outer,
                                       p(y), p(ws), n, st))
    dx, dw = nan(m, inner), nan(E, outer, inner)
    n = L.lgbm_b200_experts_matmul_backward_workspace(p(dy), outer, p(x), inner, None, p(w), m, E,
                                                      inner, outer, 1, 1)
    ws = torch.empty(max(n, 16), device="cuda", dtype=torch.uint8)
    C.check(L.lgbm_b200_experts_matmul_backward(p(dy), outer, p(x), m, inner, None, p(w), p(off), 1,
                                                1, m, E, inner, outer, p(dx), p(dw), p(ws), n, st))
    q = torch.randint(0, 256, (E, outer, (inner + 31) // 32 * 16), generator=g, device="cuda",
                      dtype=torch.uint8)
    scales = torch.randn(E, outer, -(-inner // 64), generator=g, device="cuda").to(torch.bfloat16)
    y4 = nan(m, outer)
    C.check(L.lgbm_b200_experts_matmul_w4(p(x), m, inner, None, p(q), p(scales), None, 64, p(off), 1,
                                          m, E, inner, outer, p(y4), st))

    inside = slice(lead, m - tail)
    for got, a, b, length in ((y, x, w, inner), (dx, dy, w.transpose(1, 2), outer),
                              (y4, x, unpacked(q, scales, None, inner, 64), inner)):
        assert not got[:lead].any() and not got[m - tail:].any()
        # n products summed in f32 (and scaled by group), and a rounding to bf16
        _, want, mag = product64(a[inside], b, off - lead, None)
        mag = product64(a[inside], b.abs(), off - lead, None)[2]
        lim = 1.1 * length * 2.0 ** -23 * mag + 2.0 ** -8 * want.abs() + 2.0 ** -25
        assert ((got[inside].double() - want).abs() <= lim).all()
    o = off.tolist()
    for e in range(E):
        s = slice(o[e], o[e + 1])
        want, mag = (f(dy[s].double()).T @ f(x[s].double()) for f in (lambda t: t, torch.abs))
        assert ((dw[e].double() - want).abs()
                <= counts[e] * 2.0 ** -23 * mag + 2.0 ** -8 * want.abs()).all()


def test_a_shard_of_the_experts(ops):
    """Experts 2 to 4 of six with their slice of the offsets give their rows of the whole."""
    g = gen(17)
    counts = [50, 3, 70, 0, 20, 9]
    off, m = offsets_of(counts), sum(counts)
    x = torch.randn(m, 72, generator=g, device="cuda").half()
    w = torch.randn(6, 40, 72, generator=g, device="cuda").half()
    whole = ops.grouped_matmul(x, w, off)
    part = ops.grouped_matmul(x, w[2:5], off[2:6])
    lo, hi = int(off[2]), int(off[5])
    assert torch.equal(part[lo:hi], whole[lo:hi])
    assert not part[:lo].any() and not part[hi:].any()


# --------------------------------------------------------------------------- long sums


RUN = 4096  # longest sum the tensor cores make in one piece for a result of 16 bits


def spread(g, rows, cols, dtype, lo=0.0):
    """Numbers of one sign whose columns have scales in [1/2, 1): sums over the rows fall evenly
    over the result type's spacings, so that its roundings cancel in the mean."""
    t = torch.rand(rows, cols, generator=g, device="cuda") / 16
    return t.mul_(torch.rand(cols, generator=g, device="cuda") / 2 + 0.5).to(dtype)


def bias(got, want):
    return float(((got.double() - want) / want).mean())


def bias_limit(n, dtype, independent):
    """Adding to a sum cuts off at most 2^-23 of it, RUN / 16 times in a run; the n / RUN runs are
    added in f32. The result's rounding (at most a unit, half of it in the root mean square)
    cancels over `independent` results, to six standard deviations."""
    return (RUN / 16 + n / (2 * RUN)) * 2.0 ** -23 + 6 * UNIT[dtype] / 2 / math.sqrt(independent)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n,inner,outer", [(1 << 18, 1536, 2048), (1 << 17, 64, 9600),
                                           (1 << 17, 128, 9600), (1 << 17, 19200, 100)])
def test_weight_gradient_of_long_groups(ops, n, inner, outer, dtype):
    """One expert, outputs enough that its rows are not summed in parts, all terms of one sign:
    what the additions cut off adds up. In one piece it is 1.6e-3 of the result at 2^18 rows."""
    dt, g = DTYPES[dtype], gen(n + inner)
    x, dy = spread(g, n, inner, dt), spread(g, n, outer, dt)
    w = torch.empty(2, outer, inner, device="cuda", dtype=dt)
    off = offsets_of([n, 0])
    dw = ops.grouped_matmul_backward(dy, x, w, off, need_dx=False)[1]
    want = torch.zeros(outer, inner, device="cuda", dtype=torch.float64)
    for r in range(0, n, 1 << 14):
        want += dy[r:r + (1 << 14)].double().T @ x[r:r + (1 << 14)].double()
    assert abs(bias(dw[0], want)) <= bias_limit(n, dt, max(inner, outer))
    # each element: as above, and one rounding
    lim = (RUN / 16 + n / RUN) * 2.0 ** -23 + UNIT[dt]
    assert (((dw[0].double() - want) / want).abs() <= lim).all()
    assert not dw[1].any()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,experts,cols", [(300, 1, 64), (300, 1, 128), (300, 3, 300),
                                               (300, 1, 300), (3, 1, 19200), (30, 1, 19200)])
def test_products_of_long_reductions(ops, rows, experts, cols, dtype):
    """y over 2^17 inputs and dx over 2^17 outputs, streamed (3 rows) and in every tile shape."""
    n = 1 << 17 if cols < 1000 else 1 << 16
    dt, g = DTYPES[dtype], gen(rows + cols)
    a = spread(g, n, rows, dt).t().contiguous()
    b = spread(g, n, cols, dt).t().contiguous()
    off = offsets_of([rows // experts] * experts)
    w = b.expand(experts, cols, n).contiguous()
    want = torch.cat([a.double() @ b[c:c + 512].double().T for c in range(0, cols, 512)], 1)
    got = [ops.grouped_matmul(a, w, off)]
    del w
    if cols < 1000:
        w = b.t().expand(experts, n, cols).contiguous()
        got.append(ops.grouped_matmul_backward(a, a[:, :cols], w, off, need_dw=False)[0])
    for y in got:
        assert abs(bias(y, want)) <= bias_limit(n, dt, max(rows, cols))
        lim = (RUN / 16 + n / RUN) * 2.0 ** -23 + UNIT[dt]
        assert (((y.double() - want) / want).abs() <= lim).all()


# -------------------------------------------------------------------------------- router


@pytest.mark.parametrize("tokens", [3, 100])
def test_route_gradient_of_far_logits(ops, tokens):
    """Softmax over all: the unchosen experts' gradient is -p_e p_0 g with p_e down to e^-80. In
    units of 2^-24: exp 4 (its argument is exact here), the weight's sum of up to 7 additions and
    quotient 8, p_0 g and the two products 3, the weight twice: 23. Results below 2^-126 are spaced
    by 2^-149."""
    g = gen(tokens)
    x = -(20 + torch.randint(0, 60 * 1024, (tokens, 40), generator=g, device="cuda") / 1024)
    x[:, 7] = 0
    dw = torch.randn(tokens, 1, generator=g, device="cuda")
    r = ops.route(x, 1, normalize=False)
    d = ops.route_backward(dw, x, r, normalize=False)
    p = x.double().softmax(1)
    want = -p * p[:, 7:8] * dw.double()
    off = (d.double() - want).abs()
    off[:, 7] = 0
    assert (off <= 24 * 2.0 ** -24 * want.abs() + 2.0 ** -150).all()


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("experts,k", [(1, 1), (8, 2), (31, 8), (64, 4), (130, 5), (255, 4), (512, 16)])
def test_route_does_not_depend_on_the_batch(ops, experts, k, normalize):
    """A token's choice and weights have the same bits served alone and in a batch."""
    g = gen(experts)
    x = torch.randn(130, experts, generator=g, device="cuda") * 4
    x.masked_fill_(torch.rand(130, experts, generator=g, device="cuda") > 0.8, -math.inf)
    whole = ops.route(x, k, normalize=normalize)
    for size in (1, 7, 64, 65):
        part = ops.route(x[:size], k, normalize=normalize)
        assert torch.equal(part.experts, whole.experts[:size])
        assert torch.equal(part.weights, whole.weights[:size])


# ----------------------------------------------------------------------- check_errors


def test_check_errors_waits_for_side_streams(ops):
    """A stream of torch's pool does not order with the legacy default stream: the check has to
    wait for the device, or it reads the error word of kernels that still run."""
    ops.check_errors()  # the first call loads the module, which waits too
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)  # cycles: a fifth of a second
        done = side.record_event()
    ops.check_errors()
    assert done.query()


# ----------------------------------------------------------------- the Python boundary


def test_inputs_that_want_gradients_are_refused(ops):
    """The functions record nothing for autograd: a result that does not require gradients though
    its input does would lose them without a word."""
    from lightgbm_rs_b200 import LightGBMError

    c = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    want = lambda *s: c(*s).requires_grad_()  # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    off = torch.tensor([0, 2, 4], device="cuda", dtype=torch.int32)
    pos = torch.arange(4, device="cuda", dtype=torch.int32).view(2, 2)
    q = torch.zeros(2, 8, 16, device="cuda", dtype=torch.uint8)
    r = ops.route(f32(4, 2), 1)
    calls = [
        lambda: ops.route(f32(4, 5).requires_grad_(), 2),
        lambda: ops.route_backward(f32(4, 1).requires_grad_(), f32(4, 2), r),
        lambda: ops.grouped_matmul(want(4, 8), c(2, 8, 8), off),
        lambda: ops.grouped_matmul(c(4, 8), want(2, 8, 8), off),
        lambda: ops.grouped_matmul_backward(c(4, 8), c(4, 8), want(2, 8, 8), off),
        lambda: ops.grouped_matmul_w4(c(4, 8), q, want(2, 8, 1), off, group_size=32),
        lambda: ops.combine(want(4, 8), pos),
        lambda: ops.combine(c(4, 8), pos, f32(2, 2).requires_grad_()),
        lambda: ops.combine_backward(want(2, 8), c(4, 8), pos),
        lambda: ops.dropout(want(4, 8), 0.5, 1),
        lambda: ops.dropout(c(4, 8), 0.5, 1, residual=want(4, 8)),
    ]
    for call in calls:
        with pytest.raises(LightGBMError, match="no_grad"):
            call()
        with torch.no_grad():
            call()


def test_operands_that_are_not_read_are_not_copied(ops):
    """Only dw is wanted, or only dx: w, or x, gives its shape, and its strides cost no memory."""
    dy = torch.randn(4096, 512, device="cuda").to(torch.bfloat16)
    x = torch.randn(512, 4096, device="cuda").to(torch.bfloat16).t()
    w = torch.randn(8, 512, 512, device="cuda").to(torch.bfloat16).transpose(1, 2)
    off = offsets_of([512] * 8)

    def peak(x, w, **which):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        ops.grouped_matmul_backward(dy, x, w, off, **which)
        return torch.cuda.max_memory_allocated() - before

    straight_x, straight_w = x.contiguous(), w.contiguous()
    assert peak(straight_x, w, need_dx=False) == peak(straight_x, straight_w, need_dx=False)
    assert peak(x, straight_w, need_dw=False) == peak(straight_x, straight_w, need_dw=False)


@pytest.mark.parametrize("tokens,experts,k", [(3_000_017, 16, 2), (400_003, 255, 4)])
def test_route_large_batches(ops, tokens, experts, k):
    g = gen(experts)
    x = torch.randn(tokens, experts, generator=g, device="cuda")
    x.masked_fill_(torch.rand(tokens, experts, generator=g, device="cuda") > 0.9, -math.inf)
    r = ops.route(x, k)
    top, ids = x.sort(dim=1, descending=True, stable=True)
    top, ids = top[:, :k], ids[:, :k].masked_fill(top[:, :k] == -math.inf, -1)
    assert torch.equal(r.experts.long(), ids)
    flat = torch.where(ids < 0, experts, ids).reshape(-1)
    group, order = flat.sort(stable=True)
    assert torch.equal(r.rows.long(), order // k)
    assert torch.equal(r.position.reshape(-1).long()[order], torch.arange(tokens * k, device="cuda"))
    assert torch.equal(r.offsets.long(),
                       torch.searchsorted(group, torch.arange(experts + 1, device="cuda")))


# ----------------------------------------------------------- infinities, odd addresses


def same(got, want, slack):
    """As close() of the main tests, with infinities of the same sign in the same places; `want`
    in 64 bits, beyond the type's range where that is meant."""
    w = want.to(got.dtype).double()
    g = got.double()
    assert torch.equal(torch.isnan(g), torch.isnan(w))
    inf = torch.isinf(w)
    assert torch.equal(g[inf], w[inf])
    fin = torch.isfinite(w)
    lim = slack + UNIT[got.dtype] * want.abs() + 2.0 ** -25
    assert (((g - want).abs() <= lim) | ~fin).all()


@pytest.mark.parametrize("rows", [3, 200])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_overflow_and_infinities(ops, rows, dtype):
    """Every second result row is far beyond f16's range, and one input is infinite. Whole
    numbers below 2^24: the sums are exact."""
    dt, g = DTYPES[dtype], gen(rows)
    x = torch.randint(1, 3, (rows, 64), generator=g, device="cuda").to(dt)
    x[::2] *= 64
    w = torch.randint(1, 3, (2, 72, 64), generator=g, device="cuda").to(dt)
    w[:, ::2] *= -64
    x[0, 5] = math.inf
    off = offsets_of([1, rows - 1])
    _, y64, _ = product64(x, w, off, None)
    y = ops.grouped_matmul(x, w, off)
    same(y, y64, 0.0)
    assert torch.isinf(y[0]).all() and (dtype == "bf16" or torch.isinf(y[2]).any())
    dx, dw = ops.grouped_matmul_backward(y64.clamp(-64, 64).to(dt), x, w, off)
    dy = y64.clamp(-64, 64).to(dt).double()
    same(dx, product64(dy, w.transpose(1, 2), off, None)[1], 0.0)
    for e, s in enumerate((slice(0, 1), slice(1, rows))):
        same(dw[e], dy[s].T @ x[s].double(), 0.0)


def test_rows_overflow(ops):
    y = torch.full((4, 24), 60000.0, device="cuda", dtype=torch.float16)
    y[2:] = -60000
    pos = torch.tensor([[0, 1], [2, 3]], device="cuda", dtype=torch.int32)
    out = ops.combine(y, pos)
    assert (out[0] == math.inf).all() and (out[1] == -math.inf).all()
    dy, dw = ops.combine_backward(out, y, pos, torch.full((2, 2), 0.5, device="cuda"))
    assert (dy[:2] == math.inf).all() and (dy[2:] == -math.inf).all() and (dw == math.inf).all()
    d = ops.dropout(y, 0.5, 3)
    kept = d != 0
    assert kept.any() and not kept.all()
    assert torch.equal(d[kept], torch.where(y > 0, math.inf, -math.inf).half()[kept])


@pytest.mark.parametrize("start", [1, 2, 3, 4])
@pytest.mark.parametrize("rows", [3, 40, 300])
@pytest.mark.parametrize("inner,outer", [(64, 72), (33, 130), (520, 24)])
def test_weights_at_any_address(ops, inner, outer, rows, start):
    """w starts 2 to 8 bytes past a multiple of 16, NaN around it; whole numbers, exact."""
    g, E = gen(inner + start), 3
    flat = torch.full((E * outer * inner + 16,), math.nan, device="cuda", dtype=torch.bfloat16)
    w = flat[start:start + E * outer * inner].view(E, outer, inner)
    w.copy_(torch.randint(-1, 2, (E, outer, inner), generator=g, device="cuda"))
    x = torch.randint(-2, 3, (rows, inner), generator=g, device="cuda").to(torch.bfloat16)
    dy = torch.randint(-1, 2, (rows, outer), generator=g, device="cuda").to(torch.bfloat16)
    off = offsets_of([rows // 3, 0, rows - rows // 3])
    want = product64(x, w, off, None)[1].to(torch.bfloat16)
    assert torch.equal(ops.grouped_matmul(x, w, off), want)
    want = product64(dy, w.transpose(1, 2), off, None)[1].to(torch.bfloat16)
    assert torch.equal(ops.grouped_matmul_backward(dy, x, w, off, need_dw=False)[0], want)


def test_many_narrow_rows(ops):
    """As a tree's rows are: 28 features, more than 2^31 elements, experts of one matrix a leaf.
    Small whole numbers: every sum is exact."""
    n, inner, outer, E = 80_000_003, 28, 8, 3
    g = gen(71)
    ints = lambda *s: torch.randint(-2, 3, s, generator=g, device="cuda", dtype=torch.int8)  # noqa
    x, dy = ints(n, inner).to(torch.bfloat16), ints(n, outer).to(torch.bfloat16)
    w = ints(E, outer, inner).to(torch.bfloat16)
    off = torch.tensor([2, 30_000_001, 30_000_001, n - 5], device="cuda", dtype=torch.int32)
    y = ops.grouped_matmul(x, w, off)
    dx, dw = ops.grouped_matmul_backward(dy, x, w, off, grad_dtype=torch.float32)
    o = off.tolist()
    assert not y[:2].any() and not y[-5:].any() and not dx[:2].any() and not dx[-5:].any()
    for e in range(E):
        want = torch.zeros(outer, inner, device="cuda", dtype=torch.float64)
        for a in range(o[e], o[e + 1], 1 << 23):
            s = slice(a, min(a + (1 << 23), o[e + 1]))
            assert torch.equal(y[s].float(), x[s].float() @ w[e].float().T)
            assert torch.equal(dx[s].float(), dy[s].float() @ w[e].float())
            want += dy[s].double().T @ x[s].double()
        assert torch.equal(dw[e].double(), want)
    assert not dw[1].any()
