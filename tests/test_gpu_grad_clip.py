"""The norm of many gradients and their clipping, against 64 bits.

A thread adds 32 (f32) or 64 squares in two chains of f32, so a square is rounded once and added
up to 32 times: at most 34 * 2^-24 of the sum of squares, half of that of the norm; what follows
is f64. The norm's one rounding adds 2^-24. A result is a value times a factor that holds the norm's
error and a rounding, rounded twice (once to f32, once to its type).
"""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_experts import DTYPES, UNIT, gen  # noqa: E402

NORM = 17.5 * 2.0 ** -24 + 2.0 ** -24


@pytest.fixture(scope="module")
def ops():
    from lightgbm_rs_b200 import experts

    return experts


def norm64(tensors):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in tensors))


# Below a type's normal numbers a rounding is off by half its least number (f16 2^-24, bf16 2^-133,
# f32 2^-149) whatever the value, and the product's rounding to f32 by half of f32's.
LEAST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def check_scaled(got, grads, factor):
    for o, t in zip(got, grads):
        want = t.double() * factor
        lim = want.abs() * (UNIT[t.dtype] + NORM + 2.0 ** -22) + LEAST[t.dtype] + 2.0 ** -150
        assert o.dtype == t.dtype and o.shape == t.shape
        assert ((o.double() - want).abs() <= lim).all()


def tensors(sizes, kinds, seed, scale=1.0):
    g = gen(seed)
    return [(torch.randn(n, generator=g, device="cuda") * scale).to(DTYPES[kinds[i % len(kinds)]])
            for i, n in enumerate(sizes)]


SIZES = [
    [1], [0, 5, 0], [8191, 8192, 8193], [16385] * 3, [100_003], [3_000_001, 7],
    list(range(0, 70)), [17] * 1500, [1000 + 37 * i for i in range(1100)], [40_000_000],
]


@pytest.mark.parametrize("kinds", [["f32"], ["bf16"], ["f16"], ["f32", "bf16", "f16"]])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clip(ops, sizes, kinds):
    grads = tensors(sizes, kinds, len(sizes) + max(sizes))
    n = norm64(grads)
    got = ops.grad_norm(grads)
    assert got.shape == () and got.dtype is torch.float32
    assert abs(float(got) - n) <= NORM * n
    for most in (n / 3, n * 2):
        out = [torch.full_like(t, math.nan) for t in grads]
        kept = [t.clone() for t in grads]
        norm = ops.clip_grads(grads, most, out=out)
        assert torch.equal(norm, got)
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))
        if most > n:
            assert all(torch.equal(a, b) for a, b in zip(out, grads))
        else:
            check_scaled(out, grads, most / n)
        assert torch.equal(ops.clip_grads(kept, most), got)
        assert all(torch.equal(a, b) for a, b in zip(out, kept))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_tensors_at_any_address(ops, dtype):
    """One behind the other in a buffer, so that they start anywhere; results start elsewhere. What
    lies between and around them stays."""
    g, dt = gen(3), DTYPES[dtype]
    sizes = [1, 2, 3, 7, 8, 9, 31, 4097, 8189, 20_000, 16_390, 5]
    for shift in (0, 1, 3):
        src = torch.randn(sum(sizes) + 16, generator=g, device="cuda").to(dt)
        dst = torch.full((sum(sizes) + 40 + len(sizes),), 7.0, device="cuda", dtype=dt)
        grads, out, a, b = [], [], 1, shift
        for n in sizes:
            grads.append(src[a:a + n])
            out.append(dst[b:b + n])
            a, b = a + n, b + n + 1
        n = norm64(grads)
        before = src.clone()
        assert abs(float(ops.clip_grads(grads, n / 2, out=out)) - n) <= NORM * n
        check_scaled(out, grads, 0.5)
        around = torch.ones(dst.numel(), dtype=torch.bool, device="cuda")
        b = shift
        for k in sizes:
            around[b:b + k] = False
            b += k + 1
        assert (dst[around] == 7).all()
        ops.clip_grads(grads, n / 2)
        assert all(torch.equal(x, y) for x, y in zip(grads, out))
        assert torch.equal(src[:1], before[:1]) and torch.equal(src[a:], before[a:])


@pytest.mark.parametrize("scale", [1e-37, 1e-30, 1e-24, 1e-20, 1e-15, 1.0, 1e15, 1e18, 1e20, 1e30])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_squares_outside_of_f32(ops, dtype, scale):
    """Squares that overflow f32 or vanish in it, alone and beside ordinary values."""
    grads = tensors([1000, 50_001], [dtype], 5, scale)
    n = norm64(grads)
    assert abs(float(ops.grad_norm(grads)) - n) <= NORM * n + 2.0 ** -149
    both = grads + tensors([3000], [dtype], 6)
    n = norm64(both)
    assert abs(float(ops.grad_norm(both)) - n) <= NORM * n
    out = [torch.empty_like(t) for t in both]
    ops.clip_grads(both, n / 4, out=out)
    check_scaled(out, both, 0.25)


def test_norm_of_everything_the_type_holds(ops):
    big = torch.full((4,), torch.finfo(torch.float32).max / 2, device="cuda")
    assert float(ops.grad_norm([big])) == torch.finfo(torch.float32).max
    one = torch.zeros(100, device="cuda")
    one[57] = 2.0 ** -149
    assert float(ops.grad_norm([one])) == 2.0 ** -149
    assert float(ops.grad_norm([torch.zeros(10, device="cuda")])) == 0


def test_zeros_infinities_and_nan(ops):
    z = torch.zeros(100, device="cuda")
    assert float(ops.clip_grads([z], 1.0)) == 0 and not z.any()
    assert float(ops.clip_grads([z], 0.0)) == 0 and not z.any()
    a = torch.ones(5, device="cuda")
    ops.clip_grads([a], 0.0)
    assert not a.any()
    a = torch.tensor([1.0, math.inf, -2.0], device="cuda")
    assert float(ops.clip_grads([a], 1.0)) == math.inf
    assert a[[0, 2]].tolist() == [0, 0] and torch.isnan(a[1])
    a, b = torch.tensor([1.0, math.nan], device="cuda"), torch.ones(70_000, device="cuda").half()
    assert math.isnan(ops.clip_grads([a, b], 1.0))
    assert torch.isnan(a).all() and torch.isnan(b).all()
    a = torch.tensor([3.0, 4.0], device="cuda")
    assert float(ops.clip_grads([a], math.inf)) == 5 and a.tolist() == [3, 4]
    assert float(ops.clip_grads([a], 5.0)) == 5 and a.tolist() == [3, 4]
    e = torch.empty(0, 4, device="cuda")
    assert float(ops.clip_grads([e], 1.0)) == 0 and float(ops.grad_norm([e, e])) == 0


@pytest.mark.parametrize("size", [5, 300_000])
@pytest.mark.parametrize("max_norm", [1e39, 1.7e308])
def test_a_largest_norm_beyond_f32(ops, size, max_norm):
    """Finite, so above every norm of f32 but an infinite one, for which the factor is 0."""
    a = torch.full((size,), 2.0, device="cuda")
    ops.clip_grads([a], max_norm)
    assert (a == 2).all()
    a[1] = math.inf
    assert float(ops.clip_grads([a], max_norm)) == math.inf
    assert torch.isnan(a[1]) and a[0] == 0 and not a[2:].any()
    a = torch.tensor([1.0, math.inf], device="cuda")
    assert float(ops.clip_grads([a], math.inf)) == math.inf and a.tolist() == [1, math.inf]


def test_in_inference_mode(ops):
    with torch.inference_mode():
        a = torch.full((4,), 3.0, device="cuda")
        assert float(ops.clip_grads([a], 3.0)) == 6 and a.tolist() == [1.5] * 4
    with pytest.raises(Exception, match="inference"):  # as for any write outside of that mode
        ops.clip_grads([a], 1.0)
    assert a.tolist() == [1.5] * 4 and float(ops.grad_norm([a])) == 3


def test_counts_as_a_write_for_autograd(ops):
    a = torch.full((4,), 3.0, device="cuda")
    b = torch.zeros(4, device="cuda")
    before = a._version, b._version
    ops.clip_grads([a], 3.0, out=[b])
    assert (a._version, b._version > before[1]) == (before[0], True)
    ops.clip_grads([a], 3.0)
    assert a._version > before[0]


def lazy_values():
    """Tensors whose memory does not hold their values as they are."""
    z = torch.ones(4, dtype=torch.complex64, device="cuda")
    return [z.conj().imag, z[:1].conj().imag, torch.ones(3, 3, device="cuda").to_sparse()]


@pytest.mark.parametrize("i", range(3))
def test_lazy_values_are_refused(ops, i):
    from lightgbm_rs_b200 import LightGBMError

    t = lazy_values()[i]
    for call in (lambda: ops.grad_norm([t]), lambda: ops.clip_grads([t], 1.0),
                 lambda: ops.dropout(t, 0.5, 1)):
        with pytest.raises(LightGBMError, match="want tensors"):
            call()


def test_strides(ops):
    """Transposed tensors are taken as they lie; others go through a copy."""
    g = gen(9)
    base = torch.randn(60, 90, generator=g, device="cuda")
    for t in (base.t(), base[:, 5:40], base[::2], base.view(60, 9, 10).permute(2, 0, 1)[1:5]):
        kept = t.clone()
        n = norm64([t])
        assert abs(float(ops.grad_norm([t, base[:1]])) - norm64([t, base[:1]])) <= NORM * n * 2
        outside = base.clone()
        inside = torch.zeros_like(base, dtype=torch.bool)
        inside.as_strided(t.shape, t.stride(), t.storage_offset())[...] = True
        out = torch.empty(t.shape, device="cuda")
        ops.clip_grads([t], n / 2, out=[out])
        check_scaled([out], [kept], 0.5)
        wide = torch.full((*t.shape, 2), 3.0, device="cuda")
        ops.clip_grads([t], n / 2, out=[wide[..., 1]])
        assert torch.equal(wide[..., 1], out) and (wide[..., 0] == 3).all()
        version = t._version
        ops.clip_grads([t], n / 2)
        assert torch.equal(t, out) and t._version > version
        assert torch.equal(base[~inside], outside[~inside])
        base.copy_(outside)


def test_broadcast_gradient(ops):
    """An expanded gradient counts every element; it cannot be written."""
    from lightgbm_rs_b200 import LightGBMError

    t = torch.full((1,), 0.5, device="cuda").expand(64)
    assert float(ops.grad_norm([t])) == 4
    with pytest.raises(LightGBMError):
        ops.clip_grads([t], 1.0)
    out = torch.empty(64, device="cuda")
    assert float(ops.clip_grads([t], 2.0, out=[out])) == 4 and (out == 0.25).all()


def test_more_than_32_bits_of_elements(ops):
    n = (1 << 32) + 4099
    t = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    t[-4099:] = 1
    want = math.sqrt(4099)
    assert abs(float(ops.clip_grads([t], want / 2)) - want) <= NORM * want
    assert (t[-4099:] == 0.5).all() and not t[:-4099].any()


def test_same_bits_streams_and_graphs(ops):
    grads = tensors([70_001, 5, 900_000], ["f32", "bf16"], 21)
    out = [torch.empty_like(t) for t in grads]
    first = ops.clip_grads(grads, 1.0, out=out)
    kept = [t.clone() for t in out]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = ops.clip_grads(grads, 1.0, out=out)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(first, again) and all(torch.equal(a, b) for a, b in zip(out, kept))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads(grads, 1.0, out=out)
    for t in grads:
        t.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(norm, ops.grad_norm(grads)) and abs(float(norm) / float(first) - 2) < 1e-5


def refusals():
    c = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa
    a = c(100)
    return [
        lambda o: o.grad_norm([]),
        lambda o: o.grad_norm([c(3).double()]),
        lambda o: o.grad_norm([c(3).cpu()]),
        lambda o: o.grad_norm([c(3), None]),
        lambda o: o.clip_grads([c(3)], -1.0),
        lambda o: o.clip_grads([c(3)], math.nan),
        lambda o: o.clip_grads([c(3)], 1.0, out=[]),
        lambda o: o.clip_grads([c(3)], 1.0, out=[c(4)]),
        lambda o: o.clip_grads([c(3)], 1.0, out=[c(3).half()]),
        lambda o: o.clip_grads([a, a], 1.0),
        lambda o: o.clip_grads([a[:50], a[49:]], 1.0),
        lambda o: o.clip_grads([c(50), c(50)], 1.0, out=[a[:50], a[49:99]]),
        lambda o: o.clip_grads([a[:50]], 1.0, out=[a[10:60]]),
        lambda o: o.clip_grads([a[:50], a[50:]], 1.0, out=[a[50:], a[:50]]),
        lambda o: o.clip_grads([torch.zeros(3, device="cuda", requires_grad=True)], 1.0),
    ]


@pytest.mark.parametrize("i", range(15))
def test_refusals(ops, i):
    from lightgbm_rs_b200 import LightGBMError

    calls = refusals()
    assert len(calls) == 15
    with pytest.raises(LightGBMError):
        calls[i](ops)


def test_reading_the_same_tensor_twice(ops):
    a = torch.tensor([3.0, 4.0], device="cuda")
    out = [torch.empty_like(a) for _ in range(2)]
    assert abs(float(ops.clip_grads([a, a], 5.0, out=out)) - math.sqrt(50)) <= NORM * 8
    check_scaled(out, [a, a], 5 / math.sqrt(50))
    assert abs(float(ops.grad_norm([a, a, a[:1]])) - math.sqrt(59)) <= NORM * 8
