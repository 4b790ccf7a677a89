"""Calls of clip_grads and grad_norm that are refused, and what they leave behind; tensors that lie
between one another; factors near the ends of f32.

Bounds as in test_gpu_grad_clip.py."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_experts import DTYPES, UNIT, gen  # noqa: E402
from test_gpu_grad_clip import NORM, check_scaled, norm64  # noqa: E402


@pytest.fixture(scope="module")
def ops():
    from lightgbm_rs_b200 import experts

    return experts


def zeros(*shape, dtype=torch.float32):
    return torch.zeros(*shape, device="cuda", dtype=dtype)


REFUSED = {  # name: (grads, max_norm, results or None, part of the message)
    "twice": lambda a, b: ([a, a], 1.0, None, "overlaps"),
    "overlap": lambda a, b: ([a[:50], a[49:], b], 1.0, None, "overlaps"),
    "negative": lambda a, b: ([a, b], -1.0, None, "max_norm"),
    "nan": lambda a, b: ([a, b], math.nan, None, "max_norm"),
    "last type": lambda a, b: ([a, b, zeros(3).double()], 1.0, None, "float32, bfloat16 or"),
    "last device": lambda a, b: ([a, b, zeros(3).cpu()], 1.0, None, "the first on"),
    "last grad": lambda a, b: ([a, b, zeros(3).requires_grad_()], 1.0, None, "autograd"),
    "no tensor": lambda a, b: ([a, b, 3.0], 1.0, None, "torch tensor"),
    "result's type": lambda a, b: ([zeros(100), zeros(4)], 1.0, [a, b.half()], "result 1"),
    "result's shape": lambda a, b: ([zeros(100), zeros(5)], 1.0, [a, b], "result 1"),
    "results": lambda a, b: ([zeros(100), zeros(4)], 1.0, [a], "1 results for 2"),
    "shared places": lambda a, b: ([a, b[:1].expand(7)], 1.0, None, "in one place"),
    "results overlap": lambda a, b: ([zeros(50), zeros(60)], 1.0, [a[:50], a[40:]], "overlaps"),
}


@pytest.mark.parametrize("name", REFUSED)
def test_a_refused_call_is_no_write(ops, name):
    """Neither the values nor autograd's counts of writes change, of any tensor of the call."""
    from lightgbm_rs_b200 import LightGBMError

    a = torch.full((100,), 3.0, device="cuda")
    b = torch.full((4,), 3.0, device="cuda")
    grads, most, out, message = REFUSED[name](a, b)
    held = [t for t in [a, b, *grads, *(out or [])] if isinstance(t, torch.Tensor)]
    before = [(t._version, t.detach().clone()) for t in held]
    with pytest.raises(LightGBMError, match=message):
        ops.clip_grads(grads, most, out=out)
    for t, (version, value) in zip(held, before):
        assert t._version == version and torch.equal(t.detach(), value)


def test_backward_after_a_refused_call(ops):
    """What autograd saved can still be used."""
    from lightgbm_rs_b200 import LightGBMError

    a = torch.full((4,), 2.0, device="cuda")
    x = torch.ones(4, device="cuda", requires_grad=True)
    y = (x * a).sum()
    with pytest.raises(LightGBMError):
        ops.clip_grads([a, a], 1.0)
    y.backward()
    assert x.grad.tolist() == [2.0] * 4
    y = (x * a).sum()
    ops.clip_grads([a], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_every_result_counts_as_written(ops):
    """One write each, empty tensors, copies with gaps and tensors left alone among them."""
    base = torch.ones(6, 8, device="cuda")
    grads = [torch.ones(70_000, device="cuda"), zeros(0), torch.ones(3, device="cuda").half(),
             torch.ones(5, 7, device="cuda").t()]
    for most in (1.0, 1e9):
        before = [t._version for t in grads]
        ops.clip_grads(grads, most)
        assert all(t._version > v for t, v in zip(grads, before))
    before = [t._version for t in grads] + [base._version]
    out = [torch.empty_like(t) for t in grads]
    ops.clip_grads(grads, 1.0, out=out)
    ops.grad_norm(grads + [base])
    assert [t._version for t in grads] + [base._version] == before
    assert all(t._version > 0 for t in out)


def interleaved():
    """Tensors that share memory's range and no element of it."""
    n = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    a, b, c = n(40, 12), n(1001), n(6, 8, 10).bfloat16()
    d, e = n(30, 2), torch.full((30, 4), 1.5, device="cuda").half()  # bits of f32 may be NaN in f16
    return {
        "columns": [a[:, :5], a[:, 5:]],
        "columns and rows": [a[:20, :5], a[:20, 5:], a[20:]],
        "every third": [b[::3], b[1::3], b[2::3]],
        "blocks": [c[:, :4, :5], c[:, :4, 5:], c[:, 4:, ::2], c[:, 4:, 1::2]],
        "transposed": [a.t()[:5], a.t()[5:7], a[:, 7:]],
        "many columns": list(n(70, 300).unbind(1)),
        "two types": [d.view(torch.float16)[:, 0], d.view(torch.float16)[:, 1], d[:, 1]],
        "two types of numbers": [e[:, 0], e[:, 1], e.view(torch.float32)[:, 1]],
    }


@pytest.mark.parametrize("name", ["columns", "columns and rows", "every third", "blocks",
                                  "transposed", "many columns", "two types",
                                  "two types of numbers"])
def test_tensors_between_one_another(ops, name):
    """In place and as results: what tensors of their own give, and nothing else is written."""
    torch.manual_seed(5)
    same = lambda a, b: torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))  # noqa: E731
    grads = interleaved()[name]
    copies = [t.clone() for t in grads]
    norm = ops.clip_grads(copies, 2.0)
    held = [t.clone() for t in grads]
    out = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in grads]
    assert same(ops.clip_grads(grads, 2.0, out=out), norm)
    assert all(same(a, b) for a, b in zip(grads, held))
    assert all(same(a, b) for a, b in zip(out, copies))
    results = interleaved()[name]
    assert same(ops.clip_grads(grads, 2.0, out=results), norm)
    assert all(same(a, b) for a, b in zip(results, copies))
    assert same(ops.clip_grads(grads, 2.0), norm)
    assert all(same(a, b) for a, b in zip(grads, copies))


def test_strided_overlaps_are_found(ops):
    """Random strided pieces of one buffer, of 2 and 4 bytes an element: refused when they share a
    byte, and only then."""
    import random

    from lightgbm_rs_b200 import LightGBMError

    rng = random.Random(6)
    buffer = torch.ones(4096, device="cuda")
    seen = {True: 0, False: 0}

    def piece():
        flat = buffer.view(torch.float16) if rng.random() < 0.4 else buffer
        while True:
            dims = rng.randint(1, 3)
            size = [rng.randint(1, 7) for _ in range(dims)]
            stride, reach = [], 0
            for n in size:  # every element has a place of its own
                stride.append(reach + rng.randint(1, 9))
                reach += stride[-1] * (n - 1)
            order = rng.sample(range(dims), dims)
            start = rng.randint(0, 150)
            if start + reach < flat.numel():
                return flat.as_strided([size[i] for i in order], [stride[i] for i in order], start)

    def places(t):
        at = [t.storage_offset()]
        for n, s in zip(t.shape, t.stride()):
            at = [p + s * i for p in at for i in range(n)]
        e = t.element_size()
        return {p * e + k for p in at for k in range(e)}

    for _ in range(400):
        a, b = piece(), piece()
        share = bool(places(a) & places(b))
        buffer.fill_(1)
        try:
            ops.clip_grads([a, b], math.inf)
            refused = False
        except LightGBMError as e:
            assert "overlaps" in str(e)
            refused = True
        assert refused == share, (a.shape, a.stride(), a.storage_offset(), a.dtype, b.shape,
                                  b.stride(), b.storage_offset(), b.dtype)
        seen[share] += 1
    assert min(seen.values()) > 40


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [50, 700_000])
@pytest.mark.parametrize("scale,most", [(1e38, 1e-3), (1e36, 1e-5), (1e30, 1e-20), (1e34, 1e-30),
                                        (3e37, 2e-7), (1e20, 1e-18), (1.0, 1e-39)])
def test_factors_below_f32(ops, scale, most, size, dtype):
    """max_norm / norm from 1e-38 down to 1e-65: the results have the wanted norm where the type
    holds them, and their digits."""
    dt = DTYPES[dtype]
    g = (torch.rand(size, generator=gen(8), device="cuda") * scale / size ** 0.5).to(dt)
    small = g.clone()
    small[::2] *= 1e-3
    grads = [g, small[1:]]  # one that starts off 16 bytes
    n = norm64(grads)
    out = [torch.empty_like(t) for t in grads]
    assert abs(float(ops.clip_grads(grads, most, out=out)) - n) <= NORM * n
    check_scaled(out, grads, most / n)
    ops.clip_grads(grads, most)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))
    assert abs(norm64(out) / most - 1) < UNIT[dt] + 2.0 ** -16 or most < 1e-35


def test_a_norm_at_the_end_of_f32(ops):
    """Norm and max_norm above 3.4e38, both finite."""
    top = torch.finfo(torch.float32).max
    a = torch.full((4,), top / 2, device="cuda")
    most = top * (1 - 2.0 ** -12)
    assert float(ops.clip_grads([a], most)) == top
    assert (a.double() / (top / 2) - (1 - 2.0 ** -12)).abs().max() <= 2.0 ** -22


@pytest.mark.parametrize("value,most,want", [
    (1.0, 2.0 ** -151, 0.0), (2.0 ** -149, 2.0 ** -150, 0.0), (2.0 ** -148, 2.0 ** -148, 2.0 ** -149),
    (1.0, 2.0 ** -149, 0.0), (1.0, 2.0 ** -140, 2.0 ** -141), (2.0 ** 126, 2.0 ** -148, 2.0 ** -149),
    (1.0, 1e-300, 0.0)])
def test_a_largest_norm_at_the_least_of_f32(ops, value, most, want):
    """Four equal values, so a norm of twice the value; 2^-150 rounds to the even 0."""
    a = torch.full((4,), value, device="cuda")
    assert float(ops.clip_grads([a], most)) == 2 * value
    assert a.tolist() == [want] * 4
