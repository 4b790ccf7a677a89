"""Calls of clip_grads and grad_norm that are refused, and what they leave behind; tensors that lie
between one another; factors near the ends of f32.

Bounds as in test_gpu_grad_clip.py."""

import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


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
