"""Expert layers on the device: rows routed to experts, products grouped by expert.

A layer of E experts works on T rows ("tokens", [T, ...] tensors). `route` picks k experts
for every token from a gate's logits (experts masked with -inf are never picked: for example
all but those of the leaf a tree sends the token to) and groups the T * k slots by expert;
`grouped_matmul` multiplies each expert's ragged range of rows by its matrix; `combine` joins
a token's k results; `dropout` regularises while training. Each has its gradient beside it.
`grouped_gated` and `grouped_linear` are products with what follows them in the same pass: the
gated half of a feed-forward layer, or bias, activation and residual. `clip_grads` scales a step's
gradients to a largest norm. `grouped_matmul_w4` serves a few rows from weights of 4 bits. The trees
do not call these functions; examples/leaf_experts.py joins both.

    r = experts.route(logits, k)                                # [T, E]
    h = experts.grouped_matmul(x, w1, r.offsets, rows=r.rows)   # x [T, K], w1 [E, H, K]
    y = experts.grouped_matmul(h, w2, r.offsets)                # w2 [E, N, H]
    out = experts.combine(y, r.position, r.weights)             # [T, N]

or, with a gated layer and its gradients,

    h, pre = experts.grouped_gated(x, w1, r.offsets, rows=r.rows, save=True)  # w1 [E, 2 H, K]
    y = experts.grouped_linear(h, w2, r.offsets, bias=b2)
    dh, dw2, db2 = experts.grouped_linear_backward(dy, None, h, w2, r.offsets)
    dx, dw1 = experts.grouped_gated_backward(dh, pre, x, w1, r.offsets, rows=r.rows)
    norm = experts.clip_grads([dw1, dw2, db2], 1.0)

Inputs and results are torch tensors on one CUDA device; the work is enqueued on torch's
current stream of that device and scratch comes from torch's allocator on that stream.
Matrices of rows (x, y, dy, dh, dout, residual, logits, dropout's 2-D inputs) may have any row
stride; one whose last axis is not contiguous is copied first. Other tensors (w, bias, q, scales,
positions) are copied first when they are not contiguous as a whole: keep w as [E, outer, inner].
The products also copy, on the device, operands that the tensor cores' loads cannot walk: x read
through `rows`, and x, dy or w whose rows do not start at multiples of 16 bytes.
The functions call the C ABI (lgbm_b200_experts_* in include/lgbm_b200.h) through the
extension module built beside the library, and raise LightGBMError for arguments it refuses;
there is no CPU path. Nothing is recorded for autograd: under gradient mode an input that requires
a gradient is refused, so call under `torch.no_grad()` (or inside a `torch.autograd.Function`) and
use the gradient beside each function.

Calls return before their kernels have run. Waits inside the product kernels are bounded (two
seconds on the device): one that runs out, which no correct run does, leaves an incomplete result
and sets a bit. `check_errors` waits for the device and raises for it; call it wherever results are
taken for good, as at the end of a step that is checked or saved.
"""

from collections import namedtuple

import torch

from . import _lib as C

C.lib()  # the library first: it names what is missing
try:
    from . import _experts as _X
except ImportError as e:
    raise ImportError("lightgbm_rs_b200/_experts.so is missing or does not fit this torch; build "
                      "it with `python -m lightgbm_rs_b200.build`") from e

__all__ = ["Routing", "route", "route_backward", "grouped_matmul", "grouped_matmul_backward",
           "grouped_linear", "grouped_linear_backward", "grouped_gated", "grouped_gated_backward",
           "grouped_matmul_w4", "quantize_w4", "combine", "combine_backward", "dropout",
           "dropout_backward", "grad_norm", "clip_grads", "check_errors"]

Routing = namedtuple("Routing", ["weights", "experts", "position", "rows", "offsets"])
Routing.__doc__ = """What `route` returns, M = T * k slots:
weights [T, k] f32 and experts [T, k] int32 (-1: none left to choose, weight 0);
position [T, k] int32, the slot's row among the grouped rows, a permutation of M;
rows [M] int32, the token of every grouped row; offsets [E + 1] int32, the experts' ranges
of grouped rows (rows from offsets[E] on belong to no expert)."""

_HALVES = (torch.bfloat16, torch.float16)


def route(logits, k, normalize=True):
    """The k largest of every row of `logits` [T, E] (f32, bf16 or f16), ties to the lower
    expert, with their softmax over the chosen (normalize) or over all E, and the grouping of
    the T * k slots by expert, stable in slot order. -inf is never chosen; NaN ranks first
    and makes its token's weights NaN."""
    return Routing._make(_X.route(logits, k, normalize))


def route_backward(dweights, logits, routing, normalize=True):
    """Gradient of the logits from that of `routing.weights` ([T, k] f32); `routing` is what
    `route` returned for these logits and this `normalize`."""
    return _X.route_backward(dweights, logits, routing.weights, routing.experts, normalize)


def grouped_matmul(x, w, offsets, rows=None):
    """y[r] = w[e] x[rows[r]] for the grouped rows r of expert e, offsets[e] <= r <
    offsets[e + 1]: x [T, inner], w [E, outer, inner] (bf16 or f16), offsets [E + 1] int32,
    rows [M] int32 the row of x of every grouped row (None: x holds the grouped rows).
    Returns [M, outer]; rows of no expert are 0."""
    return _X.grouped_matmul(x, w, offsets, rows)


def grouped_matmul_backward(dy, x, w, offsets, rows=None, grad_dtype=None, need_dx=True,
                            need_dw=True):
    """Gradients of `grouped_matmul`: (dx, dw) from dy [M, outer]. dx [M, inner] is of the
    grouped rows (with `rows`, `combine(dx, position)` sums it into the tokens); dw
    [E, outer, inner] has type `grad_dtype`: the weights' (default) or float32. One that is
    not needed is None. `grouped_linear_backward` with pre None gives the same products, sums those
    of few tiles in parts (1840 rows, 20 experts of 6400 x 64, dx: 15 us instead of 44) and so
    adds in another order; here the order stays as it was. dw in float32 takes 1.2 to 1.5 times as
    long as in 16 bits."""
    wide = _wide("grouped_matmul_backward", grad_dtype, w)
    return _X.grouped_matmul_backward(dy, x, w, offsets, rows, wide, need_dx, need_dw)


_ACTS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


def _act(what, name):
    if name not in _ACTS:
        raise C.LightGBMError(C.INVALID_ARGUMENT, f"{what}: activation {name!r} is none of {_ACTS}")
    return _ACTS[name]


def _wide(what, grad_dtype, w):
    wide = grad_dtype is torch.float32
    if grad_dtype is not None and not wide and grad_dtype is not w.dtype:
        raise C.LightGBMError(C.INVALID_ARGUMENT, f"{what}: grad_dtype {grad_dtype}")
    return wide


def grouped_linear(x, w, offsets, rows=None, bias=None, activation=None, residual=None,
                   save=False):
    """act(w[e] x[rows[r]] + bias[e]) + residual[r] for the grouped rows r of expert e, in one
    pass: x, w, offsets and rows as for `grouped_matmul`, bias [E, outer], residual [M, outer] of
    their type. activation: None, "relu", "silu" or "gelu" (by the normal distribution function).
    Rows of no expert are the residual (0 without one). With save, (y, pre) for
    `grouped_linear_backward`: pre [M, outer] is what the activation was given, rounded to x's
    type (beyond f16's range an infinity), its rows padded to 32 bytes (None without an
    activation)."""
    y, pre = _X.grouped_linear(x, w, offsets, rows, bias, _act("grouped_linear", activation),
                               residual, save)
    return (y, pre) if save else y


def grouped_linear_backward(dy, pre, x, w, offsets, rows=None, activation=None, grad_dtype=None,
                            need_dx=True, need_dw=True, need_dbias=True):
    """Gradients of `grouped_linear`: (dx, dw, dbias) from dy [M, outer], with dx and dw as of
    `grouped_matmul_backward` and dbias [E, outer] of type `grad_dtype`; pre is what the call with
    save returned. The residual's gradient is dy. dx and dw are products of dy act'(pre) rounded
    to 16 bits: dw in float32 holds the sum of those without another rounding. One that is not
    needed is None. In f16 that rounding has f16's range: beyond 65504 the rows of dx and dw that a
    value enters are not finite, however dw is stored; scale the loss so that it stays below."""
    what = "grouped_linear_backward"
    return _X.grouped_linear_backward(dy, pre, x, w, offsets, rows, _act(what, activation),
                                      _wide(what, grad_dtype, w), need_dx, need_dw, need_dbias)


def grouped_gated(x, w, offsets, rows=None, activation="silu", save=False):
    """act(gate) * up for the grouped rows, [M, hidden], in one pass: gate and up are the first
    and the last `hidden` columns of `grouped_matmul` with w [E, 2 * hidden, inner]; activation as
    for `grouped_linear`. Rows of no expert are 0. With save, (h, pre) for
    `grouped_gated_backward`: pre [M, 2, hidden] is gate and up rounded to x's type, its rows
    padded to 32 bytes."""
    h, pre = _X.grouped_gated(x, w, offsets, rows, _act("grouped_gated", activation), save)
    return (h, pre) if save else h


def grouped_gated_backward(dh, pre, x, w, offsets, rows=None, activation="silu", grad_dtype=None,
                           need_dx=True, need_dw=True):
    """Gradients of `grouped_gated`: (dx, dw) from dh [M, hidden] and what the call with save
    returned, as of `grouped_linear_backward`; dw [E, 2 * hidden, inner]. In f16 that holds where
    dh up act'(gate) and dh act(gate) stay below 65504 and so did gate and up; a gate far below zero
    passes nothing, saved as -infinity or not."""
    what = "grouped_gated_backward"
    return _X.grouped_gated_backward(dh, pre, x, w, offsets, rows, _act(what, activation),
                                     _wide(what, grad_dtype, w), need_dx, need_dw)


def grouped_matmul_w4(x, q, scales, offsets, zeros=None, rows=None, group_size=128):
    """`grouped_matmul` with 4-bit weights, for a few rows an expert: w = scales (q - zeros)
    in groups of `group_size` (32, 64 or 128) along the inner axis. q [E, outer, stride]
    uint8 packed like a 4-bit bin row (weight 2i in the low half of byte i, stride
    ceil(inner / 2) rounded up to 16); scales [E, outer, groups] of x's type; zeros
    [E, outer, groups] uint8, 0 to 15: the low 4 bits are taken (None: 8).
    `quantize_w4` makes them."""
    return _X.grouped_matmul_w4(x, q, scales, offsets, zeros, rows, group_size)


@torch.no_grad()
def quantize_w4(w, group_size=128, symmetric=False):
    """(q, scales, zeros) of weights [E, outer, inner] (bf16 or f16) for `grouped_matmul_w4`,
    once, when a trained layer is laid out for serving. Each group's range, stretched to hold
    0, is divided into 15 steps; symmetric: 7 steps to its largest magnitude, zeros None."""
    if w.dim() != 3 or w.dtype not in _HALVES or group_size not in (32, 64, 128):
        raise C.LightGBMError(C.INVALID_ARGUMENT, f"quantize_w4: {tuple(w.shape)} {w.dtype}, "
                              f"groups of {group_size}")
    experts, outer, inner = w.shape
    groups = -(-inner // group_size)
    v = torch.nn.functional.pad(w.float(), (0, groups * group_size - inner))
    v = v.view(experts, outer, groups, group_size)
    if symmetric:
        scales = v.abs().amax(3) / 7
        zero = torch.full_like(scales, 8)
    else:
        low, high = v.amin(3).clamp(max=0), v.amax(3).clamp(min=0)
        scales = (high - low) / 15
        zero = torch.where(scales > 0, -low / scales, 8.0).round().clamp(0, 15)
    scales = scales.to(w.dtype)
    s = scales.float()[..., None]
    q = (torch.where(s > 0, v / s, 0.0).round() + zero[..., None]).clamp(0, 15).to(torch.uint8)
    q = q.view(experts, outer, -1)[:, :, :inner]
    q = torch.nn.functional.pad(q, (0, (inner + 31) // 32 * 32 - inner))
    q = (q[:, :, 0::2] | q[:, :, 1::2] << 4).contiguous()
    return q, scales.contiguous(), None if symmetric else zero.to(torch.uint8).contiguous()


def combine(y, position, weights=None):
    """out[t] = sum_j weights[t, j] y[position[t, j]] in f32, rounded once: y [M, N] (f32,
    bf16 or f16), position [T, k] int32, weights [T, k] f32 (None: 1, which sums the
    gradients of grouped rows into their tokens)."""
    return _X.combine(y, position, weights)


def combine_backward(dout, y, position, weights=None):
    """Gradients of `combine`: (dy, dweights) from dout [T, N]; dweights is None without
    weights. `position` must be a permutation of y's M = T * k rows, as `route` makes it."""
    return _X.combine_backward(dout, y, position, weights)


def dropout(x, p, seed, offset=0, residual=None):
    """(residual +) x with elements dropped with probability p and the others scaled up, for
    a tensor of any shape (f32, bf16 or f16). The mask is a function of (seed, offset, the
    element's number in row-major order) and never stored; p is taken in steps of 2^-16 and
    the scale fits the rounded p exactly. `seed` and `offset` are 64-bit counters: another
    layer or step takes another offset."""
    return _X.dropout(x, p, seed, offset, residual)


def dropout_backward(dout, p, seed, offset=0):
    """Gradient of x from that of `dropout`'s result with the same p, seed and offset (the
    residual's gradient is dout itself)."""
    return _X.dropout(dout, p, seed, offset, None)


def grad_norm(grads):
    """sqrt of the sum of the squares of all elements of all tensors (f32, bf16 or f16, mixed, of
    any shapes), as an f32 tensor without dimensions: right wherever f32 can hold it."""
    return _X.clip_grads(grads, None, None)


def clip_grads(grads, max_norm, out=None):
    """Scales all tensors by min(1, max_norm / grad_norm(grads)) and returns the norm from before.
    In place, or into the tensors of `out` (like grads in shapes and types). What is written must
    not overlap what another tensor reads or writes; it may lie between its elements, as columns of
    one matrix do. An infinite norm above max_norm makes the factor 0, NaN makes every result NaN:
    check the norm where gradients may not be finite."""
    return _X.clip_grads(grads, float(max_norm), out)


def check_errors():
    """Waits for the current device and raises when a bounded wait inside a product kernel
    ran out since the last check (its outputs are then incomplete)."""
    bits = _X.errors()
    if bits:
        raise C.LightGBMError(C.RUNTIME, f"expert products: device error bits {bits:#x}")
