"""Expert layers on the device: rows routed to experts, products grouped by expert.

A layer of E experts works on T rows ("tokens", [T, ...] tensors). `route` picks k experts
for every token from a gate's logits (experts masked with -inf are never picked: for example
all but those of the leaf a tree sends the token to) and groups the T * k slots by expert;
`grouped_matmul` multiplies each expert's ragged range of rows by its matrix; `combine` joins
a token's k results; `dropout` regularises while training. Each has its gradient beside it.
`grouped_matmul_w4` serves a few rows from weights of 4 bits.

    r = experts.route(logits, k)                                # [T, E]
    h = experts.grouped_matmul(x, w1, r.offsets, rows=r.rows)   # x [T, K], w1 [E, H, K]
    y = experts.grouped_matmul(h, w2, r.offsets)                # w2 [E, N, H]
    out = experts.combine(y, r.position, r.weights)             # [T, N]

Inputs and results are torch tensors on one CUDA device; the work is enqueued on torch's
current stream of that device and scratch comes from torch's allocator on that stream. A
tensor whose last axis is not contiguous is copied first; any row stride is read in place.
The functions call the C ABI (lgbm_b200_experts_* in include/lgbm_b200.h) and raise
LightGBMError for arguments it would refuse; there is no CPU path.
"""

import ctypes
from collections import namedtuple

import torch

from . import _lib as C

__all__ = ["Routing", "route", "route_backward", "grouped_matmul", "grouped_matmul_backward",
           "grouped_matmul_w4", "quantize_w4", "combine", "combine_backward", "dropout", "dropout_backward", "check_errors"]

Routing = namedtuple("Routing", ["weights", "experts", "position", "rows", "offsets"])
Routing.__doc__ = """What `route` returns, M = T * k slots:
weights [T, k] f32 and experts [T, k] int32 (-1: none left to choose, weight 0);
position [T, k] int32, the slot's row among the grouped rows, a permutation of M;
rows [M] int32, the token of every grouped row; offsets [E + 1] int32, the experts' ranges
of grouped rows (rows from offsets[E] on belong to no expert)."""

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_HALVES = {torch.bfloat16: 1, torch.float16: 2}

_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)
_empty = torch.empty


def _refuse(msg, code=C.INVALID_ARGUMENT):
    raise C.LightGBMError(code, msg)


def _call(device, fn, *args):
    """One C call with `device` current and its current stream as the last argument."""
    index = device.index
    if index == torch.cuda.current_device():
        rc = fn(*args, _stream_of(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, _stream_of(index))
    if rc:
        C.check(rc)


def _rows2d(what, t, dtypes):
    """A [rows, width] tensor with a contiguous last axis, and its row pitch."""
    if t.dim() != 2 or t.dtype not in dtypes or not t.is_cuda:
        _refuse(f"{what}: want a 2-D CUDA tensor of {'/'.join(map(str, dtypes))}, got "
                f"{tuple(t.shape)} {t.dtype} on {t.device}")
    pitch, step = t.stride()
    rows, width = t.shape
    if rows <= 1:
        pitch = max(pitch, width)
    if (step != 1 and width > 1) or pitch < width:
        t = t.contiguous()
        pitch = width
    return t, max(pitch, width)


def _same(what, t, device, dtype, shape):
    """A contiguous tensor of exactly this type, shape and device."""
    if t.dtype != dtype or t.device != device or t.shape != shape:
        _refuse(f"{what}: want {tuple(shape)} {dtype} on {device}, got {tuple(t.shape)} "
                f"{t.dtype} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


def route(logits, k, normalize=True):
    """The k largest of every row of `logits` [T, E] (f32, bf16 or f16), ties to the lower
    expert, with their softmax over the chosen (normalize) or over all E, and the grouping of
    the T * k slots by expert, stable in slot order. -inf is never chosen; NaN ranks first
    and makes its token's weights NaN."""
    logits, pitch = _rows2d("route", logits, _DTYPES)
    (tokens, experts), dev, k = logits.shape, logits.device, int(k)
    if not 1 <= k <= experts:
        _refuse(f"route: k {k} of {experts} experts")
    L = C.lib()
    slots = tokens * k
    weights = _empty((tokens, k), dtype=torch.float32, device=dev)
    chosen = _empty((tokens, k), dtype=torch.int32, device=dev)
    position = _empty((tokens, k), dtype=torch.int32, device=dev)
    rows = _empty(slots, dtype=torch.int32, device=dev)
    offsets = _empty(experts + 1, dtype=torch.int32, device=dev)
    need = L.lgbm_b200_experts_route_workspace(tokens, experts, k)
    ws = _empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(dev, L.lgbm_b200_experts_route, logits.data_ptr(), _DTYPES[logits.dtype], tokens,
          experts, pitch, k, bool(normalize), weights.data_ptr(), chosen.data_ptr(),
          position.data_ptr(), rows.data_ptr(), offsets.data_ptr(),
          ws.data_ptr() if need else None, need)
    return Routing(weights, chosen, position, rows, offsets)


def route_backward(dweights, logits, routing, normalize=True):
    """Gradient of the logits from that of `routing.weights` ([T, k] f32); `routing` is what
    `route` returned for these logits and this `normalize`."""
    logits, pitch = _rows2d("route_backward", logits, _DTYPES)
    (tokens, experts), dev = logits.shape, logits.device
    k = routing.weights.shape[1]
    shape = torch.Size((tokens, k))
    dweights = _same("route_backward: dweights", dweights, dev, torch.float32, shape)
    weights = _same("route_backward: weights", routing.weights, dev, torch.float32, shape)
    chosen = _same("route_backward: experts", routing.experts, dev, torch.int32, shape)
    out = _empty((tokens, experts), dtype=logits.dtype, device=dev)
    _call(dev, C.lib().lgbm_b200_experts_route_backward, dweights.data_ptr(), weights.data_ptr(),
          chosen.data_ptr(), logits.data_ptr(), _DTYPES[logits.dtype], tokens, experts, pitch, k,
          bool(normalize), out.data_ptr())
    return out


def _weights3d(what, w, x):
    if w.dim() != 3 or w.dtype != x.dtype or w.device != x.device:
        _refuse(f"{what}: want w [experts, outer, inner] {x.dtype} on {x.device}, got "
                f"{tuple(w.shape)} {w.dtype} on {w.device}")
    return w if w.is_contiguous() else w.contiguous()


def _index(what, rows, x):
    """Grouped rows and their index tensor (None: the rows of x themselves)."""
    if rows is None:
        return x.shape[0], None
    if rows.dim() != 1:
        _refuse(f"{what}: rows has {rows.dim()} axes")
    return rows.shape[0], _same(f"{what}: rows", rows, x.device, torch.int32, rows.shape)


def _scratch(L, dev, mode, x, x_pitch, index, dy, dy_pitch, w, rows, experts, inner, outer):
    """Workspace of a product: none unless an operand has to be copied."""
    need = L.lgbm_b200_experts_matmul_workspace(mode, x, x_pitch, index, dy, dy_pitch, w, rows,
                                                experts, inner, outer)
    ws = _empty(need, dtype=torch.uint8, device=dev) if need else None
    return ws, ws.data_ptr() if need else None, need


def grouped_matmul(x, w, offsets, rows=None):
    """y[r] = w[e] x[rows[r]] for the grouped rows r of expert e, offsets[e] <= r <
    offsets[e + 1]: x [T, inner], w [E, outer, inner] (bf16 or f16), offsets [E + 1] int32,
    rows [M] int32 the row of x of every grouped row (None: x holds the grouped rows).
    Returns [M, outer]; rows of no expert are 0."""
    x, pitch = _rows2d("grouped_matmul", x, _HALVES)
    w = _weights3d("grouped_matmul", w, x)
    experts, outer, inner = w.shape
    dev = x.device
    if x.shape[1] != inner:
        _refuse(f"grouped_matmul: x is {x.shape[1]} wide, w takes {inner}", C.LENGTH_MISMATCH)
    offsets = _same("grouped_matmul: offsets", offsets, dev, torch.int32,
                    torch.Size((experts + 1,)))
    m, index = _index("grouped_matmul", rows, x)
    y = _empty((m, outer), dtype=x.dtype, device=dev)
    L = C.lib()
    xp, wp = x.data_ptr(), w.data_ptr()
    ip = None if index is None else index.data_ptr()
    ws, wsp, need = _scratch(L, dev, 0, xp, pitch, ip, None, 0, wp, m, experts, inner, outer)
    _call(dev, L.lgbm_b200_experts_matmul, xp, x.shape[0], pitch, ip, wp, offsets.data_ptr(),
          _HALVES[x.dtype], m, experts, inner, outer, y.data_ptr(), wsp, need)
    return y


def grouped_matmul_backward(dy, x, w, offsets, rows=None, grad_dtype=None, need_dx=True,
                            need_dw=True):
    """Gradients of `grouped_matmul`: (dx, dw) from dy [M, outer]. dx [M, inner] is of the
    grouped rows (with `rows`, `combine(dx, position)` sums it into the tokens); dw
    [E, outer, inner] has type `grad_dtype`: the weights' (default) or float32. One that is
    not needed is None."""
    x, x_pitch = _rows2d("grouped_matmul_backward", x, _HALVES)
    dy, dy_pitch = _rows2d("grouped_matmul_backward: dy", dy, (x.dtype,))
    w = _weights3d("grouped_matmul_backward", w, x)
    experts, outer, inner = w.shape
    dev = x.device
    m, index = _index("grouped_matmul_backward", rows, x)
    if x.shape[1] != inner or dy.shape != (m, outer) or dy.device != dev:
        _refuse(f"grouped_matmul_backward: dy {tuple(dy.shape)} on {dy.device}, x "
                f"{tuple(x.shape)}, w {tuple(w.shape)}, {m} rows", C.LENGTH_MISMATCH)
    offsets = _same("grouped_matmul_backward: offsets", offsets, dev, torch.int32,
                    torch.Size((experts + 1,)))
    grad_dtype = grad_dtype or w.dtype
    if grad_dtype not in (w.dtype, torch.float32):
        _refuse(f"grouped_matmul_backward: grad_dtype {grad_dtype}")
    L = C.lib()
    dtype = _HALVES[x.dtype]
    xp, wp, dyp, op = x.data_ptr(), w.data_ptr(), dy.data_ptr(), offsets.data_ptr()
    ip = None if index is None else index.data_ptr()
    dx = dw = None
    if need_dx:
        dx = _empty((m, inner), dtype=x.dtype, device=dev)
        ws, wsp, need = _scratch(L, dev, 1, None, 0, None, dyp, dy_pitch, wp, m, experts, inner,
                                 outer)
        _call(dev, L.lgbm_b200_experts_matmul_input_grad, dyp, dy_pitch, wp, op, dtype, m,
              experts, inner, outer, dx.data_ptr(), wsp, need)
    if need_dw:
        dw = _empty((experts, outer, inner), dtype=grad_dtype, device=dev)
        ws, wsp, need = _scratch(L, dev, 2, xp, x_pitch, ip, dyp, dy_pitch, None, m, experts,
                                 inner, outer)
        _call(dev, L.lgbm_b200_experts_matmul_weight_grad, dyp, dy_pitch, xp, x.shape[0],
              x_pitch, ip, op, dtype, _DTYPES[grad_dtype], m, experts, inner, outer,
              dw.data_ptr(), wsp, need)
    return dx, dw


def grouped_matmul_w4(x, q, scales, offsets, zeros=None, rows=None, group_size=128):
    """`grouped_matmul` with 4-bit weights, for a few rows an expert: w = scales (q - zeros)
    in groups of `group_size` (32, 64 or 128) along the inner axis. q [E, outer, stride]
    uint8 packed like a 4-bit bin row (weight 2i in the low half of byte i, stride
    ceil(inner / 2) rounded up to 16); scales [E, outer, groups] of x's type; zeros
    [E, outer, groups] uint8 (None: 8). `quantize_w4` makes them."""
    x, pitch = _rows2d("grouped_matmul_w4", x, _HALVES)
    inner, dev, size = x.shape[1], x.device, int(group_size)
    if q.dim() != 3 or scales.dim() != 3 or size not in (32, 64, 128):
        _refuse(f"grouped_matmul_w4: q {tuple(q.shape)}, scales {tuple(scales.shape)}, groups "
                f"of {group_size}")
    experts, outer, _ = q.shape
    q = _same("grouped_matmul_w4: q", q, dev, torch.uint8,
              torch.Size((experts, outer, (inner + 31) // 32 * 16)))
    shape = torch.Size((experts, outer, -(-inner // size)))
    scales = _same("grouped_matmul_w4: scales", scales, dev, x.dtype, shape)
    if zeros is not None:
        zeros = _same("grouped_matmul_w4: zeros", zeros, dev, torch.uint8, shape)
    offsets = _same("grouped_matmul_w4: offsets", offsets, dev, torch.int32,
                    torch.Size((experts + 1,)))
    m, index = _index("grouped_matmul_w4", rows, x)
    y = _empty((m, outer), dtype=x.dtype, device=dev)
    _call(dev, C.lib().lgbm_b200_experts_matmul_w4, x.data_ptr(), x.shape[0], pitch,
          None if index is None else index.data_ptr(), q.data_ptr(), scales.data_ptr(),
          None if zeros is None else zeros.data_ptr(), size, offsets.data_ptr(),
          _HALVES[x.dtype], m, experts, inner, outer, y.data_ptr())
    return y


def quantize_w4(w, group_size=128, symmetric=False):
    """(q, scales, zeros) of weights [E, outer, inner] (bf16 or f16) for `grouped_matmul_w4`,
    once, when a trained layer is laid out for serving. Each group's range, stretched to hold
    0, is divided into 15 steps; symmetric: 7 steps to its largest magnitude, zeros None."""
    if w.dim() != 3 or w.dtype not in _HALVES or group_size not in (32, 64, 128):
        _refuse(f"quantize_w4: {tuple(w.shape)} {w.dtype}, groups of {group_size}")
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
    y, pitch = _rows2d("combine", y, _DTYPES)
    dev = y.device
    if position.dim() != 2:
        _refuse(f"combine: position has {position.dim()} axes")
    position = _same("combine: position", position, dev, torch.int32, position.shape)
    tokens, k = position.shape
    if weights is not None:
        weights = _same("combine: weights", weights, dev, torch.float32, position.shape)
    out = _empty((tokens, y.shape[1]), dtype=y.dtype, device=dev)
    _call(dev, C.lib().lgbm_b200_experts_combine, y.data_ptr(), _DTYPES[y.dtype], y.shape[0],
          y.shape[1], pitch, position.data_ptr(),
          None if weights is None else weights.data_ptr(), tokens, k, out.data_ptr())
    return out


def combine_backward(dout, y, position, weights=None):
    """Gradients of `combine`: (dy, dweights) from dout [T, N]; dweights is None without
    weights. `position` must be a permutation of y's M = T * k rows, as `route` makes it."""
    y, pitch = _rows2d("combine_backward", y, _DTYPES)
    dout, dout_pitch = _rows2d("combine_backward: dout", dout, (y.dtype,))
    dev = y.device
    if position.dim() != 2:
        _refuse(f"combine_backward: position has {position.dim()} axes")
    position = _same("combine_backward: position", position, dev, torch.int32, position.shape)
    tokens, k = position.shape
    if dout.shape != (tokens, y.shape[1]) or dout.device != dev:
        _refuse(f"combine_backward: dout {tuple(dout.shape)} on {dout.device}, y "
                f"{tuple(y.shape)}, {tokens} tokens", C.LENGTH_MISMATCH)
    dw = None
    if weights is not None:
        weights = _same("combine_backward: weights", weights, dev, torch.float32, position.shape)
        dw = _empty((tokens, k), dtype=torch.float32, device=dev)
    dy = _empty(y.shape, dtype=y.dtype, device=dev)
    _call(dev, C.lib().lgbm_b200_experts_combine_backward, dout.data_ptr(), y.data_ptr(),
          _DTYPES[y.dtype], y.shape[0], y.shape[1], dout_pitch, pitch, position.data_ptr(),
          None if weights is None else weights.data_ptr(), tokens, k, dy.data_ptr(),
          None if dw is None else dw.data_ptr())
    return dy, dw


def _walk(what, t):
    """(tensor, rows, width, pitch): contiguous of any shape, or 2-D with a row pitch."""
    if t.is_contiguous():
        n = t.numel()
        return t, 1, n, n
    if t.dim() == 2 and t.stride(1) == 1 and t.stride(0) >= t.shape[1]:
        return t, t.shape[0], t.shape[1], t.stride(0)
    return _walk(what, t.contiguous())


def dropout(x, p, seed, offset=0, residual=None):
    """(residual +) x with elements dropped with probability p and the others scaled up, for
    a tensor of any shape (f32, bf16 or f16). The mask is a function of (seed, offset, the
    element's number in row-major order) and never stored; p is taken in steps of 2^-16 and
    the scale fits the rounded p exactly. `seed` and `offset` are 64-bit counters: another
    layer or step takes another offset."""
    if x.dtype not in _DTYPES or not x.is_cuda:
        _refuse(f"dropout: want a CUDA tensor of f32, bf16 or f16, got {x.dtype} on {x.device}")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        _refuse(f"dropout: p {p} is not in [0, 1]")
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        _refuse(f"dropout: seed {seed} and offset {offset} are 64-bit counters")
    dev, shape = x.device, x.shape
    out = _empty(shape, dtype=x.dtype, device=dev)
    if residual is not None and (residual.shape != shape or residual.dtype != x.dtype
                                 or residual.device != dev):
        _refuse(f"dropout: residual {tuple(residual.shape)} {residual.dtype} on "
                f"{residual.device}, x {tuple(shape)} {x.dtype} on {dev}", C.LENGTH_MISMATCH)
    x, rows, width, pitch = _walk("dropout", x)
    res_pitch, rp = 0, None
    if residual is not None:
        residual, res_rows, res_width, res_pitch = _walk("dropout", residual)
        if res_rows != rows or res_width != width:  # one of them is contiguous, the other not
            rows, width = shape
            pitch = width if x.is_contiguous() else x.stride(0)
            res_pitch = width if residual.is_contiguous() else residual.stride(0)
        rp = residual.data_ptr()
    _call(dev, C.lib().lgbm_b200_experts_dropout, x.data_ptr(), rp, _DTYPES[x.dtype], rows,
          width, pitch, res_pitch, p, seed, offset, out.data_ptr())
    return out


def dropout_backward(dout, p, seed, offset=0):
    """Gradient of x from that of `dropout`'s result with the same p, seed and offset (the
    residual's gradient is dout itself)."""
    return dropout(dout, p, seed, offset)


def check_errors():
    """Waits for the current device and raises when a bounded wait inside a product kernel
    ran out since the last check (its outputs are then incomplete)."""
    bits = ctypes.c_uint32(0)
    C.check(C.lib().lgbm_b200_experts_errors(ctypes.byref(bits)))
    if bits.value:
        _refuse(f"expert products: device error bits {bits.value:#x}", C.RUNTIME)
