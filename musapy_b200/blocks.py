"""Operators of a recurrent block in training and serving: the gated linear recurrence, the norms around a block
fused with its gate, dropout and residual scale, dropout from a counter, and the clipped policy loss. musapy has no
counterpart; names, argument checks, streams and errors follow the operators of ``ops.py``.

Arrays are float16, bfloat16 or float32; states, norm factors, weights and per-token values are float32. An input
whose innermost stride is not 1 (or, for the row operators, whose leading dims do not form rows of one stride) is
copied first; every other stride is read in place. Results are new arrays.
"""
from __future__ import annotations

import math
import numbers
from typing import NamedTuple, Optional

import torch

from . import dtypes as _dt
from . import errors
from ._lib import LIB, NATIVE, check
from . import streams as _streams
from .array import _LAYOUTS, _TORCH_DEVICES, Array, contiguous_strides
from .ops import _CHECK_SCAN_STATUS, _alias, _check_out, _out, _same_device, _stream, contiguous, full

_MODES = {"linear": 0, "sigmoid": 1}
_ACTIVATIONS = {"linear": 0, "sigmoid": 1, "silu": 2}
_GATE_NONE, _GATE_FULL, _GATE_ROW, _GATE_CHANNEL = range(4)
_ELEMENTS = (_dt.F16, _dt.BF16, _dt.F32)
_U64 = (1 << 64) - 1
_MOST_STRIDE = 1 << 29  # elements between rows, mpb_gated_residual_norm's limit


# ---------------------------------------------------------------- checks
def _array(name: str, what: str, x) -> Array:
    if not isinstance(x, Array):
        raise TypeError(f"{name}: {what} must be a musapy Array, got {type(x).__name__}")
    return x


def _element(name: str, what: str, x) -> Array:
    if _array(name, what, x)._dtype.code not in _ELEMENTS:
        raise errors.DtypeError(f"{name}: {what} dtype {x.dtype} not supported (float16, bfloat16, float32)")
    return x


def _of(name: str, what: str, x, shape: tuple, d: _dt.Dtype) -> Array:
    """An array of exactly `shape` and `d`."""
    if _array(name, what, x)._shape != shape:
        raise errors.ShapeError(f"{name}: {what} shape {list(x.shape)} != expected {list(shape)}")
    if x._dtype.code != d.code:
        raise errors.DtypeError(f"{name}: {what} dtype {x.dtype} != expected {d}")
    return x


def _floats(name: str, what: str, x, shape: tuple) -> Array:
    """A C-contiguous float32 array of `shape`."""
    _of(name, what, x, shape, _dt.float32)
    return x if _dense(x) else contiguous(x)


def _choice(name: str, what: str, value, table: dict) -> int:
    code = table.get(value) if isinstance(value, str) else None
    if code is None:
        raise errors.MusapyError(f"{name}: {what} {value!r} is none of {', '.join(map(repr, table))}")
    return code


def _probability(name: str, p) -> float:
    if (type(p) is not float and not isinstance(p, numbers.Real)) or not 0.0 <= p <= 1.0:
        raise errors.MusapyError(f"{name}: dropout probability {p!r} outside [0, 1]")
    return float(p)


def _counter(name: str, what: str, v) -> int:
    if type(v) is not int and not isinstance(v, numbers.Integral):
        raise TypeError(f"{name}: {what} must be an integer, got {type(v).__name__}")
    return int(v) & _U64


def _ptr(x: Optional[Array]):
    return x._ptr if x is not None else None


def _scratch(nbytes: int, dev: int):
    return torch.empty(nbytes, dtype=torch.uint8, device=f"cuda:{dev}") if nbytes else None


def _sptr(scratch):
    return scratch.data_ptr() if scratch is not None else None


_empty, _U8, _new_array = torch.empty, torch.uint8, Array.__new__


def _new(s, shape: tuple, d: _dt.Dtype, dev: int) -> Array:
    """A result on the stream `s`: what ``ops._out`` makes, with the stream looked up once per operator."""
    lay, tdev = _LAYOUTS.get(shape), _TORCH_DEVICES.get(dev)
    if lay is None or tdev is None:
        return _out(shape, d, dev)
    buf = _empty(max(16, (lay[1] * d.itemsize + 15) & ~15), dtype=_U8, device=tdev)
    buf._mpb_owner = s
    a = _new_array(Array)
    a._buf, a._shape, a._strides, a._offset, a._dtype, a._dev, a._name = buf, shape, lay[0], 0, d, dev, None
    a._dev_src = a._dt_src = "input_array"
    a._ptr = a._sid = buf.data_ptr()
    return a


def _dense(x: Array) -> bool:
    """x is C-contiguous (by the cached strides of its shape where they are known)."""
    lay = _LAYOUTS.get(x._shape)
    return (lay is not None and lay[0] == x._strides) or x._is_c_contiguous()


def _carve(s, dev: int, shape: tuple, nbytes: int, *kinds):
    """Several small results of one shape and nbytes of scratch in one allocation: an Array for each dtype, and the
    scratch's address. To the alias checks each is an allocation of its own (they do not overlap)."""
    lay, tdev = _LAYOUTS.get(shape), _TORCH_DEVICES.get(dev)
    strides, n = lay if lay is not None else (contiguous_strides(shape), _prod(shape))
    total = max(nbytes, 16)
    for d in kinds:
        total += (n * d.itemsize + 15) & ~15
    if tdev is not None:
        buf = _empty(total, dtype=_U8, device=tdev)
        buf._mpb_owner = s
    else:
        buf = _new(s, (total,), _dt.uint8, dev)._buf
    base, made, at = buf.data_ptr(), [], 0
    for d in kinds:
        a = _new_array(Array)
        a._buf, a._shape, a._strides, a._offset, a._dtype, a._dev, a._name = buf, shape, strides, at // d.itemsize, d, dev, None
        a._dev_src = a._dt_src = "input_array"
        a._ptr = a._sid = base + at
        made.append(a)
        at += (n * d.itemsize + 15) & ~15
    return made, base + at


# ------------------------------------------------------------ gated scan
def _unit_inner(x: Array) -> Array:
    return x if x._strides[-1] == 1 or x._shape[-1] <= 1 else contiguous(x)


def _btd(x: Array) -> tuple:
    """Strides over sequences and steps of a (B, T, D) or (T, D) array."""
    return x._strides[:2] if len(x._shape) == 3 else (0, x._strides[0])


def _scan_inputs(name: str, x, gate, time: bool):
    """(x, gate, B, T, D, H) of a scan (time) or of a step."""
    _element(name, "x", x)
    want = (3, 2) if time else (2,)
    if x.ndim not in want:
        raise errors.ShapeError(f"{name}: x must be {'(B, T, D) or (T, D)' if time else '(B, D)'}, got {list(x.shape)}")
    _element(name, "gate", gate)
    if gate._dtype.code not in (x._dtype.code, _dt.F32):
        raise errors.DtypeError(f"{name}: gate dtype {gate.dtype} is neither x's {x.dtype} nor float32")
    D = x._shape[-1]
    if gate._shape[:-1] != x._shape[:-1] or gate.ndim != x.ndim:
        raise errors.ShapeError(f"{name}: gate shape {list(gate.shape)} does not go with x {list(x.shape)}")
    H = gate._shape[-1]
    if H != D and (H < 1 or D % H != 0):
        raise errors.ShapeError(f"{name}: {H} gates do not divide {D} channels")
    B = x._shape[0] if x.ndim == 3 or not time else 1
    T = x._shape[-2] if time else 1
    return _unit_inner(x), _unit_inner(gate), B, T, D, H


def _scan_status(name: str, scratch, dev: int) -> None:
    """With ``ops.set_scan_status_check(True)`` (it synchronises): did a wait between the pieces of a sequence give up?"""
    if scratch is not None and _CHECK_SCAN_STATUS[0]:
        check(LIB.mpb_gated_scan_status(scratch.data_ptr(), _stream(dev)), name)


def gated_scan(x, gate, h0=None, mode="linear", return_state=False, out=None):
    """Gated linear recurrence over time: ``h[t] = a[t] h[t-1] + b[t]``.

    ``mode="linear"``: a = gate, b = x; ``mode="sigmoid"``: a = sigmoid(gate), b = (1 - a) x. x is (B, T, D) or
    (T, D); gate has x's shape, or one value for the D / H channels of each of H heads: (B, T, H). It has x's dtype or
    float32. h0, (B, D) float32 ((D,) for a 2-D x), is the state before the first step (zero when None). The state
    runs in float32. Linear gates may exceed one; what shrinks below 2^-126 of itself within 128 steps may be
    lost. Returns h in x's dtype; with ``return_state`` also the last state in float32 (h0 or zeros when T is 0). A
    zero gate drops a finite state: sequences packed along time restart where it is zero."""
    name = "gated_scan"
    m = _choice(name, "mode", mode, _MODES)
    x, gate, B, T, D, H = _scan_inputs(name, x, gate, True)
    sshape = (B, D) if x.ndim == 3 else (D,)
    ins = [x, gate]
    if h0 is not None:
        h0 = _floats(name, "h0", h0, sshape)
        ins.append(h0)
    dev = _same_device(name, *ins)
    if out is not None:
        _check_out(out, x._shape, x._dtype, dev, name)
        if _alias(out, *ins):
            raise errors.MemoryError("out= aliases an input buffer (AliasDetected)")
    s = _streams.current_stream(dev)
    h = out if out is not None else _new(s, x._shape, x._dtype, dev)
    state = _new(s, sshape, _dt.float32, dev) if return_state else None
    if B * D:
        nbytes = NATIVE.gated_scan_scratch_bytes(B, T, D, H, x._dtype.code, gate._dtype.code, 0)
        scratch = _scratch(nbytes, dev)
        xb, xt = _btd(x)
        gb, gt = _btd(gate)
        check(NATIVE.gated_scan(B, T, D, H, x._ptr, x._dtype.code, xb, xt, gate._ptr, gate._dtype.code, gb, gt,
                                _ptr(h0), m, h._ptr, _ptr(state), _sptr(scratch), nbytes,
                                _streams.launch_on(s, name, *ins, h, state)), name)
        _scan_status(name, scratch, dev)
    return (h, state) if return_state else h


def gated_scan_backward(dh, x, gate, h, h0=None, dstate=None, mode="linear"):
    """Gradients of :func:`gated_scan`: ``(dx, dgate, dh0)`` from dh, the gradient of its output, and dstate, that of
    its last state (float32, None for zero). h is the output as the forward pass returned it, h0 what it started from.
    dgate has the gate's shape and dtype, summed over the channels that share it; dh0 is float32 like the state."""
    name = "gated_scan_backward"
    m = _choice(name, "mode", mode, _MODES)
    x, gate, B, T, D, H = _scan_inputs(name, x, gate, True)
    sshape = (B, D) if x.ndim == 3 else (D,)
    dh = _unit_inner(_of(name, "dh", dh, x._shape, x._dtype))
    h = _unit_inner(_of(name, "h", h, x._shape, x._dtype))
    ins = [dh, x, gate, h]
    if h0 is not None:
        h0 = _floats(name, "h0", h0, sshape)
        ins.append(h0)
    if dstate is not None:
        dstate = _floats(name, "dstate", dstate, sshape)
        ins.append(dstate)
    dev = _same_device(name, *ins)
    s = _streams.current_stream(dev)
    dx, dgate = _new(s, x._shape, x._dtype, dev), _new(s, gate._shape, gate._dtype, dev)
    dh0 = _new(s, sshape, _dt.float32, dev)
    if B * D or dgate.size:  # without channels the gates' gradients are zeros
        nbytes = NATIVE.gated_scan_scratch_bytes(B, T, D, H, x._dtype.code, gate._dtype.code, 1)
        scratch = _scratch(nbytes, dev)
        check(NATIVE.gated_scan_backward(B, T, D, H, dh._ptr, *_btd(dh), x._ptr, x._dtype.code, *_btd(x), gate._ptr,
                                         gate._dtype.code, *_btd(gate), h._ptr, *_btd(h), _ptr(h0), _ptr(dstate), m,
                                         dx._ptr, dgate._ptr, dh0._ptr, _sptr(scratch), nbytes,
                                         _streams.launch_on(s, name, *ins, dx, dgate, dh0)), name)
        _scan_status(name, scratch, dev)
    return dx, dgate, dh0


def gated_scan_step(state, x, gate, mode="linear", out=None):
    """One step of B running sequences: x (B, D), gate (B, D) or (B, H). ``state``, a C-contiguous (B, D) float32
    array, is updated in place; returns the new state in x's dtype."""
    name = "gated_scan_step"
    m = _choice(name, "mode", mode, _MODES)
    x, gate, B, _, D, H = _scan_inputs(name, x, gate, False)
    _of(name, "state", state, (B, D), _dt.float32)
    if not _dense(state):
        raise errors.ShapeError(f"{name}: state must be C-contiguous (it is updated in place)")
    dev = _same_device(name, x, gate, state)
    if _alias(state, x, gate):
        raise errors.MemoryError("state aliases an input buffer (AliasDetected)")
    if out is not None:
        _check_out(out, x._shape, x._dtype, dev, name)
        if _alias(out, x, gate, state):
            raise errors.MemoryError("out= aliases an input buffer (AliasDetected)")
    s = _streams.current_stream(dev)
    h = out if out is not None else _new(s, x._shape, x._dtype, dev)
    if B * D:
        check(NATIVE.gated_scan_step(B, D, H, x._ptr, x._dtype.code, x._strides[0], gate._ptr, gate._dtype.code,
                                     gate._strides[0], m, state._ptr, h._ptr,
                                     _streams.launch_on(s, name, x, gate, state, h)), name)
    return h


# ----------------------------------------------------------------- norms
def _rows(x: Array):
    """(array, row stride): x with unit inner stride and its leading dims as rows one stride apart; a copy of x when
    its layout is another."""
    shape, st = x._shape, x._strides
    if _dense(x):
        return x, shape[-1]
    if st[-1] == 1 or shape[-1] == 1:
        step, extent = None, None
        for n, s in zip(reversed(shape[:-1]), reversed(st[:-1])):
            if n == 1:
                continue
            if step is None:
                step, extent = s, n
            elif s == step * extent:
                extent *= n
            else:
                break
        else:
            if step is None:
                return x, 0  # one row
            if abs(step) < _MOST_STRIDE:
                return x, step
    return contiguous(x), shape[-1]


def _prod(shape) -> int:
    n = 1
    for s in shape:
        n *= s
    return n


def _vector(name: str, what: str, w, D: int) -> Array:
    return _floats(name, what, w, (D,))


def _gate(name: str, gate, x: Array):
    """(gate, kind, row stride)."""
    if gate is None:
        return None, _GATE_NONE, 0
    if _array(name, "gate", gate)._dtype.code != x._dtype.code:
        raise errors.DtypeError(f"{name}: gate dtype {gate.dtype} != x dtype {x.dtype}")
    if gate._shape == x._shape:
        g, sr = _rows(gate)
        return g, _GATE_FULL, sr
    if gate._shape == x._shape[:-1] + (1,):
        g, sr = _rows(gate)
        return g, _GATE_ROW, sr
    if gate._shape == x._shape[-1:]:
        return (gate if _dense(gate) else contiguous(gate)), _GATE_CHANNEL, 0
    raise errors.ShapeError(f"{name}: gate shape {list(gate.shape)} is neither that of x {list(x.shape)}, a value per "
                            f"row {list(x.shape[:-1]) + [1]} nor per channel {list(x.shape[-1:])}")


def _norm_input(name: str, what: str, x) -> Array:
    _element(name, what, x)
    if x.ndim < 1:
        raise errors.ShapeError(f"{name}: {what} must have at least one dim")
    return x


def rms_norm(x, weight, eps=1e-6):
    """``(u, rstd)``: u = x rstd weight over the last dim, rstd = (mean x^2 + eps)^(-1/2) in float32, of x's shape
    without its last dim. weight is (D,) float32."""
    name = "rms_norm"
    x, xr = _rows(_norm_input(name, "x", x))
    D = x._shape[-1]
    w = _vector(name, "weight", weight, D)
    dev = _same_device(name, x, w)
    s = _streams.current_stream(dev)
    lead = x._shape[:-1]
    u, rstd = _new(s, x._shape, x._dtype, dev), _new(s, lead, _dt.float32, dev)
    R = _prod(lead)
    if R * D:
        check(NATIVE.gated_residual_norm(R, D, x._dtype.code, x._ptr, xr, None, 0, None, 0, 0, 0, None, w._ptr, 1.0,
                                         float(eps), 0.0, 0, 0, None, u._ptr, rstd._ptr,
                                         _streams.launch_on(s, name, x, w, u, rstd)), name)
    elif R:  # the mean of no squares
        rstd = full(lead, math.nan, _dt.float32, dev)
    return u, rstd


def rms_norm_backward(du, x, weight, rstd, dy=None):
    """``(dx, dweight)`` of :func:`rms_norm`; dy, when given, is added to dx (the gradient that reaches x on its other
    paths)."""
    name = "rms_norm_backward"
    dx, _, _, _, dw = _norm_backward(name, dy, du, x, None, None, weight, rstd, None, "linear", 1.0, 0.0, 0, 0)
    return dx, dw


def gated_residual_norm(x, z, w_post, w_pre, gate=None, activation="linear", scale=1.0, eps=1e-6, dropout=0.0, seed=0,
                        offset=0):
    """The way from one block to the next: ``(y, u, rstd)``.

    n = rms_norm(z, w_post) of the block's result z; y = x + scale * dropout(act(gate) * n), the residual stream;
    u = rms_norm(y, w_pre), the next block's input. x and z are (..., D); gate is None, of x's shape, (..., 1) or
    (D,), in x's dtype; act is "linear", "sigmoid" or "silu". Dropout is that of :func:`dropout` over x's shape.
    rstd, (2, ...) float32, holds the two norms' factors for the backward pass."""
    name = "gated_residual_norm"
    act = _choice(name, "activation", activation, _ACTIVATIONS)
    p, seed, offset = _probability(name, dropout), _counter(name, "seed", seed), _counter(name, "offset", offset)
    x, xr = _rows(_norm_input(name, "x", x))
    z, zr = _rows(_of(name, "z", z, x._shape, x._dtype))
    D, lead = x._shape[-1], x._shape[:-1]
    post, pre = _vector(name, "w_post", w_post, D), _vector(name, "w_pre", w_pre, D)
    g, kind, gr = _gate(name, gate, x)
    ins = [x, z, post, pre] if g is None else [x, z, post, pre, g]
    dev = _same_device(name, *ins)
    s = _streams.current_stream(dev)
    y, u = _new(s, x._shape, x._dtype, dev), _new(s, x._shape, x._dtype, dev)
    rstd = _new(s, (2,) + lead, _dt.float32, dev)
    R = _prod(lead)
    if R * D:
        check(NATIVE.gated_residual_norm(R, D, x._dtype.code, x._ptr, xr, z._ptr, zr, _ptr(g), gr, kind, act, post._ptr,
                                         pre._ptr, float(scale), float(eps), p, seed, offset, y._ptr, u._ptr, rstd._ptr,
                                         _streams.launch_on(s, name, *ins, y, u, rstd)), name)
    elif R:  # the means of no squares
        rstd = full((2,) + lead, math.nan, _dt.float32, dev)
    return y, u, rstd


def gated_residual_norm_backward(dy, du, y, z, w_post, w_pre, rstd, gate=None, activation="linear", scale=1.0,
                                 dropout=0.0, seed=0, offset=0):
    """Gradients of :func:`gated_residual_norm`: ``(dx, dz, dgate, dw_post, dw_pre)`` from dy and du (either may be
    None for zero), with y and rstd as the forward pass returned them and the other arguments as it got them. dgate
    has the gate's shape (None without one); the weights' gradients are float32, summed in a fixed order."""
    return _norm_backward("gated_residual_norm_backward", dy, du, y, z, w_post, w_pre, rstd, gate, activation, scale,
                          dropout, seed, offset)


def _norm_backward(name, dy, du, y, z, w_post, w_pre, rstd, gate, activation, scale, dropout, seed, offset):
    act = _choice(name, "activation", activation, _ACTIVATIONS)
    p, seed, offset = _probability(name, dropout), _counter(name, "seed", seed), _counter(name, "offset", offset)
    y, yr = _rows(_norm_input(name, "y" if z is not None or w_post is not None else "x", y))
    D, lead = y._shape[-1], y._shape[:-1]
    R = _prod(lead)
    ins, dyr, dur, zr, post = [y], 0, 0, 0, None
    if dy is None and du is None:
        raise errors.MusapyError(f"{name}: neither dy nor du given")
    if dy is not None:
        dy, dyr = _rows(_of(name, "dy", dy, y._shape, y._dtype))
        ins.append(dy)
    if du is not None:
        du, dur = _rows(_of(name, "du", du, y._shape, y._dtype))
        ins.append(du)
    branch = w_post is not None or z is not None
    if branch:
        z, zr = _rows(_of(name, "z", z, y._shape, y._dtype))
        post = _vector(name, "w_post", w_post, D)
        ins += [z, post]
    pre = _vector(name, "w_pre" if branch else "weight", w_pre, D)
    rstd = _floats(name, "rstd", rstd, (2,) + lead if branch else lead)
    g, kind, gr = _gate(name, gate, y)
    ins += [pre, rstd] if g is None else [pre, rstd, g]
    dev = _same_device(name, *ins)
    s = _streams.current_stream(dev)
    if R * D == 0:  # nothing to read: the sums over rows or channels are zero
        zeros = lambda shape, d: full(shape, 0.0, d, dev)
        return (_new(s, y._shape, y._dtype, dev), _new(s, y._shape, y._dtype, dev) if branch else None,
                zeros(g._shape, y._dtype) if g is not None else None, zeros((D,), _dt.float32) if branch else None,
                zeros((D,), _dt.float32))
    dx = _new(s, y._shape, y._dtype, dev)
    dz = _new(s, y._shape, y._dtype, dev) if branch else None
    dpost = _new(s, (D,), _dt.float32, dev) if branch else None
    dpre = _new(s, (D,), _dt.float32, dev)
    dgate = _new(s, g._shape, y._dtype, dev) if g is not None else None
    nbytes = NATIVE.gated_residual_norm_scratch_bytes(R, D, y._dtype.code, int(branch), kind)
    scratch = _scratch(nbytes, dev)
    check(NATIVE.gated_residual_norm_backward(
        R, D, y._dtype.code, _ptr(dy), dyr, _ptr(du), dur, y._ptr, yr, _ptr(z), zr, _ptr(g), gr, kind, act, _ptr(post),
        pre._ptr, rstd._ptr, float(scale), p, seed, offset, dx._ptr, _ptr(dz), _ptr(dgate), _ptr(dpost), dpre._ptr, _sptr(scratch), nbytes,
        _streams.launch_on(s, name, *ins, dx, dz, dgate, dpost, dpre)), name)
    return dx, dz, dgate, dpost, dpre


# --------------------------------------------------------------- dropout
def dropout(x, p, seed, offset=0, out=None):
    """x with each element dropped with probability p and the others scaled to keep the mean. The mask is never stored:
    it follows from seed, offset (two 64-bit integers; take another offset for every use) and the element's index in C
    order, so the gradient is the same call on the gradient. p acts in steps of 2^-16. A dropped element is 0 whatever
    it holds."""
    name = "dropout"
    _element(name, "x", x)
    p, seed, offset = _probability(name, p), _counter(name, "seed", seed), _counter(name, "offset", offset)
    dev = x._dev
    if out is not None:
        _check_out(out, x._shape, x._dtype, dev, name)
        if _alias(out, x):
            raise errors.MemoryError("out= aliases an input buffer (AliasDetected)")
    src = x if _dense(x) else contiguous(x)
    s = _streams.current_stream(dev)
    y = out if out is not None else _new(s, x._shape, x._dtype, dev)
    check(NATIVE.dropout(src.size, src._ptr, src._dtype.code, p, seed, offset, y._ptr, _streams.launch_on(s, name, src, y)), name)
    return y


# ----------------------------------------------------------- policy loss
class PolicyLoss(NamedTuple):
    """What :func:`policy_loss` returns: the mean loss (0-d), and per token the log-probability of its target, the KL
    estimate and whether the ratio was clipped; the logits' gradient, or None."""

    loss: Array
    logp: Array
    kl: Array
    clipped: Array
    dlogits: Optional[Array]


def policy_loss(logits, targets, old_logp, advantages, ref_logp=None, mask=None, clip_low=0.2, clip_high=None,
                kl_coef=0.0, grad=True, grad_scale=1.0):
    """Clipped policy loss with a KL term, and with ``grad`` the gradient of grad_scale * loss with respect to the
    logits, in one reading of them.

    logits are (..., V); targets (int32 or int64), old_logp, advantages, ref_logp (float32) and mask (bool, None for
    all tokens) have the leading shape. With rho = exp(logp - old_logp) a token adds
    ``-min(rho A, clip(rho, 1 - clip_low, 1 + clip_high) A) + kl_coef (exp(q) - q - 1)``, q = ref_logp - logp (no KL
    term without ref_logp, nor with kl_coef 0, where kl is still returned); the loss is the mean over the mask, 0 when
    it is empty. clip_high defaults to clip_low. Tokens outside the mask have zero gradient, logp and kl whatever they
    hold; a target outside [0, V) makes its token's values NaN."""
    name = "policy_loss"
    z, zr = _rows(_norm_input(name, "logits", logits))
    V, lead = z._shape[-1], z._shape[:-1]
    _array(name, "targets", targets)
    if targets._shape != lead:
        raise errors.ShapeError(f"{name}: targets shape {list(targets.shape)} != expected {list(lead)}")
    if targets._dtype.code not in (_dt.I32, _dt.I64):
        raise errors.DtypeError(f"{name}: targets dtype {targets.dtype} not supported (int32, int64)")
    targets = targets if _dense(targets) else contiguous(targets)
    old, adv = _floats(name, "old_logp", old_logp, lead), _floats(name, "advantages", advantages, lead)
    ins = [z, targets, old, adv]
    if ref_logp is not None:
        ref_logp = _floats(name, "ref_logp", ref_logp, lead)
        ins.append(ref_logp)
    elif kl_coef:
        raise errors.MusapyError(f"{name}: kl_coef {kl_coef!r} without ref_logp")
    if mask is not None:
        _of(name, "mask", mask, lead, _dt.bool_)
        mask = mask if _dense(mask) else contiguous(mask)
        ins.append(mask)
    if clip_high is None:
        clip_high = clip_low
    if not (clip_low >= 0.0 and clip_high >= 0.0):
        raise errors.MusapyError(f"{name}: negative clip range ({clip_low!r}, {clip_high!r})")
    N = _prod(lead)
    if N and V == 0:
        raise errors.ShapeError(f"{name}: empty vocabulary")
    dev = _same_device(name, *ins)
    s = _streams.current_stream(dev)
    nbytes = NATIVE.policy_loss_scratch_bytes(N, V, z._dtype.code)
    loss = _new(s, (), _dt.float32, dev)  # alone: programs keep it for longer than the tokens' results
    (logp, kl, clipped), scratch = _carve(s, dev, lead, nbytes, _dt.float32, _dt.float32, _dt.bool_)
    dlogits = _new(s, z._shape, z._dtype, dev) if grad else None
    check(NATIVE.policy_loss(N, V, z._ptr, z._dtype.code, zr, targets._ptr, targets._dtype.code, old._ptr, adv._ptr,
                             _ptr(ref_logp), _ptr(mask), float(clip_low), float(clip_high), float(kl_coef),
                             float(grad_scale), loss._ptr, logp._ptr, kl._ptr, clipped._ptr, _ptr(dlogits),
                             scratch, nbytes, _streams.launch_on(s, name, *ins, loss, logp, dlogits)), name)
    return PolicyLoss(loss, logp, kl, clipped, dlogits)
