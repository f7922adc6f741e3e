"""Operators around a recurrent language model: linear attention with a decay for each head, distillation from a
teacher's top logits, and the embedding with its gradient. musapy has no counterpart; conventions are those of
``blocks.py``: arrays are float16, bfloat16 or float32, states, decays and the table's gradient float32, an input whose
innermost stride is not 1 is copied first, every other stride is read in place, and results are new arrays.
"""
from __future__ import annotations

import numbers
from typing import NamedTuple, Optional

from . import dtypes as _dt
from . import errors
from . import streams as _streams
from ._lib import LIB, NATIVE, check
from .array import Array
from .blocks import (_array, _carve, _dense, _element, _floats, _new, _norm_input, _of, _prod, _ptr, _rows, _scratch, _sptr,
                     _unit_inner)
from .ops import _CHECK_SCAN_STATUS, _alias, _check_out, _same_device, contiguous

_MOST_CHANNELS = 256  # of a head
_MOST_TOP = 1024  # entries of a teacher's list


def _number(name: str, what: str, v) -> float:
    if type(v) is not float and not isinstance(v, numbers.Real):
        raise TypeError(f"{name}: {what} must be a number, got {type(v).__name__}")
    return float(v)


# ------------------------------------------------------ linear attention
def _attention_inputs(name: str, q, k, v, log_decay, time: bool):
    """(q, k, v, log_decay, its strides over sequences, steps and heads, B, T, H, Hq, DK, DV, decay by head) of a call over
    time or of a step."""
    form, nd = ("(B, T, H, D)", 4) if time else ("(B, H, D)", 3)
    for what, x in (("q", q), ("k", k), ("v", v)):
        _element(name, what, x)
        if x.ndim != nd:
            raise errors.ShapeError(f"{name}: {what} must be {form}, got {list(x.shape)}")
        if x._dtype.code != q._dtype.code:
            raise errors.DtypeError(f"{name}: {what} dtype {x.dtype} != q dtype {q.dtype}")
    if k._shape != q._shape:
        raise errors.ShapeError(f"{name}: k shape {list(k.shape)} != q shape {list(q.shape)}")
    Hq, DK = q._shape[-2:]
    H, DV = v._shape[-2:]
    if v._shape[:-2] != q._shape[:-2] or Hq < 1 or H < 1 or H % Hq:
        raise errors.ShapeError(f"{name}: v shape {list(v.shape)} does not go with q {list(q.shape)}")
    if not (1 <= DK <= _MOST_CHANNELS and 1 <= DV <= _MOST_CHANNELS):
        raise errors.ShapeError(f"{name}: {DK} and {DV} channels per head (1 to {_MOST_CHANNELS})")
    B, T = q._shape[0], q._shape[1] if time else 1
    if _array(name, "log_decay", log_decay)._dtype.code != _dt.F32:
        raise errors.DtypeError(f"{name}: log_decay dtype {log_decay.dtype} != expected float32")
    by_head = log_decay._shape == (H,)
    st = log_decay._strides
    if by_head:
        gs = (0, 0, st[0])
    elif log_decay._shape == v._shape[:-1]:
        gs = st if time else (st[0], 0, st[1])
    else:
        raise errors.ShapeError(f"{name}: log_decay shape {list(log_decay.shape)} is neither {list(v.shape[:-1])} nor one per "
                                f"head {[H]}")
    return _unit_inner(q), _unit_inner(k), _unit_inner(v), gs, B, T, H, Hq, DK, DV, by_head


def _aligned(*arrays) -> int:
    """Are these 16-byte aligned, with strides that are positive multiples of 16 bytes (of the dims that have steps)?"""
    for x in arrays:
        if x._dtype.code != _dt.BF16:  # the other types' kernels do not ask
            return 0
        unit = 16 // x._dtype.itemsize - 1
        if x._ptr & 15:
            return 0
        for n, s in zip(x._shape[:-1], x._strides):
            if s & unit or (n > 1 and s <= 0):
                return 0
    return 1


def _attention_status(name: str, scratch, dev: int) -> None:
    """With ``ops.set_scan_status_check(True)`` (it synchronises): did a wait inside the kernel give up?"""
    if scratch is not None and _CHECK_SCAN_STATUS[0]:
        check(LIB.mpb_linear_attention_status(scratch.data_ptr(), _streams.current_stream(dev).cuda_stream), name)


def linear_attention(q, k, v, log_decay, state=None, scale=None, return_state=False, out=None):
    """Linear attention with a decay for each head: ``S[t] = exp(log_decay[t]) S[t-1] + k[t] v[t]'``,
    ``o[t] = scale S[t]' q[t]``.

    q and k are (B, T, Hq, DK), v is (B, T, H, DV), all in one dtype; Hq divides H, and head h has q and k of head
    h // (H / Hq). log_decay is float32, a value for every step and head (B, T, H) or one for each head (H,); below -104
    (-inf among them) it is a decay of zero, so that sequences packed along time restart there. state,
    (B, H, DK, DV) float32, is S before the first step (zero when None). scale defaults to DK^-0.5. DK and DV are at most
    256. Returns o (B, T, H, DV) in v's dtype; with ``return_state`` also the last S in float32.

    S and every sum run in float32; where the scores meet v, and the state meets q, they keep 24 bits (float32) or 16
    (float16, bfloat16). What decays leave below 2^-102 keeps fewer bits, and below 2^-126 none, as the least floats do.
    Inputs are finite: a value that is not may reach every result of its chunk of 64 steps and the later ones. A prompt may be padded behind its end with log_decay 0 and k 0, which leaves the state as it was.

    bfloat16 heads of up to 128 channels (DV a multiple of 8) in rows of 16-byte words need little memory beside their
    results; others hold the state at every 64th step meanwhile, T DK DV / 16 bytes per sequence and head."""
    name = "linear_attention"
    q, k, v, gs, B, T, H, Hq, DK, DV, _ = _attention_inputs(name, q, k, v, log_decay, True)
    scale = DK ** -0.5 if scale is None else _number(name, "scale", scale)
    ins = [q, k, v, log_decay]
    if state is not None:
        state = _floats(name, "state", state, (B, H, DK, DV))
        ins.append(state)
    dev = _same_device(name, *ins)
    if out is not None:
        _check_out(out, v._shape, v._dtype, dev, name)
        if _alias(out, *ins):
            raise errors.MemoryError("out= aliases an input buffer (AliasDetected)")
    s = _streams.current_stream(dev)
    o = out if out is not None else _new(s, v._shape, v._dtype, dev)
    last = _new(s, (B, H, DK, DV), _dt.float32, dev) if return_state else None
    if B:
        code = q._dtype.code
        nbytes = NATIVE.linear_attention_scratch_bytes(B, T, H, Hq, DK, DV, code, 0, 0,
                                                       _aligned(q, k, v) if o._ptr & 15 == 0 else 0)
        scratch = _scratch(nbytes, dev)
        check(NATIVE.linear_attention(B, T, H, Hq, DK, DV, code, q._ptr, *q._strides[:3], k._ptr, *k._strides[:3], v._ptr,
                                      *v._strides[:3], log_decay._ptr, *gs, _ptr(state), scale, o._ptr, _ptr(last),
                                      _sptr(scratch), nbytes, _streams.launch_on(s, name, *ins, o, last)), name)
        _attention_status(name, scratch, dev)
    return (o, last) if return_state else o


def linear_attention_backward(do, q, k, v, log_decay, state=None, dstate=None, scale=None):
    """Gradients of :func:`linear_attention`: ``(dq, dk, dv, dlog_decay, dstate0)`` from do, the gradient of its output,
    and dstate, that of its last state (float32, None for zero); the other arguments as the forward pass got them. dq and
    dk are summed over the heads that share one, dlog_decay, float32, has log_decay's shape (summed over sequences and
    steps where that is (H,)), dstate0 is float32. Meanwhile it holds the state and its gradient at every 64th step, T DK
    DV / 8 bytes per sequence and head (1 GB for 8 sequences of 4096 steps, 16 heads of 128), and where heads share q and k,
    dq and dk of each in float32."""
    name = "linear_attention_backward"
    q, k, v, gs, B, T, H, Hq, DK, DV, by_head = _attention_inputs(name, q, k, v, log_decay, True)
    scale = DK ** -0.5 if scale is None else _number(name, "scale", scale)
    do = _unit_inner(_of(name, "do", do, v._shape, v._dtype))
    ins = [do, q, k, v, log_decay]
    sshape = (B, H, DK, DV)
    if state is not None:
        state = _floats(name, "state", state, sshape)
        ins.append(state)
    if dstate is not None:
        dstate = _floats(name, "dstate", dstate, sshape)
        ins.append(dstate)
    dev = _same_device(name, *ins)
    s = _streams.current_stream(dev)
    dq, dk, dv = (_new(s, x._shape, x._dtype, dev) for x in (q, k, v))
    dg, dstate0 = _new(s, log_decay._shape, _dt.float32, dev), _new(s, sshape, _dt.float32, dev)
    code = q._dtype.code
    nbytes = NATIVE.linear_attention_scratch_bytes(B, T, H, Hq, DK, DV, code, 1, int(by_head),
                                                   _aligned(do, q, k, v))
    scratch = _scratch(nbytes, dev)
    check(NATIVE.linear_attention_backward(
        B, T, H, Hq, DK, DV, code, do._ptr, *do._strides[:3], q._ptr, *q._strides[:3], k._ptr, *k._strides[:3], v._ptr,
        *v._strides[:3], log_decay._ptr, *gs, _ptr(state), _ptr(dstate), scale, dq._ptr, dk._ptr, dv._ptr, dg._ptr,
        int(by_head), dstate0._ptr, _sptr(scratch), nbytes,
        _streams.launch_on(s, name, *ins, dq, dk, dv, dg, dstate0)), name)
    _attention_status(name, scratch, dev)
    return dq, dk, dv, dg, dstate0


def linear_attention_step(state, q, k, v, log_decay, scale=None, out=None):
    """One step of B running sequences: q and k (B, Hq, DK), v (B, H, DV), log_decay (B, H) or (H,). ``state``, a
    C-contiguous (B, H, DK, DV) float32 array, is updated in place; returns o (B, H, DV) in v's dtype."""
    name = "linear_attention_step"
    q, k, v, gs, B, _, H, Hq, DK, DV, _ = _attention_inputs(name, q, k, v, log_decay, False)
    scale = DK ** -0.5 if scale is None else _number(name, "scale", scale)
    _of(name, "state", state, (B, H, DK, DV), _dt.float32)
    if not _dense(state) or state._ptr % 16:
        raise errors.ShapeError(f"{name}: state must be C-contiguous on a 16-byte boundary (it is updated in place)")
    dev = _same_device(name, q, k, v, log_decay, state)
    if _alias(state, q, k, v, log_decay):
        raise errors.MemoryError("state aliases an input buffer (AliasDetected)")
    if out is not None:
        _check_out(out, v._shape, v._dtype, dev, name)
        if _alias(out, q, k, v, log_decay, state):
            raise errors.MemoryError("out= aliases an input buffer (AliasDetected)")
    s = _streams.current_stream(dev)
    o = out if out is not None else _new(s, v._shape, v._dtype, dev)
    if B:
        check(NATIVE.linear_attention_step(B, H, Hq, DK, DV, q._dtype.code, q._ptr, *q._strides[:2], k._ptr, *k._strides[:2],
                                           v._ptr, *v._strides[:2], log_decay._ptr, gs[0], gs[2], scale, state._ptr, o._ptr,
                                           _streams.launch_on(s, name, q, k, v, log_decay, state, o)), name)
    return o


# ---------------------------------------------------------- distillation
class DistillLoss(NamedTuple):
    """What :func:`distill_loss` returns: the mean loss (0-d), the divergence per token, and the logits' gradient, or
    None."""

    loss: Array
    kl: Array
    dlogits: Optional[Array]


def _indices(name: str, what: str, x, shape=None) -> Array:
    """A C-contiguous int32 or int64 array."""
    _array(name, what, x)
    if shape is not None and x._shape != shape:
        raise errors.ShapeError(f"{name}: {what} shape {list(x.shape)} != expected {list(shape)}")
    if x._dtype.code not in (_dt.I32, _dt.I64):
        raise errors.DtypeError(f"{name}: {what} dtype {x.dtype} not supported (int32, int64)")
    return x if _dense(x) else contiguous(x)


def distill_loss(logits, ids, teacher_logits, mask=None, temperature=1.0, grad=True, grad_scale=1.0):
    """Divergence of a student from a teacher known by its top logits, and with ``grad`` the gradient of grad_scale * loss
    with respect to the student's logits, in one reading of them.

    logits are (..., V); ids (int32 or int64) and teacher_logits (float16, bfloat16 or float32) are (..., K), the
    teacher's K logits and their places in the vocabulary, K at most 1024; mask (bool, None for all tokens) has the leading
    shape. With p = softmax(teacher_logits / temperature) over the K entries and q = softmax(logits / temperature) a
    token's kl is ``sum p (log p - log q[ids])``; the loss is temperature^2 times the mean of kl over the mask, 0 when
    that is empty. A place named twice has both entries' share. An entry of -inf is left out whatever its place (shorter
    lists are padded so); a token without entries adds zero. A place outside [0, V), or a NaN entry, makes its token's
    values NaN. Tokens outside the mask have zero kl and gradient whatever they hold."""
    name = "distill_loss"
    z, zr = _rows(_norm_input(name, "logits", logits))
    V, lead = z._shape[-1], z._shape[:-1]
    t = _element(name, "teacher_logits", teacher_logits)
    if t.ndim != z.ndim or t._shape[:-1] != lead:
        raise errors.ShapeError(f"{name}: teacher_logits shape {list(t.shape)} does not go with logits {list(z.shape)}")
    K = t._shape[-1]
    if K > _MOST_TOP:
        raise errors.ShapeError(f"{name}: {K} entries per token (at most {_MOST_TOP})")
    ids = _indices(name, "ids", ids, t._shape)
    t = t if _dense(t) else contiguous(t)
    temperature, grad_scale = _number(name, "temperature", temperature), _number(name, "grad_scale", grad_scale)
    if not 1e-3 <= temperature <= 1e3:
        raise errors.MusapyError(f"{name}: temperature {temperature!r} outside [0.001, 1000]")
    ins = [z, ids, t]
    if mask is not None:
        _of(name, "mask", mask, lead, _dt.bool_)
        mask = mask if _dense(mask) else contiguous(mask)
        ins.append(mask)
    N = _prod(lead)
    if N and V == 0:
        raise errors.ShapeError(f"{name}: empty vocabulary")
    dev = _same_device(name, *ins)
    s = _streams.current_stream(dev)
    nbytes = NATIVE.distill_loss_scratch_bytes(N)
    loss = _new(s, (), _dt.float32, dev)
    (kl,), scratch = _carve(s, dev, lead, nbytes, _dt.float32)
    dlogits = _new(s, z._shape, z._dtype, dev) if grad else None
    check(NATIVE.distill_loss(N, V, K, z._ptr, z._dtype.code, zr, ids._ptr, ids._dtype.code, t._ptr, t._dtype.code, _ptr(mask),
                              temperature, grad_scale, loss._ptr, kl._ptr, _ptr(dlogits), scratch, nbytes,
                              _streams.launch_on(s, name, *ins, loss, kl, dlogits)), name)
    return DistillLoss(loss, kl, dlogits)


# ------------------------------------------------------------- embedding
def embedding(table, tokens, scale=1.0, out=None):
    """Rows of ``table`` (V, D) for tokens (int32 or int64, any shape), times scale: (..., D) in the table's dtype. A token
    outside [0, V) gives a row of NaN."""
    name = "embedding"
    _element(name, "table", table)
    if table.ndim != 2:
        raise errors.ShapeError(f"{name}: table must be (V, D), got {list(table.shape)}")
    tokens = _indices(name, "tokens", tokens)
    scale = _number(name, "scale", scale)
    V, D = table._shape
    table = _unit_inner(table)
    dev = _same_device(name, table, tokens)
    shape = tokens._shape + (D,)
    if out is not None:
        _check_out(out, shape, table._dtype, dev, name)
        if _alias(out, table, tokens):
            raise errors.MemoryError("out= aliases an input buffer (AliasDetected)")
    s = _streams.current_stream(dev)
    o = out if out is not None else _new(s, shape, table._dtype, dev)
    check(NATIVE.embedding(tokens.size, V, D, table._ptr, table._dtype.code, table._strides[0], tokens._ptr,
                           tokens._dtype.code, scale, o._ptr, _streams.launch_on(s, name, table, tokens, o)), name)
    return o


def embedding_backward(dout, tokens, rows=None, scale=1.0, into=None):
    """The gradient of :func:`embedding`'s table from dout (..., D): per row scale times the sum of the dout whose token
    names it, in the order of the tokens, in float32. Tokens outside the table have no part.

    Returns a new (rows, D) array; or adds to ``into``, a C-contiguous (V, D) float32 gradient that is there already
    (a tied table's), and returns it: only the rows that are named are touched."""
    name = "embedding_backward"
    d, dr = _rows(_norm_input(name, "dout", dout))
    tokens = _indices(name, "tokens", tokens, d._shape[:-1])
    scale = _number(name, "scale", scale)
    D = d._shape[-1]
    if into is None:
        if rows is None or not isinstance(rows, numbers.Integral):
            raise TypeError(f"{name}: rows must be the table's number of rows, got {type(rows).__name__}")
        V = int(rows)
        if V < 0:
            raise errors.ShapeError(f"{name}: {V} rows")
    else:
        _array(name, "into", into)
        if into.ndim != 2 or (rows is not None and rows != into._shape[0]):
            raise errors.ShapeError(f"{name}: into shape {list(into.shape)} is not ({'V' if rows is None else rows}, {D})")
        V = into._shape[0]
        _of(name, "into", into, (V, D), _dt.float32)
        if not _dense(into):
            raise errors.ShapeError(f"{name}: into must be C-contiguous (it is added to in place)")
    dev = _same_device(name, d, tokens) if into is None else _same_device(name, d, tokens, into)
    if into is not None and _alias(into, d, tokens):
        raise errors.MemoryError("into aliases an input buffer (AliasDetected)")
    s = _streams.current_stream(dev)
    table = into if into is not None else _new(s, (V, D), _dt.float32, dev)
    N = tokens.size
    nbytes = NATIVE.embedding_backward_scratch_bytes(N, V, D, int(into is not None))
    scratch = _scratch(nbytes, dev)
    check(NATIVE.embedding_backward(N, V, D, d._ptr, d._dtype.code, dr, tokens._ptr, tokens._dtype.code, scale,
                                    int(into is not None), table._ptr, _sptr(scratch), nbytes,
                                    _streams.launch_on(s, name, d, tokens, table)), name)
    return table
