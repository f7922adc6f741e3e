"""Linear attention, distillation and the embedding without a GPU: the tests' own 64-bit forms against autograd, and the
refusals of the Python surface and of the C entry points (nothing is launched)."""
import math

import numpy as np
import pytest
import torch

from . import sequence_plain as Q
from .test_blocks_cpu import _fake


def _leaf(*shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).requires_grad_()


# ------------------------------------------------------- the plain forms
@pytest.mark.parametrize("H,Hq", [(2, 2), (4, 2), (3, 1)])
@pytest.mark.parametrize("by_head", [False, True])
def test_attention_gradients_are_autograds(H, Hq, by_head):
    B, T, DK, DV = 2, 6, 3, 4
    q, k, v = _leaf(B, T, Hq, DK, seed=1), _leaf(B, T, Hq, DK, seed=2), _leaf(B, T, H, DV, seed=3)
    g, state = _leaf(*((H,) if by_head else (B, T, H)), seed=4, scale=0.5), _leaf(B, H, DK, DV, seed=5)
    o, last = Q.attention(q, k, v, g, state, 0.7)
    do, dstate = _leaf(B, T, H, DV, seed=6).detach(), _leaf(B, H, DK, DV, seed=7).detach()
    want = torch.autograd.grad((o * do).sum() + (last * dstate).sum(), (q, k, v, g, state))
    with torch.no_grad():
        got = list(Q.attention_backward(do, q, k, v, g, state, dstate, 0.7))
    if by_head:
        got[3] = got[3].sum((0, 1))
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)


def test_attention_restarts_are_sequences_alone():
    q, k, v = (_leaf(1, 9, 2, 3, seed=i).detach() for i in (1, 2, 3))
    g = -_leaf(1, 9, 2, seed=4).detach().abs()
    g[:, 4] = -math.inf
    o, last = Q.attention(q, k, v, g, None, 1.0)
    alone, s = Q.attention(q[:, 4:], k[:, 4:], v[:, 4:], g[:, 4:], _leaf(1, 2, 3, 3, seed=5).detach(), 1.0)
    assert torch.equal(o[:, 4:], alone) and torch.equal(last, s)


def test_distill_gradient_is_autograds():
    N, V, K, tau = 4, 9, 3, 1.7
    z = _leaf(N, V, seed=1)
    ids = torch.tensor([[0, 3, 8], [2, 2, 5], [1, 4, 6], [7, 0, 1]])
    t = _leaf(N, K, seed=2).detach()
    mask = torch.tensor([True, True, False, True])
    p = torch.softmax(t / tau, 1)
    kl = (p * (p.log() - torch.log_softmax(z / tau, 1).gather(1, ids))).sum(1)
    loss = tau * tau * (kl * mask).sum() / 3
    want, = torch.autograd.grad(0.5 * loss, z)
    with torch.no_grad():
        (got_loss, got_kl, got), _ = Q.distill(z, ids, t, mask, tau, 0.5)
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-14)
    torch.testing.assert_close(got_loss, loss.detach(), rtol=1e-12, atol=1e-14)
    torch.testing.assert_close(got_kl, (kl * mask).detach(), rtol=1e-12, atol=1e-14)


# ------------------------------------------- refusals of the Python surface
def test_attention_refusals(ms):
    f = lambda *shape, **k: _fake(ms, shape, **k)
    q, v, g, s = f(2, 5, 2, 8), f(2, 5, 4, 6), f(2, 5, 4), f(2, 4, 8, 6)
    fwd, bwd, step = ms.linear_attention, ms.linear_attention_backward, ms.linear_attention_step
    cases = [
        (TypeError, lambda: fwd(np.zeros((2, 5, 2, 8)), q, v, g)),
        (ms.ShapeError, lambda: fwd(f(5, 2, 8), q, v, g)),
        (ms.ShapeError, lambda: fwd(q, f(2, 5, 2, 7), v, g)),
        (ms.ShapeError, lambda: fwd(q, f(2, 5, 4, 8), v, g)),
        (ms.ShapeError, lambda: fwd(q, q, f(2, 5, 3, 6), g)),
        (ms.ShapeError, lambda: fwd(q, q, f(2, 4, 4, 6), g)),
        (ms.ShapeError, lambda: fwd(f(2, 5, 0, 8), f(2, 5, 0, 8), v, g)),
        (ms.ShapeError, lambda: fwd(f(2, 5, 2, 257), f(2, 5, 2, 257), v, g)),
        (ms.ShapeError, lambda: fwd(q, q, f(2, 5, 4, 300), g)),
        (ms.ShapeError, lambda: fwd(f(2, 5, 2, 0), f(2, 5, 2, 0), v, g)),
        (ms.DtypeError, lambda: fwd(f(2, 5, 2, 8, dtype="f64"), q, v, g)),
        (ms.DtypeError, lambda: fwd(q, q, f(2, 5, 4, 6, dtype="bf16"), g)),
        (ms.DtypeError, lambda: fwd(q, q, v, f(2, 5, 4, dtype="bf16"))),
        (ms.ShapeError, lambda: fwd(q, q, v, f(2, 5, 2))),
        (ms.ShapeError, lambda: fwd(q, q, v, f(5, 4))),
        (ms.ShapeError, lambda: fwd(q, q, v, g, f(2, 4, 6, 8))),
        (ms.DtypeError, lambda: fwd(q, q, v, g, f(2, 4, 8, 6, dtype="f16"))),
        (TypeError, lambda: fwd(q, q, v, g, scale="1")),
        (ms.DeviceError, lambda: fwd(q, q, f(2, 5, 4, 6, dev=1), g)),
        (ms.ShapeError, lambda: fwd(q, q, v, g, out=f(2, 5, 4, 7))),
        (ms.DtypeError, lambda: fwd(q, q, v, g, out=f(2, 5, 4, 6, dtype="f16"))),
        (ms.MemoryError, lambda: fwd(q, q, v, g, out=v)),
        (ms.ShapeError, lambda: bwd(f(2, 5, 4, 7), q, q, v, g)),
        (ms.DtypeError, lambda: bwd(f(2, 5, 4, 6, dtype="bf16"), q, q, v, g)),
        (ms.ShapeError, lambda: bwd(v, q, q, v, g, s, f(2, 4, 8, 7))),
        (ms.ShapeError, lambda: step(s, q, q, v, g)),
        (ms.ShapeError, lambda: step(f(2, 4, 8, 7), f(2, 2, 8), f(2, 2, 8), f(2, 4, 6), f(2, 4))),
        (ms.DtypeError, lambda: step(f(2, 4, 8, 6, dtype="bf16"), f(2, 2, 8), f(2, 2, 8), f(2, 4, 6), f(2, 4))),
        (ms.ShapeError, lambda: step(ms.permute(f(2, 4, 6, 8), (0, 1, 3, 2)),
                                     f(2, 2, 8), f(2, 2, 8), f(2, 4, 6), f(2, 4))),
        (ms.MemoryError, lambda: step(s, f(2, 2, 8), f(2, 2, 8), f(2, 4, 6), ms.reshape(s, (2, 4, 48))[:, :, 0])),
    ]
    for i, (err, call) in enumerate(cases):
        with pytest.raises(err):
            call()
            pytest.fail(f"case {i} was not refused")


def test_distill_refusals(ms):
    f = lambda *shape, **k: _fake(ms, shape, **k)
    z, ids, t = f(4, 8), f(4, 3, dtype="i64"), f(4, 3)
    cases = [
        (TypeError, lambda: ms.distill_loss(1.0, ids, t)),
        (ms.ShapeError, lambda: ms.distill_loss(f(), ids, t)),
        (ms.DtypeError, lambda: ms.distill_loss(f(4, 8, dtype="f64"), ids, t)),
        (ms.ShapeError, lambda: ms.distill_loss(z, ids, f(5, 3))),
        (ms.ShapeError, lambda: ms.distill_loss(z, ids, f(4))),
        (ms.ShapeError, lambda: ms.distill_loss(z, f(4, 2, dtype="i64"), t)),
        (ms.DtypeError, lambda: ms.distill_loss(z, f(4, 3, dtype="u8"), t)),
        (ms.DtypeError, lambda: ms.distill_loss(z, ids, f(4, 3, dtype="i32"))),
        (ms.ShapeError, lambda: ms.distill_loss(z, f(4, 1025, dtype="i64"), f(4, 1025))),
        (ms.ShapeError, lambda: ms.distill_loss(z, ids, t, f(4, 1, dtype="bool"))),
        (ms.DtypeError, lambda: ms.distill_loss(z, ids, t, f(4))),
        (ms.MusapyError, lambda: ms.distill_loss(z, ids, t, temperature=0.0)),
        (ms.MusapyError, lambda: ms.distill_loss(z, ids, t, temperature=math.nan)),
        (TypeError, lambda: ms.distill_loss(z, ids, t, temperature="warm")),
        (TypeError, lambda: ms.distill_loss(z, ids, t, grad_scale=None)),
        (ms.ShapeError, lambda: ms.distill_loss(f(4, 0), ids, t)),
        (ms.DeviceError, lambda: ms.distill_loss(z, ids, f(4, 3, dev=1))),
    ]
    for i, (err, call) in enumerate(cases):
        with pytest.raises(err):
            call()
            pytest.fail(f"case {i} was not refused")


def test_embedding_refusals(ms):
    f = lambda *shape, **k: _fake(ms, shape, **k)
    table, tokens, d = f(10, 8), f(4, dtype="i64"), f(4, 8)
    grad = ms.embedding_backward
    cases = [
        (TypeError, lambda: ms.embedding([1], tokens)),
        (ms.ShapeError, lambda: ms.embedding(f(10), tokens)),
        (ms.DtypeError, lambda: ms.embedding(f(10, 8, dtype="f64"), tokens)),
        (ms.DtypeError, lambda: ms.embedding(table, f(4))),
        (TypeError, lambda: ms.embedding(table, tokens, scale=None)),
        (ms.ShapeError, lambda: ms.embedding(table, tokens, out=f(4, 9))),
        (ms.MemoryError, lambda: ms.embedding(d, tokens, out=d)),
        (ms.DeviceError, lambda: ms.embedding(table, f(4, dtype="i64", dev=1))),
        (ms.ShapeError, lambda: grad(d, f(5, dtype="i64"), rows=10)),
        (ms.DtypeError, lambda: grad(d, f(4, dtype="i16"), rows=10)),
        (ms.DtypeError, lambda: grad(f(4, 8, dtype="i32"), tokens, rows=10)),
        (TypeError, lambda: grad(d, tokens)),
        (TypeError, lambda: grad(d, tokens, rows=2.5)),
        (ms.ShapeError, lambda: grad(d, tokens, rows=-1)),
        (ms.ShapeError, lambda: grad(d, tokens, rows=9, into=f(10, 8))),
        (ms.ShapeError, lambda: grad(d, tokens, into=f(10, 7))),
        (ms.ShapeError, lambda: grad(d, tokens, into=f(10))),
        (ms.DtypeError, lambda: grad(d, tokens, into=f(10, 8, dtype="bf16"))),
        (ms.ShapeError, lambda: grad(d, tokens, into=ms.transpose(f(8, 10)))),
        (ms.MemoryError, lambda: grad(d, tokens, into=d)),
    ]
    for i, (err, call) in enumerate(cases):
        with pytest.raises(err):
            call()
            pytest.fail(f"case {i} was not refused")


# --------------------------------------------- refusals of the C entry points
def test_c_entry_points_return_status():
    from musapy_b200._lib import MPB_ERR_DTYPE, MPB_ERR_INVALID, MPB_ERR_SCRATCH, MPB_ERR_SHAPE, MPB_OK, NATIVE as N, last_error

    f32, f16, bf16, i32, i64 = 10, 9, 12, 3, 4
    # strides of 6 channels are no multiples of 16 bytes
    need = N.linear_attention_scratch_bytes(2, 70, 4, 2, 8, 6, bf16, 0, 0, 0)
    assert N.linear_attention_scratch_bytes(2, 70, 4, 2, 8, 8, bf16, 0, 0, 1) < need
    assert need > 0 and N.linear_attention_scratch_bytes(2, 70, 4, 3, 8, 6, bf16, 0, 0, 1) == 0
    att = lambda **k: N.linear_attention(*{**dict(
        B=2, T=70, H=4, Hq=2, DK=8, DV=6, dt=bf16, q=16, a=1120, b=16, c=8, k=16, d=1120, e=16, f=8, v=16, g=1680, h=24, i=6,
        g_=16, j=280, l=4, m=1, s0=0, scale=1.0, o=16, s=0, sc=16, nb=need, st=0), **k}.values())
    assert att(B=-1) == MPB_ERR_SHAPE and att(H=5) == MPB_ERR_SHAPE and att(Hq=0) == MPB_ERR_SHAPE and att(T=-2) == MPB_ERR_SHAPE
    assert att(DK=257) == MPB_ERR_SHAPE and att(DV=0) == MPB_ERR_SHAPE and att(dt=11) == MPB_ERR_DTYPE
    assert att(T=1 << 40) == MPB_ERR_SHAPE and att(B=1 << 40) == MPB_ERR_SHAPE and "too many" in last_error()
    for x in ("q", "k", "v", "g_", "o"):
        assert att(**{x: 0}) == MPB_ERR_INVALID
    assert att(nb=need - 1) == MPB_ERR_SCRATCH and att(sc=0) == MPB_ERR_SCRATCH and att(sc=24) == MPB_ERR_INVALID
    assert att(B=0, q=0, o=0) == MPB_OK and att(T=0, q=0, o=0) == MPB_OK
    need = N.linear_attention_scratch_bytes(2, 70, 4, 2, 8, 6, f32, 1, 1, 0)
    back = lambda **k: N.linear_attention_backward(*{**dict(
        B=2, T=70, H=4, Hq=2, DK=8, DV=6, dt=f32, do=16, x=1680, y=24, z=6, q=16, a=1120, b=16, c=8, k=16, d=1120, e=16, f=8, v=16,
        g=1680, h=24, i=6, g_=16, j=0, l=0, m=1, s0=0, ds=0, scale=1.0, dq=16, dk=16, dv=16, dg=16, by=1, ds0=16, sc=16, nb=need,
        st=0), **k}.values())
    assert back(H=3) == MPB_ERR_SHAPE and back(dt=i32) == MPB_ERR_DTYPE and back(DK=1000) == MPB_ERR_SHAPE
    for x in ("do", "q", "k", "v", "g_", "dq", "dk", "dv", "dg", "ds0"):
        assert back(**{x: 0}) == MPB_ERR_INVALID
    assert back(nb=need - 1) == MPB_ERR_SCRATCH and back(sc=40) == MPB_ERR_INVALID and back(B=0, dg=0) == MPB_OK
    step = lambda **k: N.linear_attention_step(*{**dict(B=2, H=4, Hq=2, DK=8, DV=6, dt=f16, q=16, a=16, b=8, k=16, c=16, d=8, v=16,
                                                        e=24, f=6, g=16, h=4, i=1, scale=1.0, state=16, o=16, st=0), **k}.values())
    assert step(H=3) == MPB_ERR_SHAPE and step(dt=i64) == MPB_ERR_DTYPE and step(state=0) == MPB_ERR_INVALID
    assert step(state=24) == MPB_ERR_INVALID and step(o=0) == MPB_ERR_INVALID and step(B=0, o=0) == MPB_OK

    need = N.distill_loss_scratch_bytes(4)
    dis = lambda **k: N.distill_loss(*{**dict(N=4, V=8, K=2, z=16, dt=f32, sr=8, ids=16, idt=i64, t=16, tdt=bf16, mask=0, tau=1.0,
                                              gs=1.0, loss=16, kl=16, grad=16, sc=16, nb=need, st=0), **k}.values())
    assert dis(N=-1) == MPB_ERR_SHAPE and dis(V=0) == MPB_ERR_SHAPE and dis(K=1025) == MPB_ERR_SHAPE and dis(V=1 << 33) == MPB_ERR_SHAPE
    assert dis(idt=f32) == MPB_ERR_DTYPE and dis(tdt=i32) == MPB_ERR_DTYPE and dis(dt=11) == MPB_ERR_DTYPE
    assert dis(tau=0.0) == MPB_ERR_INVALID and dis(tau=math.nan) == MPB_ERR_INVALID and dis(z=0) == MPB_ERR_INVALID
    assert dis(loss=0) == MPB_ERR_INVALID and dis(t=0) == MPB_ERR_INVALID
    assert dis(nb=need - 1) == MPB_ERR_SCRATCH and dis(sc=24) == MPB_ERR_INVALID

    emb = lambda **k: N.embedding(*{**dict(N=4, V=8, D=3, t=16, dt=f32, sr=3, ids=16, idt=i32, scale=1.0, o=16, st=0), **k}.values())
    assert emb(N=-1) == MPB_ERR_SHAPE and emb(N=1 << 31) == MPB_ERR_SHAPE and emb(idt=f32) == MPB_ERR_DTYPE and emb(dt=i64) == MPB_ERR_DTYPE
    assert emb(t=0) == MPB_ERR_INVALID and emb(o=0) == MPB_ERR_INVALID and emb(N=0, ids=0) == MPB_OK and emb(D=0, o=0) == MPB_OK
    need = N.embedding_backward_scratch_bytes(200, 8, 3, 0)
    assert N.embedding_backward_scratch_bytes(200, 8, 3, 0) > N.embedding_backward_scratch_bytes(200, 8, 3, 1) > 0 and N.embedding_backward_scratch_bytes(0, 8, 3, 0) == 0
    grad = lambda **k: N.embedding_backward(*{**dict(N=200, V=8, D=3, d=16, dt=f32, sr=3, ids=16, idt=i32, scale=1.0, into=0, t=16,
                                                     sc=16, nb=need, st=0), **k}.values())
    assert grad(V=-1) == MPB_ERR_SHAPE and grad(N=1 << 31) == MPB_ERR_SHAPE and grad(V=1 << 31) == MPB_ERR_SHAPE
    assert grad(idt=bf16) == MPB_ERR_DTYPE and grad(dt=11) == MPB_ERR_DTYPE and grad(d=0) == MPB_ERR_INVALID and grad(t=0) == MPB_ERR_INVALID
    assert grad(nb=need - 1) == MPB_ERR_SCRATCH and grad(sc=0) == MPB_ERR_SCRATCH and grad(sc=8) == MPB_ERR_INVALID
    assert grad(V=0, t=0) == MPB_OK and grad(N=0, into=1) == MPB_OK


def test_native_bindings_check_their_arguments():
    from musapy_b200._lib import NATIVE

    for name in ("linear_attention", "linear_attention_backward", "linear_attention_step", "distill_loss", "embedding",
                 "embedding_backward"):
        with pytest.raises(TypeError):
            getattr(NATIVE, name)(1, 2)
    with pytest.raises(TypeError):
        NATIVE.embedding_backward_scratch_bytes(1, "2", 3, 0)
