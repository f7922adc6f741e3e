"""The block operators without a GPU: the tests' own 64-bit forms against known answers, autograd and differences,
and the refusals of the Python surface and of the C entry points (nothing is launched)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from . import blocks_plain as P


# ------------------------------------------------------- the plain forms
@pytest.mark.parametrize("key,counter,want", [
    # the known answers that come with the method's publication
    ((0, 0), (0, 0, 0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    ((0xFFFFFFFF,) * 2, (0xFFFFFFFF,) * 4, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    ((0xA4093822, 0x299F31D0), (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344),
     (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_philox_known_answers(key, counter, want):
    assert tuple(P.philox(key, counter)) == want


def test_bits16_is_philox_by_halves():
    seed, offset = 0x0123456789ABCDEF, 0xFEDCBA9876543210
    for first, n in ((0, 24), (5, 13), (8 * (1 << 33) + 3, 20)):
        got = P.bits16(seed, offset, first, n)
        for j in range(n):
            i = first + j
            blk = i // 8
            w = P.philox((seed & 0xFFFFFFFF, seed >> 32), (blk & 0xFFFFFFFF, blk >> 32, offset & 0xFFFFFFFF, offset >> 32))
            assert got[j] == (w[i % 8 // 2] >> (16 * (i % 2))) & 0xFFFF


def _leaf(*shape, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * scale).requires_grad_()


@pytest.mark.parametrize("mode", ["linear", "sigmoid"])
@pytest.mark.parametrize("H", [6, 2, 1])
def test_scan_gradients_are_autograds(mode, H):
    B, T, D = 2, 7, 6
    x, gate, h0 = _leaf(B, T, D, seed=1), _leaf(B, T, H, seed=2, scale=0.5), _leaf(B, D, seed=3)
    h, last, _, _ = P.scan(x, gate, h0, mode)
    dh, dstate = _leaf(B, T, D, seed=4).detach(), _leaf(B, D, seed=5).detach()
    want = torch.autograd.grad((h * dh).sum() + (last * dstate).sum(), (x, gate, h0))
    with torch.no_grad():
        got, _ = P.scan_backward(dh, x, gate, h, h0, dstate, mode)
    for g, w in zip(got, want):
        torch.testing.assert_close(g, w, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("activation", ["linear", "sigmoid", "silu"])
def test_norm_gradients_are_autograds(activation):
    R, D, eps = 5, 9, 1e-6
    x, z, gate = _leaf(R, D, seed=1), _leaf(R, D, seed=2), _leaf(R, D, seed=3)
    wp, wq = _leaf(D, seed=4), _leaf(D, seed=5)
    m = torch.where(torch.rand(R, D, generator=torch.Generator().manual_seed(6)) < 0.3, 0.0, 0.7).double()
    (y, u, r_z, r_y), _ = P.norm(x, z, wp, wq, gate, activation, 0.7, eps, m)
    dy, du = _leaf(R, D, seed=7).detach(), _leaf(R, D, seed=8).detach()
    want = torch.autograd.grad((y * dy).sum() + (u * du).sum(), (x, z, gate, wp, wq))
    with torch.no_grad():
        out, _ = P.norm_backward(dy, du, y, z, wp, wq, r_z, r_y, gate, activation, m)
    for g, w in zip((out["dx"], out["dz"], out["gate"], out["post"].sum(0), out["pre"].sum(0)), want):
        torch.testing.assert_close(g, w, rtol=1e-10, atol=1e-12)


def test_policy_gradient_is_differences():
    N, V = 6, 11
    z = _leaf(N, V, seed=1, scale=2.0).detach()
    t = torch.arange(N) % V
    logp = torch.log_softmax(z, 1)[torch.arange(N), t]
    old = logp - torch.tensor([0.0, 0.5, -0.5, 0.1, -0.1, 0.3]).double()
    adv = torch.tensor([1.0, 1.0, 1.0, -1.0, -1.0, -2.0]).double()
    ref = logp + _leaf(N, seed=2, scale=0.3).detach()
    mask = torch.tensor([True, True, True, True, True, False])
    args = (t, old, adv, ref, mask, 0.2, 0.28, 0.1, 1.5)
    out, _ = P.policy(z, *args)
    assert out["clipped"].tolist() == [False, True, False, False, False, False]
    step = 1e-5
    for i in range(N):
        for j in range(V):
            a, b = z.clone(), z.clone()
            a[i, j] += step
            b[i, j] -= step
            d = 1.5 * (P.policy(a, *args)[0]["loss"] - P.policy(b, *args)[0]["loss"]) / (2 * step)
            assert abs(float(d - out["dlogits"][i, j])) < 1e-8


# ------------------------------------------- refusals of the Python surface
def _fake(ms, shape, dtype="f32", dev=0):
    """An Array whose buffer is host memory: good for every check that comes before a launch."""
    from musapy_b200 import dtypes as _dt
    from musapy_b200.array import Array, contiguous_strides

    d = _dt.parse(dtype)
    n = max(1, math.prod(shape)) * d.itemsize
    return Array(torch.zeros(n, dtype=torch.uint8), shape, contiguous_strides(shape), 0, d, dev)


def test_scan_refusals(ms):
    x, g, h0 = _fake(ms, (2, 5, 6)), _fake(ms, (2, 5, 6)), _fake(ms, (2, 6))
    cases = [
        (TypeError, lambda: ms.gated_scan(np.zeros((2, 5, 6)), g)),
        (ms.ShapeError, lambda: ms.gated_scan(_fake(ms, (6,)), _fake(ms, (6,)))),
        (ms.ShapeError, lambda: ms.gated_scan(_fake(ms, (1, 2, 5, 6)), g)),
        (ms.DtypeError, lambda: ms.gated_scan(_fake(ms, (2, 5, 6), "f64"), g)),
        (ms.DtypeError, lambda: ms.gated_scan(_fake(ms, (2, 5, 6), "bf16"), _fake(ms, (2, 5, 6), "f16"))),
        (ms.DtypeError, lambda: ms.gated_scan(x, _fake(ms, (2, 5, 6), "bf16"))),
        (ms.ShapeError, lambda: ms.gated_scan(x, _fake(ms, (2, 4, 6)))),
        (ms.ShapeError, lambda: ms.gated_scan(x, _fake(ms, (2, 5, 4)))),
        (ms.ShapeError, lambda: ms.gated_scan(x, _fake(ms, (2, 5, 0)))),
        (ms.ShapeError, lambda: ms.gated_scan(x, g, _fake(ms, (2, 5)))),
        (ms.DtypeError, lambda: ms.gated_scan(x, g, _fake(ms, (2, 6), "bf16"))),
        (ms.MusapyError, lambda: ms.gated_scan(x, g, mode="tanh")),
        (ms.MusapyError, lambda: ms.gated_scan(x, g, mode=["linear"])),
        (ms.DeviceError, lambda: ms.gated_scan(x, _fake(ms, (2, 5, 6), dev=1))),
        (ms.ShapeError, lambda: ms.gated_scan(x, g, out=_fake(ms, (2, 5, 7)))),
        (ms.DtypeError, lambda: ms.gated_scan(x, g, out=_fake(ms, (2, 5, 6), "bf16"))),
        (ms.MemoryError, lambda: ms.gated_scan(x, g, out=x)),
        (ms.ShapeError, lambda: ms.gated_scan_backward(_fake(ms, (2, 5, 7)), x, g, x)),
        (ms.DtypeError, lambda: ms.gated_scan_backward(x, x, g, _fake(ms, (2, 5, 6), "f16"))),
        (ms.ShapeError, lambda: ms.gated_scan_backward(x, x, g, x, h0, _fake(ms, (6,)))),
        (ms.ShapeError, lambda: ms.gated_scan_step(h0, x, g)),
        (ms.ShapeError, lambda: ms.gated_scan_step(_fake(ms, (3, 6)), _fake(ms, (2, 6)), _fake(ms, (2, 6)))),
        (ms.DtypeError, lambda: ms.gated_scan_step(_fake(ms, (2, 6), "f16"), _fake(ms, (2, 6)), _fake(ms, (2, 6)))),
        (ms.ShapeError, lambda: ms.gated_scan_step(ms.transpose(_fake(ms, (6, 2))), _fake(ms, (2, 6)), _fake(ms, (2, 6)))),
        (ms.MemoryError, lambda: ms.gated_scan_step(h0, h0, _fake(ms, (2, 6)))),
    ]
    for err, call in cases:
        with pytest.raises(err):
            call()


def test_norm_refusals(ms):
    x, w = _fake(ms, (3, 8)), _fake(ms, (8,))
    r2 = _fake(ms, (2, 3))
    cases = [
        (TypeError, lambda: ms.rms_norm(1.0, w)),
        (ms.ShapeError, lambda: ms.rms_norm(_fake(ms, ()), w)),
        (ms.DtypeError, lambda: ms.rms_norm(_fake(ms, (3, 8), "i32"), w)),
        (ms.ShapeError, lambda: ms.rms_norm(x, _fake(ms, (7,)))),
        (ms.DtypeError, lambda: ms.rms_norm(x, _fake(ms, (8,), "bf16"))),
        (ms.ShapeError, lambda: ms.gated_residual_norm(x, _fake(ms, (3, 7)), w, w)),
        (ms.DtypeError, lambda: ms.gated_residual_norm(x, _fake(ms, (3, 8), "bf16"), w, w)),
        (ms.ShapeError, lambda: ms.gated_residual_norm(x, x, w, w, gate=_fake(ms, (3,)))),
        (ms.ShapeError, lambda: ms.gated_residual_norm(x, x, w, w, gate=_fake(ms, (1, 8)))),
        (ms.DtypeError, lambda: ms.gated_residual_norm(x, x, w, w, gate=_fake(ms, (8,), "f16"))),
        (ms.MusapyError, lambda: ms.gated_residual_norm(x, x, w, w, activation="relu")),
        (ms.MusapyError, lambda: ms.gated_residual_norm(x, x, w, w, dropout=1.5)),
        (ms.MusapyError, lambda: ms.gated_residual_norm(x, x, w, w, dropout=float("nan"))),
        (ms.MusapyError, lambda: ms.gated_residual_norm_backward(None, None, x, x, w, w, r2)),
        (ms.ShapeError, lambda: ms.gated_residual_norm_backward(x, x, x, x, w, w, _fake(ms, (3,)))),
        (TypeError, lambda: ms.gated_residual_norm_backward(x, x, x, None, w, w, r2)),
        (ms.ShapeError, lambda: ms.rms_norm_backward(x, x, w, r2)),
    ]
    for err, call in cases:
        with pytest.raises(err):
            call()


def test_dropout_and_policy_refusals(ms):
    x = _fake(ms, (4, 8))
    t, f = _fake(ms, (4,), "i64"), _fake(ms, (4,))
    cases = [
        (ms.DtypeError, lambda: ms.dropout(_fake(ms, (4,), "f64"), 0.1, 1)),
        (ms.MusapyError, lambda: ms.dropout(x, -0.1, 1)),
        (ms.MusapyError, lambda: ms.dropout(x, "0.1", 1)),
        (TypeError, lambda: ms.dropout(x, 0.1, 1.5)),
        (TypeError, lambda: ms.dropout(x, 0.1, 1, None)),
        (ms.ShapeError, lambda: ms.dropout(x, 0.1, 1, out=_fake(ms, (8, 4)))),
        (ms.MemoryError, lambda: ms.dropout(x, 0.1, 1, out=x)),
        (ms.ShapeError, lambda: ms.policy_loss(x, _fake(ms, (5,), "i64"), f, f)),
        (ms.DtypeError, lambda: ms.policy_loss(x, _fake(ms, (4,), "u8"), f, f)),
        (ms.DtypeError, lambda: ms.policy_loss(_fake(ms, (4, 8), "f64"), t, f, f)),
        (ms.ShapeError, lambda: ms.policy_loss(x, t, _fake(ms, (4, 1)), f)),
        (ms.DtypeError, lambda: ms.policy_loss(x, t, f, _fake(ms, (4,), "f16"))),
        (ms.DtypeError, lambda: ms.policy_loss(x, t, f, f, mask=f)),
        (ms.MusapyError, lambda: ms.policy_loss(x, t, f, f, kl_coef=0.1)),
        (ms.MusapyError, lambda: ms.policy_loss(x, t, f, f, clip_low=-0.1)),
        (ms.ShapeError, lambda: ms.policy_loss(_fake(ms, (4, 0)), t, f, f)),
        (ms.DeviceError, lambda: ms.policy_loss(x, _fake(ms, (4,), "i64", dev=1), f, f)),
    ]
    for err, call in cases:
        with pytest.raises(err):
            call()


# --------------------------------------------- refusals of the C entry points
def test_c_entry_points_return_status():
    """Malformed calls come back as a status with a message: null pointers, extents, types, scratch."""
    from musapy_b200._lib import MPB_ERR_DTYPE, MPB_ERR_INVALID, MPB_ERR_SCRATCH, MPB_ERR_SHAPE, MPB_OK, NATIVE, last_error

    N = NATIVE
    f32, f16, i64 = 10, 9, 4
    scan = lambda **k: N.gated_scan(*{**dict(B=2, T=3, D=4, H=4, x=16, xd=f32, xb=12, xt=4, g=16, gd=f32, gb=12, gt=4,
                                             h0=0, mode=0, h=16, s=0, sc=0, nb=0, st=0), **k}.values())
    assert scan(B=-1) == MPB_ERR_SHAPE and scan(H=3) == MPB_ERR_SHAPE and scan(H=0) == MPB_ERR_SHAPE
    assert scan(mode=7) == MPB_ERR_INVALID and scan(xd=11) == MPB_ERR_DTYPE and scan(gd=f16) == MPB_ERR_DTYPE
    assert scan(x=0) == MPB_ERR_INVALID and "null pointer" in last_error()
    assert scan(B=0, x=0) == MPB_OK and scan(D=0, H=0, x=0) == MPB_OK
    assert N.gated_scan_backward(2, 3, 4, 4, 0, 12, 4, 16, f32, 12, 4, 16, f32, 12, 4, 16, 12, 4, 0, 0, 0, 16, 16, 0, 0,
                                 0, 0) == MPB_ERR_INVALID
    assert N.gated_scan_step(2, 4, 3, 16, f32, 4, 16, f32, 3, 0, 16, 16, 0) == MPB_ERR_SHAPE

    norm = lambda **k: N.gated_residual_norm(*{**dict(R=2, D=4, dt=f32, x=16, xr=4, z=16, zr=4, g=0, gr=0, kind=0,
                                                      act=0, post=16, pre=16, scale=1.0, eps=1e-6, p=0.0, seed=0, off=0,
                                                      y=16, u=16, r=16, st=0), **k}.values())
    assert norm(R=-1) == MPB_ERR_SHAPE and norm(kind=4) == MPB_ERR_INVALID and norm(kind=1) == MPB_ERR_INVALID
    assert norm(act=3) == MPB_ERR_INVALID and norm(p=1.1) == MPB_ERR_INVALID and norm(p=math.nan) == MPB_ERR_INVALID
    assert norm(dt=i64) == MPB_ERR_DTYPE and norm(u=0) == MPB_ERR_INVALID and norm(post=0) == MPB_ERR_INVALID
    assert norm(R=0) == MPB_OK
    need = N.gated_residual_norm_scratch_bytes(100, 64, f32, 1, 0)
    assert need > 0
    back = lambda nb, dx=16: N.gated_residual_norm_backward(
        100, 64, f32, 16, 64, 16, 64, 16, 64, 16, 64, 0, 0, 0, 0, 16, 16, 16, 1.0, 0.0, 0, 0, dx, 16, 0, 16, 16, 16, nb, 0)
    assert back(need - 1) == MPB_ERR_SCRATCH and back(need, dx=0) == MPB_ERR_INVALID

    assert N.dropout(-1, 16, f32, 0.1, 0, 0, 16, 0) == MPB_ERR_SHAPE
    assert N.dropout(4, 16, i64, 0.1, 0, 0, 16, 0) == MPB_ERR_DTYPE
    assert N.dropout(4, 0, f32, 0.1, 0, 0, 16, 0) == MPB_ERR_INVALID
    assert N.dropout(4, 16, f32, 2.0, 0, 0, 16, 0) == MPB_ERR_INVALID
    assert N.dropout(0, 0, f32, 0.1, 0, 0, 0, 0) == MPB_OK

    need = N.policy_loss_scratch_bytes(4, 8, f32)
    pol = lambda **k: N.policy_loss(*{**dict(N=4, V=8, z=16, dt=f32, sr=8, t=16, tdt=i64, old=16, adv=16, ref=0, mask=0,
                                             lo=0.2, hi=0.2, kl=0.0, gs=1.0, loss=16, logp=16, klo=16, cl=16, grad=16,
                                             sc=16, nb=need, st=0), **k}.values())
    assert pol(N=-1) == MPB_ERR_SHAPE and pol(V=0) == MPB_ERR_SHAPE and pol(tdt=f32) == MPB_ERR_DTYPE
    assert pol(dt=11) == MPB_ERR_DTYPE and pol(lo=-1.0) == MPB_ERR_INVALID and pol(hi=math.nan) == MPB_ERR_INVALID
    assert pol(z=0) == MPB_ERR_INVALID and pol(loss=0) == MPB_ERR_INVALID
    if need:
        assert pol(nb=need - 1) == MPB_ERR_SCRATCH and pol(sc=0) == MPB_ERR_SCRATCH
        assert pol(sc=24) == MPB_ERR_INVALID and "aligned" in last_error()
    long_need = N.gated_scan_scratch_bytes(1, 1000, 4, 4, f32, f32, 0)
    assert long_need > 0
    assert scan(B=1, T=1000, sc=16, nb=long_need - 1) == MPB_ERR_SCRATCH and scan(B=1, T=1000, sc=24, nb=long_need) == MPB_ERR_INVALID


def test_native_bindings_check_their_arguments():
    from musapy_b200._lib import NATIVE

    with pytest.raises(TypeError):
        NATIVE.dropout(1, 2, 3)
    with pytest.raises(TypeError):
        NATIVE.gated_scan_scratch_bytes(1, 2, 3, "4", 5, 6, 7)
    with pytest.raises(OverflowError):
        NATIVE.gated_scan_scratch_bytes(1 << 70, 2, 3, 4, 5, 6, 7)
    with pytest.raises(TypeError):
        NATIVE.dropout(4, 16, 10, "p", 0, 0, 16, 0)
