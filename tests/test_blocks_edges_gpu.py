"""The block operators at the edges of their ranges on the GPU, against their formulas in 64 bits: results without
elements to sum, factors of zero beside exponentials that overflow, products of gates that leave the float range,
saturated gates, and what a result keeps alive. Tolerances are the bounds that blocks_plain derives."""
import math

import pytest
import torch

from . import blocks_plain as P
from .test_blocks_gpu import TORCH, check_scan, gates, make_policy, rand

pytestmark = pytest.mark.gpu


def used_memory():
    """Leaves ones in the allocator's small free blocks, so that a result nobody writes is not zero by chance."""
    held = [torch.ones(64, device="cuda") for _ in range(32)]
    torch.cuda.synchronize()
    del held


# ------------------------------------------------------------ no elements
@pytest.mark.parametrize("mode", ["linear", "sigmoid"])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_gates_of_no_channels_have_zero_gradients(ms, dtype, mode):
    """D = 0 with H gates: a gate's gradient is a sum over no channels."""
    A = ms.from_torch
    x, gate = rand(2, 5, 0, seed=1, dtype=dtype), rand(2, 5, 3, seed=2, dtype=dtype)
    used_memory()
    h = ms.gated_scan(A(x), A(gate), mode=mode)
    dx, dgate, dh0 = ms.gated_scan_backward(A(x), A(x), A(gate), h, mode=mode)
    assert h.shape == dx.shape == (2, 5, 0) and dh0.shape == (2, 0) and dgate.shape == (2, 5, 3)
    assert torch.equal(dgate.torch(), torch.zeros_like(gate))


def test_gates_of_no_channels_at_the_c_entry(ms):
    from musapy_b200._lib import MPB_ERR_INVALID, MPB_OK, NATIVE

    dgate = torch.ones(2 * 5 * 3, device="cuda")
    call = lambda to: NATIVE.gated_scan_backward(2, 5, 0, 3, 0, 0, 0, 0, 10, 0, 0, 0, 10, 15, 3, 0, 0, 0, 0, 0, 0, 0, to, 0, 0,
                                                 0, torch.cuda.current_stream().cuda_stream)
    assert call(dgate.data_ptr()) == MPB_OK
    assert not bool(dgate.any())
    assert call(0) == MPB_ERR_INVALID


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_factors_of_rows_without_channels(ms, dtype):
    """The mean of no squares is NaN, as ms.mean's is, not what the memory held."""
    A = ms.from_torch
    e, w = rand(40, 0, seed=1, dtype=dtype), rand(0, seed=1)
    used_memory()
    _, rstd = ms.rms_norm(A(e), A(w))
    assert rstd.shape == (40,) and bool(rstd.torch().isnan().all())
    used_memory()
    _, _, rstd = ms.gated_residual_norm(A(e), A(e), A(w), A(w))
    assert rstd.shape == (2, 40) and bool(rstd.torch().isnan().all())


def test_rows_without_channels_at_the_c_entry(ms):
    from musapy_b200._lib import MPB_OK, NATIVE

    s = torch.cuda.current_stream().cuda_stream
    rstd = torch.ones(2 * 7, device="cuda")
    assert NATIVE.gated_residual_norm(7, 0, 10, 16, 0, 16, 0, 0, 0, 0, 0, 16, 16, 1.0, 1e-6, 0.0, 0, 0, 16, 16,
                                      rstd.data_ptr(), s) == MPB_OK
    assert bool(rstd.isnan().all())
    rstd = torch.ones(2 * 7, device="cuda")  # the plain norm has one factor per row
    assert NATIVE.gated_residual_norm(7, 0, 10, 16, 0, 0, 0, 0, 0, 0, 0, 0, 16, 1.0, 1e-6, 0.0, 0, 0, 0, 16,
                                      rstd.data_ptr(), s) == MPB_OK
    assert bool(rstd[:7].isnan().all()) and bool((rstd[7:] == 1).all())
    dgate = torch.ones(7, device="cuda")  # a gate per row: a sum over no channels
    assert NATIVE.gated_residual_norm_backward(7, 0, 10, 16, 0, 16, 0, 16, 0, 16, 0, 16, 1, 2, 0, 16, 16, 16, 1.0, 0.0, 0, 0,
                                               16, 16, dgate.data_ptr(), 16, 16, 0, 0, s) == MPB_OK
    assert not bool(dgate.any())


# ------------------------------------------- zero times an exponential
@pytest.mark.parametrize("layout", ["aligned", "apart"])
@pytest.mark.parametrize("V", [40, 5000])
def test_policy_zero_factors_beside_large_exponentials(ms, V, layout):
    """A token of advantage zero whose ratio is beyond float, and a KL term of coefficient zero whose estimate is:
    both add nothing to the loss and its gradient."""
    A = ms.from_torch
    c = make_policy(24, V, "f32", 0.0)
    if layout == "apart":  # logits and gradient start at different places of a 16-byte word
        w = torch.zeros(24, V + 3, device="cuda")
        w[:, 3:] = c["z"]
        c["z"] = w[:, 3:]
    c["adv"][::3] = 0.0
    c["old"][::3] -= 150.0
    args = lambda beta, ref: P.policy(c["z"].double(), c["t"], c["old"].double(), c["adv"].double(), ref.double(), c["mask"],
                                      0.2, 0.3, beta, 1.0)
    for beta in (0.0, 0.1):
        ref = c["ref"].clone()
        if beta == 0.0:
            ref[1::3] += 150.0
        r = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(ref), clip_low=0.2, clip_high=0.3, kl_coef=beta)
        want, err = args(beta, ref)
        for k in ("logp", "loss", "dlogits"):
            P.close(getattr(r, k).torch(), want[k], err[k], f"beta {beta} {k}")
    # what the formula itself makes NaN stays NaN: an infinite ratio, a target outside
    c["old"][0], c["t"][3] = -math.inf, V
    r = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), clip_low=0.2, clip_high=0.3)
    rows = r.dlogits.torch().isnan().all(1)
    assert bool(rows[0]) and bool(rows[3]) and int(rows.sum()) == 2 and bool(r.loss.torch().isnan())


def test_policy_ratio_keeps_its_precision(ms):
    """One word in the vocabulary: logp is exactly 0, and with advantage -1 the loss is e^-old alone, to the error of a
    float exponential (an ulp, here allowed two) whatever its size; so is the per-token slope in the gradient of two
    even words."""
    A = ms.from_torch
    for old in (-80.0, -40.5, -20.25, -3.0, 0.0, 7.5, 30.0):
        z, t = torch.zeros(1, 1, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")
        o, a = torch.full((1,), old, device="cuda"), torch.full((1,), -1.0, device="cuda")
        loss = float(ms.policy_loss(A(z), A(t), A(o), A(a), clip_low=1.0).loss.torch())
        want = math.exp(-old)
        assert abs(loss - want) <= 2 * 2.0 ** -23 * want, (old, loss, want)
        # two even words: logp = -ln 2 in float, so e^(logp - old) is taken of the same float here
        z = torch.zeros(1, 2, device="cuda")
        r = ms.policy_loss(A(z), A(t), A(o), A(a), clip_low=1.0)
        x = float(r.logp.torch()) - old
        x = float(torch.tensor(x, dtype=torch.float32))
        want = math.exp(x) / 2
        g = r.dlogits.torch()[0].double()
        assert float((g - torch.tensor([want, -want], device="cuda")).abs().max()) <= 4 * 2.0 ** -23 * want, (old, g, want)


# ------------------------------------- products of gates beyond float
def _swings(B, T, H, up, run, seed, sign):
    """Gates near `up` for `run` steps, then near 0.55 until that is undone, in turn; each channel starts
    elsewhere. Nothing shrinks below 2^-126 of itself in 128 steps, so nothing may count as zero."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    period = run + int(run * math.log2(up) / -math.log2(0.55))
    t = torch.arange(T, device="cuda")[None, :, None] + torch.randint(0, period, (B, 1, H), device="cuda", generator=g)
    gate = torch.where(t % period < run, up, 0.55) * (torch.rand(B, T, H, device="cuda", generator=g) * 0.1 + 0.95)
    return gate * (torch.where(t % 3 == 0, -1.0, 1.0) if sign else 1.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,D,H", [(1, 700, 40, 40), (1, 1500, 64, 64), (2, 700, 96, 6), (3, 700, 1500, 1500),
                                     (170, 300, 60, 60), (3, 401, 2048, 32)])
@pytest.mark.parametrize("up,run,sign", [(2.5, 110, True), (1024.0, 16, False), (2.0 ** 20, 9, True)])
def test_scan_with_gates_beyond_one(ms, B, T, D, H, up, run, sign, dtype):
    """States that grow and shrink again by up to 2^180 within float, while the products of the gates alone do not stay
    in it: in few chains and in many."""
    gate = _swings(B, T, H, up, run, 1, sign).to(TORCH[dtype])
    gate[:, 0] = 0.0
    gate[:, T // 2] = 0.0
    tiny = 2.0 ** -100
    x = (rand(B, T, D, seed=2) * tiny).to(TORCH[dtype])
    A = ms.from_torch
    for h0 in (None, rand(B, D, seed=3) * tiny):
        if h0 is not None:
            gate[:, 0] = up
        opt = None if h0 is None else h0.double()
        h, last = ms.gated_scan(A(x), A(gate), None if h0 is None else A(h0), return_state=True)
        wh, wl, eh, el = P.scan(x.double(), gate.double(), opt, "linear")
        P.close(h.torch(), wh, eh, "h")
        P.close(last.torch(), wl, el, "state")
        dh, ds = (rand(B, T, D, seed=4) * tiny).to(x.dtype), rand(B, D, seed=5) * tiny
        got = ms.gated_scan_backward(A(dh), A(x), A(gate), h, None if h0 is None else A(h0), A(ds))
        want, err = P.scan_backward(dh.double(), x.double(), gate.double(), h.torch().double(), opt, ds.double(), "linear")
        # a gate's gradient sums products that may each be rounded below the normal range, to half of 2^-149
        for g, w, e, n in zip(got, want, (err[0], err[1] + D // H * 2.0 ** -150, err[2]), ("dx", "dgate", "dh0")):
            P.close(g.torch(), w, e, n)


@pytest.mark.parametrize("B,T,D", [(1, 900, 70), (4, 900, 900)])
def test_scan_with_gates_beyond_one_is_repeatable(ms, B, T, D):
    gate, x = _swings(B, T, D, 1024.0, 16, 1, True), rand(B, T, D, seed=2) * 2.0 ** -100
    A = ms.from_torch
    runs = []
    for _ in range(6):
        used_memory()
        h = ms.gated_scan(A(x), A(gate))
        runs.append((h.torch(),) + tuple(v.torch() for v in ms.gated_scan_backward(A(x), A(x), A(gate), h)))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_scan_long_look_back_without_maps(ms):
    """Every tile of a long sequence waits for the state of the one before it, and no wait gives up."""
    T = 12000
    gate, x = _swings(1, T, 5, 2.0 ** 20, 9, 1, False), rand(1, T, 5, seed=2) * 2.0 ** -100
    A = ms.from_torch
    from musapy_b200 import ops

    ops.set_scan_status_check(True)
    try:
        h = ms.gated_scan(A(x), A(gate))
        got = ms.gated_scan_backward(A(x), A(x), A(gate), h)
        nan = ms.gated_scan(A(torch.full((1, 400000, 2), math.nan, device="cuda")), A(torch.ones(1, 400000, 2, device="cuda")))
    finally:
        ops.set_scan_status_check(False)
    wh, _, eh, _ = P.scan(x.double(), gate.double(), None, "linear")
    P.close(h.torch(), wh, eh)
    want, err = P.scan_backward(x.double(), x.double(), gate.double(), h.torch().double(), None, None, "linear")
    for g, w, e in zip(got, want, err):
        P.close(g.torch(), w, e)
    assert bool(nan.torch().isnan().all())


@pytest.mark.parametrize("B,T,D", [(2, 300, 36), (4, 300, 900)])
def test_scan_keeps_what_is_not_finite_in_its_channel(ms, B, T, D):
    """Linear: an infinite or NaN gate or input makes its channel what the formula makes it from that step on, up to
    where the gate is zero again (zero times an infinity stays NaN); the other channels keep their values."""
    x, g, h0 = rand(B, T, D, seed=1), gates(B, T, D, "linear", "f32", 2), rand(B, D, seed=3)
    A = ms.from_torch
    clean = ms.gated_scan(A(x), A(g), A(h0)).torch()
    x[0, 40, 3], g[0, 90, 9], g[1, 100, 20], x[1, 7, 30] = math.inf, math.nan, math.inf, math.nan
    h = ms.gated_scan(A(x), A(g), A(h0)).torch()
    want, _, _, _ = P.scan(x.double(), g.double(), h0.double(), "linear")
    assert torch.equal(h.isnan(), want.isnan()) and torch.equal(h.isinf(), want.isinf())
    same = torch.ones(B, T, D, dtype=torch.bool, device="cuda")
    for b, t, d in ((0, 40, 3), (0, 90, 9), (1, 100, 20), (1, 7, 30)):
        same[b, t:, d] = False
    torch.testing.assert_close(h[same], clean[same], rtol=1e-5, atol=1e-5)


# ------------------------------------------------------ saturated gates
@pytest.mark.parametrize("B,T,D,H", [(2, 1, 64, 64), (3, 40, 33, 33), (1, 300, 70, 70), (4, 200, 900, 900), (2, 60, 96, 6)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scan_saturated_float_gates(ms, B, T, D, H, dtype, sign):
    """Gates of 16 to 64 in 32 bits: one minus the sigmoid, or the sigmoid, is as small as 2^-92 and keeps its
    relative precision, and so do the gradients that it enters."""
    g = torch.Generator(device="cuda").manual_seed(1)
    gate = (torch.rand(B, T, H, device="cuda", generator=g) * 48 + 16) * sign
    check_scan(ms, rand(B, T, D, seed=2, dtype=dtype), gate, torch.zeros(B, D, device="cuda") if sign > 0 else rand(B, D, seed=3),
               "sigmoid")
    x = rand(B, D, seed=4, dtype=dtype) if sign > 0 else torch.zeros(B, D, dtype=TORCH[dtype], device="cuda")
    s0 = torch.zeros(B, D, device="cuda") if sign > 0 else rand(B, D, seed=5)
    want, wl, e, el = P.scan(x[:, None].double(), gate[:, :1].double(), s0.double(), "sigmoid")
    state = ms.from_torch(s0.clone())
    h = ms.gated_scan_step(state, ms.from_torch(x), ms.from_torch(gate[:, 0].contiguous()), mode="sigmoid")
    P.close(h.torch(), want[:, 0], e[:, 0], "step")
    P.close(state.torch(), wl, el, "state")


# --------------------------------------------------------------- memory
def test_a_kept_loss_keeps_only_itself(ms):
    """A program that collects the losses of its steps holds 16 bytes for each, not the tokens' results."""
    A = ms.from_torch
    c = make_policy(5000, 40, "f32", 0.0)
    r = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]))
    assert r.loss.torch().untyped_storage().nbytes() <= 16
