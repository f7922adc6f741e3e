"""The block operators at the edges of their ranges on the GPU, against their formulas in 64 bits: results without
elements to sum and factors of zero beside exponentials that overflow. Tolerances are the bounds that blocks_plain
derives."""
import math

import pytest
import torch

from . import blocks_plain as P
from .test_blocks_gpu import make_policy, rand

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
