"""The block operators at the edges of their ranges on the GPU, against their formulas in 64 bits: results without
elements to sum."""
import pytest
import torch

from .test_blocks_gpu import rand

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
