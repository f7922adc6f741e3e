"""Waits between the warps of linear attention's walk that run out: the limit is shortened on the host, the block ends in
order, the status says so, and the calls that follow are right."""
import contextlib

import pytest
import torch

from .test_sequence_gpu import decays, rand

pytestmark = pytest.mark.gpu

TWO_SECONDS = 2_000_000_000


@contextlib.contextmanager
def limit(ns):
    from musapy_b200._lib import LIB

    assert LIB.mpb_linear_attention_wait_limit(ns) == TWO_SECONDS
    try:
        yield
    finally:
        torch.cuda.synchronize()
        assert LIB.mpb_linear_attention_wait_limit(TWO_SECONDS) == ns


@pytest.fixture
def checked(ms):
    ms.ops.set_scan_status_check(True)
    yield ms
    ms.ops.set_scan_status_check(False)


def inputs(DK, DV, T, H):
    q, k = rand(1, T, H, DK, seed=1, dtype="bf16"), rand(1, T, H, DK, seed=2, dtype="bf16")
    v, do = rand(1, T, H, DV, seed=3, dtype="bf16"), rand(1, T, H, DV, seed=7, dtype="bf16")
    return q, k, v, decays(1, T, H, seed=4), rand(1, H, DK, DV, seed=5), rand(1, H, DK, DV, seed=6), do


def forward(ms, x):
    A = ms.from_torch
    return [y.torch() for y in ms.linear_attention(*(A(t) for t in x[:5]), return_state=True)]


def backward(ms, x):
    A = ms.from_torch
    q, k, v, g, state, dstate, do = x
    return [y.torch() for y in ms.linear_attention_backward(*(A(t) for t in (do, q, k, v, g, state, dstate)))]


# whole rows of heads, and rows in segments; widths with two and with three chunks under way
SIZES = [(128, 128, 500, 200), (64, 64, 500, 200), (64, 128, 3000, 2), (128, 64, 3000, 2)]


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_a_wait_that_runs_out_is_an_error(checked, size):
    ms, x = checked, inputs(*size)
    want = [forward(ms, x), backward(ms, x)]
    for run, w in zip((forward, backward), want):
        with limit(0):
            with pytest.raises(ms.errors.KernelError, match="gave up"):
                run(ms, x)
        assert all(torch.equal(a, b) for a, b in zip(run(ms, x), w))


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("ns", [4000, 8000, 12000, 20000, 60000])
def test_waits_that_run_out_on_the_way(checked, size, ns):
    """Some blocks may finish and some not, at any chunk: the call is right or says that it is not."""
    ms, x = checked, inputs(*size)
    want = [forward(ms, x), backward(ms, x)]
    for _ in range(3):
        for run, w in zip((forward, backward), want):
            with limit(ns):
                try:
                    got = run(ms, x)
                except ms.errors.KernelError:
                    got = None
            assert got is None or all(torch.equal(a, b) for a, b in zip(got, w))
            assert all(torch.equal(a, b) for a, b in zip(run(ms, x), w))


def test_the_limit_is_two_seconds_at_most(ms):
    from musapy_b200._lib import LIB

    for asked, kept in ((-5, 0), (1 << 40, TWO_SECONDS), (7, 7)):
        LIB.mpb_linear_attention_wait_limit(asked)
        assert LIB.mpb_linear_attention_wait_limit(TWO_SECONDS) == kept


@pytest.mark.parametrize("size", SIZES, ids=str)
def test_what_a_block_that_gave_up_leaves_is_nan(ms, size):
    x = inputs(*size)
    with limit(0):
        got = [*forward(ms, x), *backward(ms, x)]
    assert all(y.isnan().all() for y in got)


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("ns", [4000, 8000, 12000, 20000, 60000])
def test_every_value_is_right_or_nan(ms, size, ns):
    x = inputs(*size)
    want = [*forward(ms, x), *backward(ms, x)]
    for _ in range(3):
        with limit(ns):
            got = [*forward(ms, x), *backward(ms, x)]
        assert all(((a == b) | a.isnan()).all() for a, b in zip(got, want))


def test_rows_of_others_stay(ms):
    """What a block that gave up fills is its own: nothing behind the outputs' last step."""
    big = torch.full((1, 200, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    x = inputs(64, 64, 70, 2)
    with limit(0):
        ms.linear_attention(*(ms.from_torch(t) for t in x[:5]), out=ms.from_torch(big[:, :70]))
    assert big[:, :70].isnan().all() and (big[:, 70:] == 7.0).all()
