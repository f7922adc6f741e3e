"""Linear attention where its inputs lie so that whole rows are walked (bf16, 16-byte words): the layouts, sizes and
heads that choose between the walk and the kernels of single chunks, several calls at once, and graphs."""
import math

import pytest
import torch

from . import sequence_plain as Q
from .test_sequence_gpu import check_attention, decays, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("DK,DV", [(8, 8), (64, 64), (64, 128), (128, 64), (128, 128), (72, 136), (136, 72), (120, 56), (16, 72), (96, 8)])
@pytest.mark.parametrize("T", [1, 63, 64, 65, 257])
def test_widths_and_lengths(ms, DK, DV, T):
    B, H = 2, 2
    check_attention(ms, rand(B, T, H, DK, seed=1, dtype="bf16"), rand(B, T, H, DK, seed=2, dtype="bf16"),
                    rand(B, T, H, DV, seed=3, dtype="bf16"), decays(B, T, H, seed=4), rand(B, H, DK, DV, seed=5), rand(B, H, DK, DV, seed=6))


@pytest.mark.parametrize("B,T,H,Hq", [(1, 4000, 1, 1), (1, 1500, 4, 2), (3, 700, 49, 7), (1, 520, 150, 150), (40, 70, 4, 1), (2, 20000, 1, 1)])
def test_rows_and_heads(ms, B, T, H, Hq):
    """From one head, whose row is cut into many segments, to more heads than there are places for blocks."""
    D = 64
    check_attention(ms, rand(B, T, Hq, D, seed=1, dtype="bf16"), rand(B, T, Hq, D, seed=2, dtype="bf16"),
                    rand(B, T, H, D, seed=3, dtype="bf16"), decays(B, T, H, seed=4, mean=5.0), rand(B, H, D, D, seed=5),
                    rand(B, H, D, D, seed=6))


def test_without_states(ms):
    B, T, H, D = 2, 300, 3, 128
    check_attention(ms, *(rand(B, T, H, D, seed=i, dtype="bf16") for i in (1, 2, 3)), decays(B, T, H, seed=4), None)


@pytest.mark.parametrize("kind", ["one projection", "heads first", "time first", "every second step", "odd strides", "one head for all",
                                  "odd offset"])
def test_layouts(ms, kind):
    B, T, H, D = 2, 200, 4, 64

    def make(seed):
        if kind == "one projection":  # q, k and v as slices of one product
            return rand(B, T, 3 * H * D, seed=1, dtype="bf16")[..., (seed - 1) * H * D:seed * H * D].unflatten(-1, (H, D))
        if kind == "heads first":
            return rand(B, H, T, D, seed=seed, dtype="bf16").transpose(1, 2)
        if kind == "time first":
            return rand(T, B, H, D, seed=seed, dtype="bf16").transpose(0, 1)
        if kind == "every second step":
            return rand(B, 2 * T, H, D, seed=seed, dtype="bf16")[:, ::2]
        if kind == "odd strides":  # multiples of 16 bytes, but of nothing more
            return rand(B, T, H, D + 8, seed=seed, dtype="bf16")[..., 8:]
        if kind == "one head for all":
            return rand(B, T, 1, D, seed=seed, dtype="bf16").expand(B, T, H, D)
        return rand(B, T, H, D + 8, seed=seed, dtype="bf16")[..., 1:D + 1]

    check_attention(ms, make(1), make(2), make(3), decays(B, T, H, seed=4), rand(B, H, D, D, seed=5), None, make(3), what=kind)


def test_restarts_and_strong_decays(ms):
    B, T, H, D = 1, 1000, 2, 64
    g = decays(B, T, H, seed=4)
    g[0, ::97, 0] = -math.inf
    g[0, 64:128, 1] = -60.0
    g[0, 500, 1] = -150.0
    check_attention(ms, *(rand(B, T, H, D, seed=i, dtype="bf16") for i in (1, 2, 3)), g, rand(B, H, D, D, seed=5), rand(B, H, D, D, seed=6))


def test_rows_behind_the_last_step_stay(ms):
    """Outputs of 70 steps: what lies behind them in the same allocation is not written."""
    B, T, H, D = 1, 70, 2, 64
    big = torch.full((B, T + 58, H, D), 7.0, dtype=torch.bfloat16, device="cuda")
    out = ms.from_torch(big[:, :T])
    ms.linear_attention(*(ms.from_torch(rand(B, T, H, D, seed=i, dtype="bf16")) for i in (1, 2, 3)), ms.from_torch(decays(B, T, H, seed=4)),
                        out=out)
    assert (big[:, T:] == 7.0).all() and (big[:, :T] != 7.0).any()


def test_out_that_no_copy_may_write(ms):
    """An out= that begins between 16-byte words takes the other kernels, and the same values up to their rounding."""
    B, T, H, D = 1, 130, 2, 64
    q, k, v = (ms.from_torch(rand(B, T, H, D, seed=i, dtype="bf16")) for i in (1, 2, 3))
    g = ms.from_torch(decays(B, T, H, seed=4))
    room = torch.zeros(B * T * H * D + 1, dtype=torch.bfloat16, device="cuda")
    out = room[1:].view(B, T, H, D)
    ms.linear_attention(q, k, v, g, out=ms.from_torch(out))
    o = ms.linear_attention(q, k, v, g).torch()
    args = [x.torch().double() for x in (q, k, v, g)]
    slack = Q.attention_bounds(*args, None, D ** -0.5, torch.bfloat16)[0]
    assert ((o.double() - out.double()).abs() <= 2 * slack + 2.0 ** -7 * o.double().abs()).all()


def test_status_of_the_waits(ms):
    ms.ops.set_scan_status_check(True)
    try:
        x = ms.from_torch(rand(1, 300, 2, 64, seed=1, dtype="bf16"))
        ms.linear_attention(x, x, x, ms.from_torch(decays(1, 300, 2, seed=2)))
        ms.linear_attention_backward(x, x, x, x, ms.from_torch(decays(1, 300, 2, seed=2)))
    finally:
        ms.ops.set_scan_status_check(False)


def _both(ms, t):
    A = ms.from_torch
    o, s = ms.linear_attention(*(A(x) for x in t), return_state=True)
    return [x.torch() for x in (o, s, *ms.linear_attention_backward(o, *(A(x) for x in t)))]


def _inputs(seed, B=2, T=600, H=3, D=64):
    return [*(rand(B, T, H, D, seed=seed + i, dtype="bf16") for i in range(3)), decays(B, T, H, seed=seed + 3), rand(B, H, D, D, seed=seed + 4)]


def test_in_graphs_and_on_streams_at_once(ms):
    sets = [_inputs(10), _inputs(20)]
    want = [[x.clone() for x in _both(ms, t)] for t in sets]
    streams = [ms.Stream("cuda:0") for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, t in zip(streams, sets):
            with ms.stream(s):
                got.append(_both(ms, t))
    for s in streams:
        s.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(want[i % 2], g))
    held = [x.clone() for x in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _both(ms, held)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            graphs.append((graph, _both(ms, held)))
    for t, w in zip(sets, want):
        for a, b in zip(held, t):
            a.copy_(b)
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(w, outs))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_status_after_memory_that_was_another_calls(ms, dtype):
    """Scratch that holds what a wait that gave up would leave, from whoever had the memory before."""
    x = rand(1, 300, 2, 64, seed=1, dtype=dtype)
    g = ms.from_torch(decays(1, 300, 2, seed=2))
    ms.ops.set_scan_status_check(True)
    try:
        for _ in range(3):
            used = [torch.full((n,), 6, dtype=torch.int32, device="cuda") for n in (256, 4096, 1 << 16, 1 << 18, 1 << 20, 1 << 22)]
            del used
            A = ms.from_torch
            ms.linear_attention(A(x), A(x), A(x), g)
            ms.linear_attention_backward(A(x), A(x), A(x), A(x), g)
    finally:
        ms.ops.set_scan_status_check(False)
