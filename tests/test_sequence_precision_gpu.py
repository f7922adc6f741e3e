"""How many bits linear attention keeps on its way to 16-bit results, on each of its paths: scores and states that meet a
bf16 operand go there as two bf16 numbers, whose sum is off by 2^-16 at most (each is the rounding, by 2^-8 at most, of
what the one before left)."""
import pytest
import torch

from . import blocks_plain as P
from . import sequence_plain as Q
from .test_sequence_gpu import decays, rand

pytestmark = pytest.mark.gpu

TWO = 2.0 ** -16

# (DK, DV, elements before a row's channels): rows that are walked, and what takes the chunks' kernels by width or alignment
PATHS = [(64, 64, 0), (128, 128, 0), (64, 128, 0), (128, 64, 0), (40, 72, 0), (64, 64, 1), (136, 72, 0), (64, 256, 0)]


def inputs(DK, DV, before, T=500, dtype="bf16", std=1.5, mean=3.0):
    B, H, Hq = 2, 4, 2
    make = lambda h, d, seed: rand(B, T, h, d + 8 * bool(before), seed=seed, dtype=dtype)[..., before:before + d]
    q, k, v, do = make(Hq, DK, 1), make(Hq, DK, 2), make(H, DV, 3), make(H, DV, 7)
    return q, k, v, decays(B, T, H, seed=4), rand(B, H, DK, DV, seed=5), rand(B, H, DK, DV, seed=6), do


@pytest.mark.parametrize("DK,DV,before", PATHS)
def test_bf16_outputs_are_their_rounding(ms, DK, DV, before):
    q, k, v, g, state, _, _ = inputs(DK, DV, before)
    A, by = ms.from_torch, DK ** -0.5
    o = ms.linear_attention(A(q), A(k), A(v), A(g), A(state)).torch()
    args = [x.double() for x in (q, k, v, g, state)]
    want = Q.attention(*args, by)[0]
    mag = Q.attention(*(x if x is args[3] else x.abs() for x in args), by)[0]
    P.close(o, want, (Q.roundings(q.shape[1], DK, DV) * Q.EPS32 + TWO) * mag, "o")


@pytest.mark.parametrize("DK,DV,before", PATHS)
def test_bf16_gradients_are_their_rounding(ms, DK, DV, before):
    q, k, v, g, state, dstate, do = inputs(DK, DV, before)
    A, by = ms.from_torch, DK ** -0.5
    got = [x.torch() for x in ms.linear_attention_backward(A(do), A(q), A(k), A(v), A(g), A(state), A(dstate))]
    args = [x.double() for x in (do, q, k, v, g, state, dstate)]
    want = Q.attention_backward(*args, by)
    mag = Q.attention_backward(*(x if x is args[4] else x.abs() for x in args), by)
    n = Q.roundings(q.shape[1], DK, DV) * Q.EPS32
    for x, w, m, what in zip(got[:3], want, mag, ("dq", "dk", "dv")):
        P.close(x, w, (n + TWO) * m, what)


def test_bf16_outputs_do_not_depend_on_alignment(ms):
    """The same values in rows of 16-byte words and between them: two results that each keep 16 bits."""
    q, k, v, g, state, _, _ = inputs(64, 64, 0)
    A = ms.from_torch
    shift = lambda x: torch.nn.functional.pad(x, (1, 7))[..., 1:65]
    o, p = (ms.linear_attention(A(f(q)), A(f(k)), A(f(v)), A(g), A(state)).torch() for f in (lambda x: x, shift))
    args = [x.double() for x in (q, k, v, g, state)]
    mag = Q.attention(*(x if x is args[3] else x.abs() for x in args), 0.125)[0]
    P.close(p, o.double(), 2 * (Q.roundings(q.shape[1], 64, 64) * Q.EPS32 + TWO) * mag + 2.0 ** -8 * o.double().abs(), "o")
