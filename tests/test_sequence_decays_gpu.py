"""The gradient of linear attention's decays where they are strong, weak and mixed: each step's by what passes through
that step, not by what lies around it."""
import math

import pytest
import torch

from . import blocks_plain as P
from . import sequence_plain as Q
from .test_sequence_gpu import NORM, near, rand

pytestmark = pytest.mark.gpu


def check(ms, q, k, v, g, state, dstate, do, what=""):
    """Each element within the roundings on its way (sequence_plain.roundings) of the magnitudes that pass through its own
    step, from the steps before it to the steps from it on; a decay of zero has no gradient."""
    A, opt, by = ms.from_torch, lambda f, x: None if x is None else f(x), q.shape[-1] ** -0.5
    got = ms.linear_attention_backward(A(do), A(q), A(k), A(v), A(g), opt(A, state), opt(A, dstate))[3].torch()
    args = [opt(torch.Tensor.double, x) for x in (do, q, k, v, g, state, dstate)]
    want = Q.attention_backward(*args, by)[3]
    mag = Q.attention_backward(*(x if i == 4 else opt(torch.abs, x) for i, x in enumerate(args)), by)[3]
    slack = Q.roundings(q.shape[1], q.shape[3], v.shape[3]) * Q.EPS32 * mag
    if g.dim() == 1:
        n = want.shape[0] * want.shape[1]
        slack = slack.sum((0, 1)) + (Q.CHUNK + n / Q.CHUNK + 2) * Q.EPS32 * want.abs().sum((0, 1))
        want = want.sum((0, 1))
    P.close(got, want, slack, what)
    near(got, want, NORM[torch.float32], what)


# (dtype, DK, DV, elements before a row's channels): the gradients' two kernels, in each type
PATHS = [("bf16", 64, 64, 0), ("bf16", 128, 128, 0), ("bf16", 128, 40, 0), ("bf16", 64, 64, 1), ("f16", 40, 72, 0), ("f32", 64, 64, 0),
         ("f32", 96, 80, 0)]


def inputs(dtype, DK, DV, before, T=300, B=1, H=4, Hq=2):
    make = lambda h, d, seed: rand(B, T, h, d + 8 * bool(before), seed=seed, dtype=dtype)[..., before:before + d]
    return make(Hq, DK, 1), make(Hq, DK, 2), make(H, DV, 3), make(H, DV, 7), rand(B, H, DK, DV, seed=5), rand(B, H, DK, DV, seed=6)


@pytest.mark.parametrize("mean", [-0.01, -1.0, -10.0, -30.0, -80.0])
@pytest.mark.parametrize("path", PATHS, ids=str)
def test_strength(ms, path, mean):
    q, k, v, do, state, dstate = inputs(*path)
    g = mean * (0.9 + 0.1 * rand(1, 300, 4, seed=4).tanh())
    check(ms, q, k, v, g, None, None, do, "without states")
    check(ms, q, k, v, g, state, dstate, do, "with states")


@pytest.mark.parametrize("path", PATHS, ids=str)
def test_strong_steps_among_weak_ones(ms, path):
    """Single strong decays, at every place of a chunk: what neighbours pass on is a million million times as large."""
    q, k, v, do, state, dstate = inputs(*path)
    g = -0.02 * torch.ones(1, 300, 4, device="cuda")
    for h in range(4):
        g[0, h::7, h] = -25.0 - 10 * h
    g[0, 150, 1] = -math.inf
    check(ms, q, k, v, g, state, dstate, do)


@pytest.mark.parametrize("path", PATHS, ids=str)
def test_one_decay_per_head(ms, path):
    q, k, v, do, state, dstate = inputs(*path, B=2)
    state, dstate = (x.expand(2, -1, -1, -1) for x in (state[:1], dstate[:1]))
    check(ms, q, k, v, torch.tensor([-0.01, -3.0, -20.0, -70.0], device="cuda"), state, dstate, do)


@pytest.mark.parametrize("T", [1, 2, 31, 32, 33, 63, 64, 65, 97])
@pytest.mark.parametrize("path", PATHS[:6], ids=str)
def test_lengths(ms, path, T):
    """Pairs on both sides of the places where a chunk's columns are shared out."""
    q, k, v, do, state, dstate = inputs(*path, T=T)
    g = -5.0 - 10 * rand(1, T, 4, seed=4).abs()
    check(ms, q, k, v, g.clamp(min=-40), state, dstate, do)


@pytest.mark.parametrize("dtype,D,before,fore,back", [("f32", 32, 0, (1540, 1900), (1540, 1900)),
                                                      ("bf16", 64, 0, (1600, 2000), (1000, 1400)),
                                                      ("bf16", 64, 1, (1540, 1900), (1540, 1900))])
def test_states_that_overflowed_are_dropped(ms, dtype, D, before, fore, back):
    """Decays above one that carry the state past the largest float, over chunks of one segment of a row, and a decay of zero
    behind them: what follows is as if the row began there. Backward, the same for what comes before them."""
    B, T, H = 1, 3000, 60
    make = lambda seed: rand(B, T, H, D + 8 * before, seed=seed, dtype=dtype)[..., before:before + D]
    q, k, v, do = (make(s) for s in (1, 2, 3, 7))
    state, dstate = rand(B, H, D, D, seed=5), rand(B, H, D, D, seed=6)
    A, n = ms.from_torch, 2 * (Q.roundings(T, D, D) * Q.EPS32 + Q.SCORES[q.dtype])

    def grows(lo, hi, restart):
        g = -0.05 * torch.ones(B, T, H, device="cuda")
        g[:, lo:hi] = 0.5
        g[:, restart] = -math.inf
        return g

    lo, at = fore
    g = grows(lo, at, at)
    o, last = [x.torch() for x in ms.linear_attention(A(q), A(k), A(v), A(g), A(state), return_state=True)]
    w, wlast = [x.torch() for x in ms.linear_attention(*(A(x[:, at:]) for x in (q, k, v, g)), return_state=True)]
    assert not o[:, at - 1].isfinite().all()  # it did overflow
    mag = Q.attention(*(x[:, at:].double().abs() for x in (q, k, v)), g[:, at:].double(), None, D ** -0.5)
    P.close(o[:, at:], w.double(), n * mag[0] + P.ROUND[o.dtype][0] * w.double().abs(), "o")
    P.close(last, wlast.double(), n * mag[1], "state")
    cut, hi = back
    g = grows(cut, hi, cut)
    got = [x.torch() for x in ms.linear_attention_backward(A(do), A(q), A(k), A(v), A(g), A(state), A(dstate))]
    want = [x.torch() for x in ms.linear_attention_backward(*(A(x[:, :cut]) for x in (do, q, k, v, g)), A(state))]
    assert not got[2][:, cut].isfinite().all()
    mag = Q.attention_backward(*(x[:, :cut].double().abs() for x in (do, q, k, v)), g[:, :cut].double(), state.double().abs(), None,
                               D ** -0.5)
    for x, y, m, what in zip(got, want, mag, ("dq", "dk", "dv", "dlog_decay", "dstate0")):
        x = x if what == "dstate0" else x[:, :cut]
        P.close(x, y.double(), n * m + P.ROUND[x.dtype][0] * y.double().abs(), what)
