"""Linear attention, distillation and the embedding on the GPU against their formulas in 64 bits, at the sizes, layouts
and values where they can go wrong. Tolerances are the bounds that sequence_plain derives."""
import math

import pytest
import torch

from . import blocks_plain as P
from . import sequence_plain as Q

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rand(*shape, seed, dtype="f32", std=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(TORCH[dtype])


def whole(lo, hi, *shape, seed, dtype=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi, shape, device="cuda", generator=g).to(dtype)


def decays(*shape, seed, mean=3.0):
    return torch.log(torch.sigmoid(rand(*shape, seed=seed, std=1.5, mean=mean)))


def near(got, want, limit, what):
    """The 2-norm of what is off, against the result's: roundings that point in no direction. Of many values only: a
    single one may be a sum whose terms cancel, a - b with a = 1 and b = 1 - 2^-4, say, of which bf16 scores may
    lose 2^-8 a, a sixteenth of the result; over 256 values and more such ones weigh no more than their terms."""
    w = want.double()
    if w.numel() < 256:
        return
    off, size = (got.double() - w).norm().item(), w.norm().item()
    assert off <= limit * size + 1e-30, f"{what}: {off / max(size, 1e-300):.3g} of the result's norm, over {limit:.3g}"


# 64 units for results of 32 bits: the root of some thousand roundings; a unit or two of a 16-bit result's rounding
NORM = {torch.float32: 64 * Q.EPS32, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def check_attention(ms, q, k, v, g, state, dstate=None, do=None, scale=None, what=""):
    """Forward and backward of torch tensors of any layout."""
    A = ms.from_torch
    opt = lambda x: None if x is None else A(x)
    d = lambda x: None if x is None else x.double()
    by = q.shape[-1] ** -0.5 if scale is None else scale
    o, last = ms.linear_attention(A(q), A(k), A(v), A(g), opt(state), scale=scale, return_state=True)
    wo, ws = Q.attention(d(q), d(k), d(v), d(g), d(state), by)
    eo, es = Q.attention_bounds(d(q), d(k), d(v), d(g), d(state), by, q.dtype)
    P.close(o.torch(), wo, eo, f"{what} o")
    P.close(last.torch(), ws, es, f"{what} state")
    near(o.torch(), wo, NORM[q.dtype], f"{what} o")
    near(last.torch(), ws, NORM[torch.float32], f"{what} state")
    if do is None:
        do = rand(*v.shape, seed=77).to(v.dtype)
    got = ms.linear_attention_backward(A(do), A(q), A(k), A(v), A(g), opt(state), opt(dstate), scale=scale)
    args = (d(do), d(q), d(k), d(v), d(g), d(state), d(dstate), by)
    want, err = Q.attention_backward(*args), Q.attention_backward_bounds(*args, q.dtype)
    for x, w, e, n in zip(got, want, err, ("dq", "dk", "dv", "dlog_decay", "dstate0")):
        if n == "dlog_decay" and g.dim() == 1:
            # the sum over a chunk's steps, then over the chunks
            e = e.sum((0, 1)) + (Q.CHUNK + w.shape[0] * w.shape[1] / Q.CHUNK + 2) * Q.EPS32 * w.abs().sum((0, 1))
            w = w.sum((0, 1))
        P.close(x.torch(), w, e, f"{what} {n}")
        if n != "dlog_decay":
            near(x.torch(), w, NORM[x.torch().dtype], f"{what} {n}")
    assert got[3].shape == tuple(g.shape) and got[3].torch().dtype == got[4].torch().dtype == torch.float32


SHAPES = [  # B, T, H, Hq, DK, DV
    (1, 1, 1, 1, 1, 1), (2, 1, 3, 3, 16, 64), (1, 7, 2, 1, 5, 3), (2, 63, 2, 2, 64, 64), (1, 64, 1, 1, 128, 128),
    (3, 65, 4, 2, 40, 72), (2, 128, 2, 2, 17, 33), (1, 200, 6, 3, 96, 80), (1, 129, 2, 1, 256, 256), (2, 150, 1, 1, 100, 130),
    (1, 700, 1, 1, 64, 48), (1, 2000, 2, 2, 32, 24), (5, 90, 8, 2, 20, 20), (1, 330, 4, 1, 128, 64),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(ms, shape, dtype):
    B, T, H, Hq, DK, DV = shape
    check_attention(ms, rand(B, T, Hq, DK, seed=1, dtype=dtype), rand(B, T, Hq, DK, seed=2, dtype=dtype),
                    rand(B, T, H, DV, seed=3, dtype=dtype), decays(B, T, H, seed=4), rand(B, H, DK, DV, seed=5),
                    rand(B, H, DK, DV, seed=6))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_one_decay_per_head(ms, dtype):
    B, T, H, D = 2, 300, 5, 48
    check_attention(ms, rand(B, T, H, D, seed=1, dtype=dtype), rand(B, T, H, D, seed=2, dtype=dtype),
                    rand(B, T, H, D, seed=3, dtype=dtype), decays(H, seed=4), None, None, scale=0.3)


@pytest.mark.parametrize("value", [-math.inf, -200.0, -1e30])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attention_restarts(ms, dtype, value):
    """Decays of zero: the sequences of a packed row do not meet, nor the state before it where the first step drops it."""
    B, T, H, D = 2, 400, 2, 32
    g = decays(B, T, H, seed=4)
    for b, t, h in ((0, 1, 0), (0, 63, 0), (0, 64, 0), (0, 65, 1), (0, 200, 0), (1, 0, 0), (1, 0, 1), (1, 127, 1), (1, 128, 1),
                    (1, 399, 0)):
        g[b, t, h] = value
    q, k, v = (rand(B, T, H, D, seed=i, dtype=dtype) for i in (1, 2, 3))
    state = rand(B, H, D, D, seed=5)
    check_attention(ms, q, k, v, g, state, rand(B, H, D, D, seed=6))
    A = ms.from_torch
    dg = ms.linear_attention_backward(A(q), A(q), A(k), A(v), A(g), A(state))[3].torch()
    assert (dg[g == value] == 0).all()
    # a packed sequence alone gives the same
    o = ms.linear_attention(A(q), A(k), A(v), A(g), A(state)).torch()
    part = slice(200, 400)
    alone = ms.linear_attention(A(q[:1, part]), A(k[:1, part]), A(v[:1, part]), A(g[:1, part])).torch()
    P.close(o[:1, part, :1], alone[:, :, :1].double(), 2 * Q.attention_bounds(
        *(x[:1, part].double() for x in (q, k, v, g)), None, D ** -0.5, q.dtype)[0][:, :, :1] + P.ROUND[q.dtype][0] *
        alone[:, :, :1].double().abs())


def test_attention_drops_any_state(ms):
    """A decay of zero drops what came before, whatever that was: here infinities and NaN in the first state."""
    B, T, H, D = 1, 100, 1, 16
    q, k, v = (rand(B, T, H, D, seed=i) for i in (1, 2, 3))
    g = decays(B, T, H, seed=4)
    g[:, 0] = -math.inf
    bad = torch.full((B, H, D, D), math.inf, device="cuda")
    bad[..., ::2] = math.nan
    A = ms.from_torch
    o, last = ms.linear_attention(A(q), A(k), A(v), A(g), A(bad), return_state=True)
    w, wl = ms.linear_attention(A(q), A(k), A(v), A(g), return_state=True)
    assert torch.equal(o.torch(), w.torch()) and torch.equal(last.torch(), wl.torch())
    state = bad.clone()
    ms.linear_attention_step(A(state), A(q[:, 0]), A(k[:, 0]), A(v[:, 0]), A(g[:, 0]))
    assert state.isfinite().all()


@pytest.mark.parametrize("mean", [-30.0, 0.0, 9.0])
def test_attention_decays_strong_and_weak(ms, mean):
    """Decays that forget within a step, and decays so near one that a row of thousands is remembered."""
    B, T, H, D = 1, 1500, 2, 16
    g = -torch.nn.functional.softplus(-rand(B, T, H, seed=4, std=2.0, mean=mean))
    check_attention(ms, *(rand(B, T, H, D, seed=i) for i in (1, 2, 3)), g, rand(B, H, D, D, seed=5), rand(B, H, D, D, seed=6))


def test_attention_growing_states(ms):
    """Log-decays above zero are decays above one."""
    B, T, H, D = 1, 130, 2, 16
    check_attention(ms, *(rand(B, T, H, D, seed=i) for i in (1, 2, 3)), rand(B, T, H, seed=4, std=0.3, mean=0.05),
                    rand(B, H, D, D, seed=5), rand(B, H, D, D, seed=6))


def _odd(kind, B, T, H, D, seed, dtype):
    if kind == "heads first":
        return rand(B, H, T, D, seed=seed, dtype=dtype).transpose(1, 2)
    if kind == "time first":
        return rand(T, B, H, D, seed=seed, dtype=dtype).transpose(0, 1)
    if kind == "odd offset":
        return rand(B, T, H, D + 3, seed=seed, dtype=dtype)[..., 1:D + 1]
    if kind == "channels outside":
        return rand(B, D, T, H, seed=seed, dtype=dtype).permute(0, 2, 3, 1)
    if kind == "every second step":
        return rand(B, 2 * T, H, D, seed=seed, dtype=dtype)[:, ::2]
    return rand(1, T, 1, D, seed=seed, dtype=dtype).expand(B, T, H, D)


@pytest.mark.parametrize("kind", ["heads first", "time first", "odd offset", "channels outside", "every second step", "broadcast"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_layouts(ms, kind, dtype):
    B, T, H, D = 2, 100, 3, 40
    q, k, v = (_odd(kind, B, T, H, D, i, dtype) for i in (1, 2, 3))
    g = torch.log(torch.sigmoid(_odd(kind, B, T, H, 1, 4, "f32")[..., 0] + 2))
    check_attention(ms, q, k, v, g, rand(B, H, D, D, seed=5), None, _odd(kind, B, T, H, D, 6, dtype), what=kind)


def test_attention_views_of_one_projection(ms):
    """q, k, v and the decays as slices of one product."""
    B, T, H, D = 2, 130, 4, 32
    proj = rand(B, T, H * (3 * D) + H, seed=1, dtype="bf16")
    q, k, v = (proj[..., i * H * D:(i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3))
    check_attention(ms, q, k, v, torch.log(torch.sigmoid(proj[..., 3 * H * D:].float())), None)


def test_attention_reversed_time(ms):
    q, k, v = (rand(1, 90, 2, 24, seed=i) for i in (1, 2, 3))
    g = decays(1, 90, 2, seed=4)
    A, f = ms.from_torch, lambda x: ms.flip(ms.from_torch(x), 1)
    o = ms.linear_attention(f(q), f(k), f(v), f(g))
    args = [x.flip(1).double() for x in (q, k, v, g)]
    P.close(o.torch(), Q.attention(*args, None, 24 ** -0.5)[0], Q.attention_bounds(*args, None, 24 ** -0.5, torch.float32)[0])


@pytest.mark.parametrize("B,T", [(0, 5), (2, 0), (0, 0)])
@pytest.mark.parametrize("by_head", [False, True])
def test_attention_empty(ms, B, T, by_head):
    A, H, D = ms.from_torch, 2, 8
    x, state = rand(B, T, H, D, seed=1), rand(B, H, D, D, seed=2)
    g = decays(H, seed=3) if by_head else decays(B, T, H, seed=3)
    o, last = ms.linear_attention(A(x), A(x), A(x), A(g), A(state), return_state=True)
    assert o.shape == (B, T, H, D) and torch.equal(last.torch(), state)
    _, last = ms.linear_attention(A(x), A(x), A(x), A(g), return_state=True)
    assert torch.equal(last.torch(), torch.zeros_like(state))
    dq, dk, dv, dg, ds = ms.linear_attention_backward(A(x), A(x), A(x), A(x), A(g), A(state), A(state))
    assert dq.shape == dk.shape == dv.shape == x.shape and torch.equal(ds.torch(), state)
    assert torch.equal(dg.torch(), torch.zeros_like(g))
    assert torch.equal(ms.linear_attention_backward(A(x), A(x), A(x), A(x), A(g))[4].torch(), torch.zeros_like(state))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 4, 2, 128, 128), (64, 2, 2, 64, 64), (2, 6, 3, 40, 72), (1, 2, 1, 256, 256),
                                   (2, 3, 3, 7, 5), (1, 1, 1, 100, 130)], ids=str)
def test_attention_steps_are_the_row(ms, shape, dtype):
    """Steps from a state against the formula, several one after the other."""
    B, H, Hq, DK, DV = shape
    T = 4
    q, k, v = (rand(B, T, h, d, seed=i, dtype=dtype) for i, h, d in ((1, Hq, DK), (2, Hq, DK), (3, H, DV)))
    g = decays(B, T, H, seed=4)
    state = rand(B, H, DK, DV, seed=5)
    args = [x.double() for x in (q, k, v, g, state)]
    wo, ws = Q.attention(*args, DK ** -0.5)
    eo, es = Q.attention_bounds(*args, DK ** -0.5, torch.float32)
    A = ms.from_torch
    for t in range(T):
        o = ms.linear_attention_step(A(state), A(q[:, t]), A(k[:, t]), A(v[:, t]), A(g[:, t]))
        P.close(o.torch(), wo[:, t], eo[:, t], f"o {t}")
    P.close(state, ws, es, "state")


def test_attention_step_by_head_and_out(ms):
    B, H, D = 3, 2, 16
    A = ms.from_torch
    q, k, v = (rand(B, H, D, seed=i) for i in (1, 2, 3))
    g, s1 = decays(H, seed=4), rand(B, H, D, D, seed=5)
    s2 = s1.clone()
    out = ms.empty((B, H, D), "f32", "cuda:0")
    assert ms.linear_attention_step(A(s1), A(q), A(k), A(v), A(g), scale=2.0, out=out) is out
    o = ms.linear_attention_step(A(s2), A(q), A(k), A(v), A(g.expand(B, H)), scale=2.0)
    assert torch.equal(out.torch(), o.torch()) and torch.equal(s1, s2)


def test_attention_out(ms):
    A = ms.from_torch
    q, k, v = (rand(2, 70, 2, 16, seed=i, dtype="bf16") for i in (1, 2, 3))
    g = decays(2, 70, 2, seed=4)
    out = ms.empty((2, 70, 2, 16), "bf16", "cuda:0")
    assert ms.linear_attention(A(q), A(k), A(v), A(g), out=out) is out
    assert torch.equal(out.torch(), ms.linear_attention(A(q), A(k), A(v), A(g)).torch())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_repeats_its_bits(ms, dtype):
    A = ms.from_torch
    q, k = (A(rand(2, 1000, 2, 64, seed=i, dtype=dtype)) for i in (1, 2))
    v, g = A(rand(2, 1000, 4, 64, seed=3, dtype=dtype)), A(decays(2, 1000, 4, seed=4))
    s = A(rand(2, 4, 64, 64, seed=5))
    run = lambda: [x.torch().clone() for x in (*ms.linear_attention(q, k, v, g, s, return_state=True),
                                               *ms.linear_attention_backward(v, q, k, v, g, s, s))]
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_attention_gradients_are_differences(ms):
    """The gradients against differences of the kernel's own forward pass, along one direction for each input."""
    B, T, H, Hq, D = 1, 150, 2, 1, 16
    t = {"q": rand(B, T, Hq, D, seed=1), "k": rand(B, T, Hq, D, seed=2), "v": rand(B, T, H, D, seed=3),
         "log_decay": decays(B, T, H, seed=4), "state": rand(B, H, D, D, seed=5)}
    do, ds = rand(B, T, H, D, seed=6), rand(B, H, D, D, seed=7)
    A = ms.from_torch

    def value(t):
        o, s = ms.linear_attention(*(A(x) for x in t.values()), return_state=True)
        return float((o.torch().double() * do).sum() + (s.torch().double() * ds).sum())

    grads = dict(zip(t, ms.linear_attention_backward(A(do), *(A(x) for x in t.values()), A(ds))))
    for i, n in enumerate(t):
        way = rand(*t[n].shape, seed=20 + i)
        h = 2.0 ** -7 / float(way.abs().max())
        up, down = value({**t, n: t[n] + h * way}), value({**t, n: t[n] - h * way})
        want = float((grads[n].torch().double() * way).sum())
        # float results summed over 5000 values of about 4, over 2h: 1e-3 of the slopes' root sum of squares
        size = float((grads[n].torch().double() * way).norm())
        assert abs((up - down) / (2 * h) - want) < 0.02 * size + 1e-2 * abs(want), n


def test_attention_on_a_long_row(ms):
    """Many chunks, few heads: segments that are joined; against the same row with a whole number of heads more."""
    B, T, H, D = 1, 20000, 1, 64
    q, k, v = (rand(B, T, H, D, seed=i) for i in (1, 2, 3))
    g = decays(B, T, H, seed=4, mean=6.0)
    state, dstate, do = rand(B, H, D, D, seed=5), rand(B, H, D, D, seed=6), rand(B, T, H, D, seed=7)
    check_attention(ms, q, k, v, g, state, dstate, do)


# ---------------------------------------------------------- distillation
def check_distill(ms, z, ids, t, mask, tau=1.0, grad_scale=1.0):
    A = ms.from_torch
    m = torch.ones(z.shape[0], dtype=torch.bool, device="cuda") if mask is None else mask
    r = ms.distill_loss(A(z), A(ids), A(t), None if mask is None else A(mask), temperature=tau, grad_scale=grad_scale)
    (loss, kl, grad), (el, ek, eg) = Q.distill(z.double(), ids.long(), t.double(), m, tau, grad_scale)
    P.close(r.kl.torch(), kl, ek, "kl")
    P.close(r.loss.torch(), loss, el, "loss")
    P.close(r.dlogits.torch(), grad, eg, "dlogits")
    only = ms.distill_loss(A(z), A(ids), A(t), None if mask is None else A(mask), temperature=tau, grad=False)
    assert only.dlogits is None
    P.close(only.kl.torch(), kl, ek, "kl alone")  # another alignment may take another kernel: the same bound, not the same bits
    return r


def teacher(N, V, K, seed, dtype="f32"):
    ids = torch.stack([torch.randperm(V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed + i))[:K]
                       for i in range(N)])
    return ids, rand(N, K, seed=seed, std=2.0).to(TORCH[dtype])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V,K", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 1000, 20), (7, 1003, 64), (3, 4096, 1), (2, 33000, 100),
                                   (2, 140001, 8), (33, 520, 9), (2, 2048, 1024), (1, 270000, 5)], ids=str)
def test_distill(ms, N, V, K, dtype):
    ids, t = teacher(N, V, K, 5, dtype)
    check_distill(ms, rand(N, V, seed=1, std=2.0, dtype=dtype), ids, t, None)


@pytest.mark.parametrize("tau", [0.5, 2.0, 10.0])
@pytest.mark.parametrize("teacher_dtype,ids_dtype", [("f32", torch.int32), ("bf16", torch.int64), ("f16", torch.int32)])
def test_distill_temperature_and_types(ms, tau, teacher_dtype, ids_dtype):
    ids, t = teacher(6, 5000, 30, 3, teacher_dtype)
    mask = torch.tensor([True, False, True, True, False, True], device="cuda")
    check_distill(ms, rand(6, 5000, seed=1, std=3.0, dtype="bf16"), ids.to(ids_dtype), t, mask, tau, 0.25)


def test_distill_masked_rows_may_hold_anything(ms):
    z, (ids, t) = rand(4, 300, seed=1), teacher(4, 300, 5, 3)
    mask = torch.tensor([True, False, False, True], device="cuda")
    z[1], z[2, 3], t[1], ids[2] = math.nan, math.inf, math.nan, -5
    r = check_distill(ms, z, ids, t, mask)
    assert torch.equal(r.dlogits.torch()[1:3], torch.zeros(2, 300, device="cuda")) and r.loss.torch().isfinite()
    none = check_distill(ms, z, ids, t, torch.zeros(4, dtype=torch.bool, device="cuda"))
    assert float(none.loss.torch()) == 0.0 and torch.equal(none.dlogits.torch(), torch.zeros_like(z))


def test_distill_short_lists(ms):
    """Entries of -inf are left out, whatever their place; a token without entries adds nothing."""
    z, (ids, t) = rand(5, 400, seed=1), teacher(5, 400, 6, 3)
    t[0, 3:], t[1], t[2, :5] = -math.inf, -math.inf, -math.inf
    ids[0, 3:], ids[1] = -1, 1 << 40
    r = check_distill(ms, z, ids, t, None)
    assert float(r.kl.torch()[1]) == 0.0 and torch.equal(r.dlogits.torch()[1], torch.zeros(400, device="cuda"))


def test_distill_places_named_twice(ms):
    z = rand(3, 5000, seed=1)
    ids = torch.tensor([[7, 7, 9, 7], [0, 4999, 0, 4999], [1, 1, 1, 1]], device="cuda")
    check_distill(ms, z, ids, rand(3, 4, seed=2), None)


@pytest.mark.parametrize("V", [257, 4096, 40003])
def test_distill_bad_places_and_nan(ms, V):
    z, (ids, t) = rand(5, V, seed=1), teacher(5, V, 4, 3)
    ids[0, 2], ids[1, 0], t[2, 1] = V, -1, math.nan
    r = check_distill(ms, z, ids, t, None)
    assert r.kl.torch()[:3].isnan().all() and r.kl.torch()[3:].isfinite().all()


def test_distill_padded_vocabulary(ms):
    """-inf in the student's logits, the type's lowest value, and large ones."""
    z, (ids, t) = rand(4, 1000, seed=1, dtype="bf16"), teacher(4, 900, 8, 3)
    z[:2, 900:], z[2:, 900:] = -math.inf, torch.finfo(torch.bfloat16).min
    z[1] += 30000.0
    z[3, :900] += 1e6
    check_distill(ms, z, ids, t, None)
    r = ms.distill_loss(ms.from_torch(z), ms.from_torch(ids * 0 + 950), ms.from_torch(t))
    assert (r.kl.torch()[:2] == math.inf).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["odd rows", "odd offset", "rows apart", "columns outside"])
def test_distill_layouts(ms, kind, dtype):
    N, V = 6, 777
    z = {"odd rows": lambda: rand(N, V, seed=1, dtype=dtype), "odd offset": lambda: rand(N, V + 5, seed=1, dtype=dtype)[:, 3:V + 3],
         "rows apart": lambda: rand(2 * N, V + 1, seed=1, dtype=dtype)[::2, :V],
         "columns outside": lambda: rand(V, N, seed=1, dtype=dtype).t()}[kind]()
    ids, t = teacher(N, V, 10, 3)
    wide = torch.zeros(N, 20, device="cuda", dtype=torch.int64)
    wide[:, ::2] = ids
    check_distill(ms, z, wide[:, ::2], t.t().contiguous().t(), None)


def test_distill_many_rows(ms):
    """More tokens than a block counts for itself, in several leading dims."""
    N, V, K = 9000, 64, 3
    z, ids, t = rand(90, 100, V, seed=1), whole(0, V, 90, 100, K, seed=2), rand(90, 100, K, seed=3)
    mask = whole(0, 2, 90, 100, seed=4).bool()
    A = ms.from_torch
    r = ms.distill_loss(A(z), A(ids), A(t), A(mask))
    p = torch.softmax(t.double(), -1)
    logq = torch.log_softmax(z.double(), -1)
    kl = (p * (p.log() - logq.gather(-1, ids))).sum(-1) * mask
    count = int(mask.sum())
    grad = logq.exp().scatter_add_(-1, ids, -p) * mask[..., None] / count
    P.close(r.kl.torch(), kl, 1024 * Q.EPS32 * (1 + kl.abs()))
    P.close(r.loss.torch(), kl.sum() / count, 1024 * Q.EPS32 * (1 + kl.abs()).mean())
    P.close(r.dlogits.torch(), grad, 256 * Q.EPS32 / count)
    assert r.kl.shape == (90, 100) and r.dlogits.shape == (90, 100, V)


def test_distill_without_tokens_or_entries(ms):
    A = ms.from_torch
    r = ms.distill_loss(A(rand(0, 10, seed=1)), A(whole(0, 10, 0, 3, seed=2)), A(rand(0, 3, seed=3)))
    assert float(r.loss.torch()) == 0.0 and r.dlogits.shape == (0, 10)
    r = ms.distill_loss(A(rand(4, 10, seed=1)), A(whole(0, 10, 4, 0, seed=2)), A(rand(4, 0, seed=3)))
    assert float(r.loss.torch()) == 0.0 and torch.equal(r.dlogits.torch(), torch.zeros(4, 10, device="cuda"))
    z, ids, t = rand(10, seed=1), whole(0, 10, 3, seed=2), rand(3, seed=3)  # one token without a leading dim
    assert ms.distill_loss(A(z), A(ids), A(t)).kl.shape == ()


def test_distill_repeats_its_bits(ms):
    A = ms.from_torch
    ids, t = teacher(50, 30000, 20, 3)
    z = A(rand(50, 30000, seed=1, dtype="bf16"))
    first = ms.distill_loss(z, A(ids), A(t))
    for _ in range(3):
        r = ms.distill_loss(z, A(ids), A(t))
        assert all(torch.equal(a.torch(), b.torch()) for a, b in zip(first, r))


# ------------------------------------------------------------- embedding
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V,D", [(1, 1, 1), (5, 10, 3), (64, 1000, 256), (1000, 50, 769), (33, 7, 4096), (2, 5, 20000), (4000, 300, 8)],
                         ids=str)
@pytest.mark.parametrize("tokens_dtype", [torch.int64, torch.int32])
def test_embedding(ms, N, V, D, dtype, tokens_dtype):
    table, tokens = rand(V, D, seed=1, dtype=dtype), whole(0, V, N, seed=2, dtype=tokens_dtype)
    for scale in (1.0, math.sqrt(D)):
        o = ms.embedding(ms.from_torch(table), ms.from_torch(tokens), scale=scale).torch()
        want = table.double()[tokens.long()] * scale
        P.close(o, want, 2 * Q.EPS32 * want.abs())
        if scale == 1.0:
            assert torch.equal(o, table[tokens.long()])


def test_embedding_tokens_outside(ms):
    table = rand(10, 40, seed=1)
    tokens = torch.tensor([[0, -1, 9], [10, 1 << 40, 3]], device="cuda")
    o = ms.embedding(ms.from_torch(table), ms.from_torch(tokens)).torch()
    assert o.shape == (2, 3, 40)
    bad = torch.tensor([[False, True, False], [True, True, False]], device="cuda")
    assert o[bad].isnan().all() and torch.equal(o[~bad], table[tokens[~bad]])
    d = ms.embedding_backward(ms.from_torch(rand(2, 3, 40, seed=2)), ms.from_torch(tokens), rows=10).torch()
    assert d.isfinite().all() and int((d.abs().sum(1) > 0).sum()) == 3


@pytest.mark.parametrize("kind", ["odd offset", "rows apart", "columns outside", "one row", "reversed"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_embedding_layouts(ms, kind, dtype):
    V, D, N = 50, 96, 120
    make = {"odd offset": lambda n, s: rand(n, D + 3, seed=s, dtype=dtype)[:, 1:D + 1],
            "rows apart": lambda n, s: rand(2 * n, D, seed=s, dtype=dtype)[::2],
            "columns outside": lambda n, s: rand(D, n, seed=s, dtype=dtype).t(),
            "one row": lambda n, s: rand(1, D, seed=s, dtype=dtype).expand(n, D),
            "reversed": lambda n, s: rand(n, D, seed=s, dtype=dtype)}[kind]
    A = (lambda x: ms.flip(ms.from_torch(x), 0)) if kind == "reversed" else ms.from_torch
    see = (lambda x: x.flip(0)) if kind == "reversed" else (lambda x: x)
    table, dout, tokens = make(V, 1), make(N, 2), whole(0, V, 2 * N, seed=3)[::2]
    assert torch.equal(ms.embedding(A(table), ms.from_torch(tokens)).torch(), see(table)[tokens])
    got = ms.embedding_backward(A(dout), ms.from_torch(tokens), rows=V, scale=0.5).torch()
    want, e = Q.embedding_gradient(see(dout).double(), tokens, V, 0.5)
    P.close(got, want, e)


def tokens_of(kind, N, V, seed):
    if kind == "one":
        return torch.full((N,), V // 2, device="cuda")
    if kind == "few":
        return whole(0, min(V, 3), N, seed=seed)
    if kind == "frequent":
        u = torch.rand(N, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
        return (V * u**3).long().clamp(max=V - 1)
    if kind == "runs":  # lists around the length at which they are cut
        return (torch.arange(N, device="cuda") // 33) % V
    return whole(0, V, N, seed=seed)


@pytest.mark.parametrize("kind", ["spread", "one", "few", "frequent", "runs"])
@pytest.mark.parametrize("N,V,D,dtype", [(1, 5, 8, "f32"), (31, 4, 6, "f32"), (32, 3, 16, "bf16"), (33, 1, 64, "f16"), (100, 700, 33, "bf16"),
                                         (4097, 50257, 65, "f32"), (8192, 40, 24, "bf16"), (8193, 300, 72, "f32"),
                                         (20000, 1500, 40, "f16"), (30000, 300000, 8, "bf16"), (3000, 129, 4500, "bf16"),
                                         (70000, 520, 2, "f32")], ids=str)
def test_embedding_gradient(ms, kind, N, V, D, dtype):
    dout, tokens = rand(N, D, seed=1, dtype=dtype), tokens_of(kind, N, V, 2)
    A = ms.from_torch
    want, e = Q.embedding_gradient(dout.double(), tokens, V, 3.0)
    got = ms.embedding_backward(A(dout), A(tokens), rows=V, scale=3.0).torch()
    P.close(got, want, e, "new")
    into = rand(V, D, seed=3)
    before = into.clone()
    same = A(into)
    assert ms.embedding_backward(A(dout), A(tokens.int()), scale=3.0, into=same) is same
    P.close(into, want + before.double(), e + 2 * Q.EPS32 * (want.abs() + before.double().abs()), "into")
    idle = torch.ones(V, dtype=torch.bool, device="cuda")
    idle[tokens] = False
    assert torch.equal(into[idle], before[idle]) and (got[idle] == 0).all()
    assert torch.equal(ms.embedding_backward(A(dout), A(tokens), rows=V, scale=3.0).torch(), got)


def test_embedding_gradient_empty(ms):
    A = ms.from_torch
    none = whole(0, 5, 0, seed=1)
    assert torch.equal(ms.embedding_backward(A(rand(0, 4, seed=1)), A(none), rows=3).torch(), torch.zeros(3, 4, device="cuda"))
    into = rand(3, 4, seed=2)
    before = into.clone()
    ms.embedding_backward(A(rand(0, 4, seed=1)), A(none), into=A(into))
    assert torch.equal(into, before)
    assert ms.embedding_backward(A(rand(7, 4, seed=1)), A(whole(0, 5, 7, seed=1)), rows=0).shape == (0, 4)
    assert ms.embedding(A(rand(5, 0, seed=1)), A(whole(0, 5, 7, seed=1))).shape == (7, 0)
    assert ms.embedding(A(rand(0, 6, seed=1)), A(whole(0, 5, 7, seed=1))).torch().isnan().all()
    assert ms.embedding(A(rand(5, 6, seed=1)), A(none)).shape == (0, 6)
    one = ms.embedding(A(rand(5, 6, seed=1)), A(torch.tensor(3, device="cuda")))
    assert one.shape == (6,)
    assert torch.equal(ms.embedding_backward(one, A(torch.tensor(3, device="cuda")), rows=5).torch()[3], one.torch())


# ------------------------------------------------- streams, graphs, several together
def _model(ms, t):
    """Tokens through the embedding, linear attention and distillation, forward and backward."""
    A = ms.from_torch
    x = ms.embedding(A(t["table"]), A(t["tokens"]), scale=2.0)
    B, T, D = x.shape
    H = t["g"].shape[-1]
    heads = ms.reshape(x, (B, T, H, D // H))
    o, s = ms.linear_attention(heads, heads, heads, A(t["g"]), A(t["state"]), return_state=True)
    r = ms.distill_loss(ms.reshape(o, (B, T, D)), A(t["ids"]), A(t["teacher"]), A(t["mask"]))
    do = ms.reshape(r.dlogits, (B, T, H, D // H))
    dq, dk, dv, dg, ds = ms.linear_attention_backward(do, heads, heads, heads, A(t["g"]), A(t["state"]))
    dx = ms.add(ms.add(dq, dk), dv)
    dtable = ms.embedding_backward(ms.reshape(dx, (B, T, D)), A(t["tokens"]), rows=t["table"].shape[0], scale=2.0)
    step = ms.linear_attention_step(A(t["running"]), *[ms.from_torch(heads.torch()[:, 0])] * 3, ms.from_torch(t["g"][:, 0]))
    return [y.torch() for y in (r.loss, r.kl, r.dlogits, dg, ds, dtable, step, s)]


def _model_inputs(seed=0, B=2, T=150, H=4, D=64, V=90):
    return {"table": rand(V, D, seed=seed + 1), "tokens": whole(0, V, B, T, seed=seed + 2), "g": decays(B, T, H, seed=seed + 3),
            "state": rand(B, H, D // H, D // H, seed=seed + 4), "ids": whole(0, D, B, T, 5, seed=seed + 5),
            "teacher": rand(B, T, 5, seed=seed + 6), "mask": whole(0, 4, B, T, seed=seed + 7) > 0,
            "running": rand(B, H, D // H, D // H, seed=seed + 8)}


def test_model_gradient_is_autograds(ms):
    """The operators run together as a model does, its table's gradient against autograd in 64 bits."""
    t = _model_inputs()
    got = _model(ms, dict(t, running=t["running"].clone()))
    table = t["table"].double().requires_grad_()
    g = t["g"].double().requires_grad_()
    x = table[t["tokens"]] * 2.0
    B, T, D = x.shape
    H = g.shape[-1]
    h = x.unflatten(-1, (H, D // H))
    o, s = Q.attention(h, h, h, g, t["state"].double(), (D // H) ** -0.5)
    z = o.flatten(2)
    p = torch.softmax(t["teacher"].double(), -1)
    kl = (p * (p.log() - torch.log_softmax(z, -1).gather(-1, t["ids"]))).sum(-1) * t["mask"]
    loss = kl.sum() / t["mask"].sum()
    want = torch.autograd.grad(loss, (table, g))
    assert abs(float(got[0]) - float(loss.detach())) < 1e-5 * (1 + abs(float(loss.detach())))
    # float all the way, a few hundred roundings of values that cancel by less than ten: 1e-4 of the largest
    assert (got[5].double() - want[0]).abs().max() < 1e-4 * want[0].abs().max()
    assert (got[3].double() - want[1]).abs().max() < 1e-4 * want[1].abs().max()


def test_model_on_a_stream_and_in_a_graph(ms):
    t = _model_inputs()
    want = [x.clone() for x in _model(ms, dict(t, running=t["running"].clone()))]
    stream = ms.Stream("cuda:0")
    with ms.stream(stream):
        got = _model(ms, dict(t, running=t["running"].clone()))
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    buffers = {k: v.clone() for k, v in t.items()}
    with torch.cuda.stream(side):
        _model(ms, dict(buffers, running=buffers["running"].clone()))
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs, each with scratch of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            graphs.append((graph, _model(ms, buffers)))
    for seed in (0, 50):
        new = _model_inputs(seed)
        expect = _model(ms, dict(new, running=new["running"].clone()))
        for graph, outs in graphs:
            for k in buffers:
                buffers[k].copy_(new[k])
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(expect, outs))


def test_model_on_two_streams_at_once(ms):
    """Two models' calls interleaved on two streams: no workspace is shared."""
    inputs = [_model_inputs(0), _model_inputs(50)]
    want = [[x.clone() for x in _model(ms, dict(t, running=t["running"].clone()))] for t in inputs]
    streams = [ms.Stream("cuda:0"), ms.Stream("cuda:0")]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, t in zip(streams, inputs):
            with ms.stream(s):
                got.append(_model(ms, dict(t, running=t["running"].clone())))
    for s in streams:
        s.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(want[i % 2], g))
