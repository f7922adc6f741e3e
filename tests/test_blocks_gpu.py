"""The block operators on the GPU against their formulas in 64 bits, at the sizes, layouts and masks where they can go
wrong. Tolerances are the bounds that blocks_plain derives."""
import math

import pytest
import torch

from . import blocks_plain as P

pytestmark = pytest.mark.gpu

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rand(*shape, seed, dtype="f32", std=1.0, mean=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * std + mean).to(TORCH[dtype])


def gates(B, T, H, mode, dtype, seed):
    g = rand(B, T, H, seed=seed, std=1.5, mean=2.0)
    return g.to(TORCH[dtype]) if mode == "sigmoid" else torch.sigmoid(g).to(TORCH[dtype])


def check_scan(ms, x, gate, h0, mode, what=""):
    """Forward, backward and (T == 1) step of torch tensors of any layout."""
    A = ms.from_torch
    opt = lambda t: None if t is None else A(t)
    B, T, D = x.shape
    h, last = ms.gated_scan(A(x), A(gate), opt(h0), mode=mode, return_state=True)
    d = lambda t: None if t is None else t.double()
    wh, wl, eh, el = P.scan(d(x), d(gate), d(h0), mode)
    P.close(h.torch(), wh, eh, f"{what} h")
    P.close(last.torch(), wl, el, f"{what} state")
    dh, dstate = rand(B, T, D, seed=77).to(x.dtype), rand(B, D, seed=78)
    got = ms.gated_scan_backward(A(dh), A(x), A(gate), h, opt(h0), A(dstate), mode=mode)
    want, err = P.scan_backward(d(dh), d(x), d(gate), h.torch().double(), d(h0), d(dstate), mode)
    for g, w, e, n in zip(got, want, err, ("dx", "dgate", "dh0")):
        P.close(g.torch(), w, e, f"{what} {n}")
    assert got[1].torch().dtype == gate.dtype and got[2].torch().dtype == torch.float32


SHAPES = [  # B, T, D, H
    (1, 1, 1, 1), (2, 1, 64, 64), (3, 7, 5, 5), (1, 2, 63, 63), (2, 129, 33, 33), (1, 1000, 70, 70), (4, 513, 256, 256),
    (1, 5000, 8, 8), (1, 2049, 66, 66), (300, 33, 130, 130), (2, 257, 96, 6), (1, 300, 160, 2), (2, 65, 128, 1),
    (4, 513, 256, 4), (2, 100, 7, 1), (1, 1025, 48, 3), (1, 70, 1040, 4), (33, 64, 24, 12),
]


@pytest.mark.parametrize("mode", ["linear", "sigmoid"])
@pytest.mark.parametrize("dtype,gate_dtype", [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"),
                                              ("f16", "f32")])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan(ms, shape, dtype, gate_dtype, mode):
    B, T, D, H = shape
    check_scan(ms, rand(B, T, D, seed=1, dtype=dtype), gates(B, T, H, mode, gate_dtype, 2), rand(B, D, seed=3), mode)


def _odd_views(B, T, D, H, dtype, kind):
    """x (B, T, D) and gate (B, T, H) in other layouts."""
    def view(n, seed):
        if kind == "time first":
            return rand(T, B, n, seed=seed, dtype=dtype).permute(1, 0, 2)
        if kind == "odd offset":  # rows that start at any multiple of the element size
            return rand(B, T, n + 3, seed=seed, dtype=dtype)[:, :, 1:n + 1]
        if kind == "channels outside":
            return rand(B, n, T, seed=seed, dtype=dtype).permute(0, 2, 1)
        if kind == "every second step":
            return rand(B, 2 * T, n, seed=seed, dtype=dtype)[:, ::2]
        return rand(1, T, n, seed=seed, dtype=dtype).expand(B, T, n)  # one sequence for the whole batch
    return view(D, 5), view(H, 6)


@pytest.mark.parametrize("kind", ["time first", "odd offset", "channels outside", "every second step", "broadcast"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H", [68, 4])
def test_scan_layouts(ms, kind, dtype, H):
    x, gate = _odd_views(3, 150, 68, H, dtype, kind)
    check_scan(ms, x, gate, rand(3, 68, seed=3), "sigmoid", kind)


def test_scan_reversed_view(ms):
    """Negative strides: the recurrence over the flipped time axis."""
    x, g = rand(2, 77, 40, seed=1), gates(2, 77, 40, "linear", "f32", 2)
    h = ms.gated_scan(ms.flip(ms.from_torch(x), 1), ms.flip(ms.from_torch(g), 1))
    want, _, e, _ = P.scan(x.flip(1).double(), g.flip(1).double(), None, "linear")
    P.close(h.torch(), want, e)


@pytest.mark.parametrize("shape", [(2, 0, 5), (0, 4, 5), (2, 4, 0)])
def test_scan_empty(ms, shape):
    B, T, D = shape
    x, h0, ds = rand(B, T, D, seed=1), rand(B, D, seed=2), rand(B, D, seed=3)
    A = ms.from_torch
    h, last = ms.gated_scan(A(x), A(x), A(h0), return_state=True)
    assert h.shape == shape and torch.equal(last.torch(), h0)
    dx, dg, dh0 = ms.gated_scan_backward(A(x), A(x), A(x), h, A(h0), A(ds))
    assert dx.shape == dg.shape == shape and torch.equal(dh0.torch(), ds)
    _, last = ms.gated_scan(A(x), A(x), return_state=True)
    assert torch.equal(last.torch(), torch.zeros_like(h0)) or T > 0


def test_scan_without_batch_and_out(ms):
    x, g, h0 = rand(50, 12, seed=1, dtype="f16"), gates(1, 50, 12, "sigmoid", "f16", 2)[0], rand(12, seed=3)
    out = ms.empty((50, 12), "f16", "cuda:0")
    h, last = ms.gated_scan(ms.from_torch(x), ms.from_torch(g), ms.from_torch(h0), mode="sigmoid", return_state=True, out=out)
    assert h is out and last.shape == (12,)
    full, flast = ms.gated_scan(ms.from_torch(x[None]), ms.from_torch(g[None]), ms.from_torch(h0[None]), mode="sigmoid",
                                return_state=True)
    assert torch.equal(h.torch(), full.torch()[0]) and torch.equal(last.torch(), flast.torch()[0])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,T,D", [(1, 1000, 70), (1, 300, 33), (2, 4000, 64), (1, 6000, 1), (120, 500, 64)])
def test_scan_carries_the_first_state_undiminished(ms, B, T, D, dtype):
    """Gates of one and no input: every state is the first one, whichever pieces a long sequence was joined from and
    however early they met; backward every gradient is that of the last state."""
    A = ms.from_torch
    one, zero = torch.ones(B, T, D, dtype=TORCH[dtype], device="cuda"), torch.zeros(B, T, D, dtype=TORCH[dtype], device="cuda")
    h0 = rand(B, D, seed=1)
    want = h0.to(TORCH[dtype])[:, None].expand(B, T, D)
    for _ in range(20):
        h, last = ms.gated_scan(A(zero), A(one), A(h0), return_state=True)
        assert torch.equal(h.torch(), want) and torch.equal(last.torch(), h0)
        dx, _, dh0 = ms.gated_scan_backward(A(zero), A(zero), A(one), h, A(h0), A(h0))
        assert torch.equal(dx.torch(), want) and torch.equal(dh0.torch(), h0)


@pytest.mark.parametrize("T", [5, 700, 20000])
def test_scan_restarts_where_the_gate_is_zero(ms, T):
    """Sequences packed along time: a zero gate drops what came before it, in every layout of the pieces."""
    x, g = rand(1, T, 40, seed=1), gates(1, T, 40, "linear", "f32", 2)
    cut = T // 2 + 1
    g[:, cut] = 0.0
    h = ms.gated_scan(ms.from_torch(x), ms.from_torch(g)).torch()
    second = ms.gated_scan(ms.from_torch(x[:, cut:].contiguous()), ms.from_torch(g[:, cut:].contiguous())).torch()
    want, _, e, _ = P.scan(x[:, cut:].double(), g[:, cut:].double(), None, "linear")
    P.close(h[:, cut:].contiguous(), want, e)
    P.close(second, want, e)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_scan_extreme_gates(ms, dtype):
    """Gates at the ends of the sigmoid (infinities, the type's extremes) keep or replace the state; a NaN stays in its
    channel from its step on."""
    big = torch.finfo(TORCH[dtype]).max
    x, g = rand(2, 300, 36, seed=1, dtype=dtype), gates(2, 300, 36, "sigmoid", dtype, 2)
    g[:, 10], g[:, 20], g[:, 30], g[:, 200] = math.inf, -math.inf, big, -big
    check_scan(ms, x, g, rand(2, 36, seed=3), "sigmoid")
    x[0, 100, 7] = math.nan
    h = ms.gated_scan(ms.from_torch(x), ms.from_torch(g), mode="sigmoid").torch()
    nan = torch.zeros(2, 300, 36, dtype=torch.bool, device="cuda")
    want, _, _, _ = P.scan(x.double(), g.double(), None, "sigmoid")
    assert torch.equal(h.isnan(), want.isnan()) and bool(h[0, 100, 7].isnan()) and not bool(h[1].isnan().any())


@pytest.mark.parametrize("B,D,H", [(1, 1, 1), (3, 65, 65), (64, 4096, 4096), (7, 96, 6), (130, 1001, 1001)])
@pytest.mark.parametrize("dtype,gate_dtype", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("mode", ["linear", "sigmoid"])
def test_scan_steps_are_the_scan(ms, B, D, H, dtype, gate_dtype, mode):
    """Three single steps update the state in place and give what the formula gives for three tokens."""
    x, g, h0 = rand(B, 3, D, seed=1, dtype=dtype), gates(B, 3, H, mode, gate_dtype, 2), rand(B, D, seed=3)
    want, wl, e, el = P.scan(x.double(), g.double(), h0.double(), mode)
    state = ms.from_torch(h0.clone())
    for t in range(3):
        out = ms.empty((B, D), dtype, "cuda:0") if t == 1 else None
        h = ms.gated_scan_step(state, ms.from_torch(x[:, t]), ms.from_torch(g[:, t]), mode=mode, out=out)
        assert out is None or h is out
        P.close(h.torch(), want[:, t], e[:, t], f"step {t}")
    P.close(state.torch(), wl, el, "state")


def test_scan_gradient_is_differences(ms):
    """The kernel's gradient along a direction against central differences of the 64-bit forward."""
    B, T, D, H = 2, 70, 12, 3
    x, g, h0 = rand(B, T, D, seed=1), gates(B, T, H, "sigmoid", "f32", 2), rand(B, D, seed=3)
    dh, ds = rand(B, T, D, seed=4), rand(B, D, seed=5)
    A = ms.from_torch
    h = ms.gated_scan(A(x), A(g), A(h0), mode="sigmoid")
    grads = ms.gated_scan_backward(A(dh), A(x), A(g), h, A(h0), A(ds), mode="sigmoid")
    dirs = [rand(*t.shape, seed=10 + i).double() for i, t in enumerate((x, g, h0))]

    def loss(s):
        hh, last, _, _ = P.scan(x.double() + s * dirs[0], g.double() + s * dirs[1], h0.double() + s * dirs[2], "sigmoid")
        return float((hh * dh.double()).sum() + (last * ds.double()).sum())

    want = (loss(1e-4) - loss(-1e-4)) / 2e-4
    got = sum(float((a.torch().double() * d).sum()) for a, d in zip(grads, dirs))
    size = sum(float((a.torch().double() * d).abs().sum()) for a, d in zip(grads, dirs))
    # float gradients to 1e-5 of their size; the step's third-order term is below 1e-7 of it
    assert abs(got - want) < 1.1e-5 * size


def test_scan_is_repeatable(ms):
    """The same bits every time, whichever way the pieces of a long sequence meet."""
    x, g = rand(1, 30000, 200, seed=1), gates(1, 30000, 200, "linear", "f32", 2)
    a = [ms.gated_scan(ms.from_torch(x), ms.from_torch(g)).torch() for _ in range(5)]
    assert all(torch.equal(a[0], b) for b in a[1:])
    gh = gates(1, 30000, 2, "linear", "f32", 3)
    r = [ms.gated_scan_backward(ms.from_torch(x), ms.from_torch(x), ms.from_torch(gh), ms.from_torch(a[0])) for _ in range(5)]
    for other in r[1:]:
        assert all(torch.equal(p.torch(), q.torch()) for p, q in zip(r[0], other))


def test_scan_offsets_beyond_32_bits(ms):
    """Sequences 2^31 + 2 elements apart (8 GiB of float16)."""
    gap = (1 << 31) + 2
    buf = torch.empty(gap + 4096, dtype=torch.float16, device="cuda")
    x = torch.as_strided(buf, (2, 64, 50), (gap, 50, 1))
    x.copy_(rand(2, 64, 50, seed=1))
    check_scan(ms, x, gates(2, 64, 50, "sigmoid", "f16", 2), None, "sigmoid")


def test_scan_long(ms):
    """A sequence over 2^31 / 256 steps long in one channel block: 2^23 + 5 steps."""
    T, D = (1 << 23) + 5, 3
    x, g = rand(1, T, D, seed=1), torch.full((1, T, D), 0.5, device="cuda")
    h, last = ms.gated_scan(ms.from_torch(x), ms.from_torch(g), return_state=True)
    h = h.torch()
    # with a decay of one half a step is settled by the 60 before it
    w = (0.5 ** torch.arange(60, dtype=torch.float64, device="cuda")).flip(0)
    for at in (59, 1000, T // 2, T - 1):
        win = x[0, at - 59:at + 1].double()
        want = (win * w[:, None]).sum(0)
        P.close(h[0, at], want, 16 * P.EPS32 * 2 * (win.abs() * w[:, None]).sum(0) + 2.0 ** -55)
    assert torch.equal(last.torch()[0], h[0, -1])


# --------------------------------------------------------------- dropout
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 63, 1000, 4096 * 37 + 5])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0 - 2.0 ** -16, 1.0])
def test_dropout(ms, dtype, n, p):
    """Bit for bit: the kept elements are x times the factor in float, rounded once."""
    x = rand(n, seed=n, dtype=dtype)
    seed, offset = 0x123456789ABCDEF0 + n, 0xF0000000_00000001
    kept, up = P.keep_mask((n,), p, seed, offset, "cuda")
    want = torch.where(kept, x.float() * up, 0.0).to(x.dtype)
    got = ms.dropout(ms.from_torch(x), p, seed, offset).torch()
    assert torch.equal(got, want)


def test_dropout_masks_infinities_and_nan(ms):
    x = torch.tensor([math.inf, -math.inf, math.nan, 1.0] * 64, device="cuda")
    kept, up = P.keep_mask((256,), 0.5, 3, 4, "cuda")
    got = ms.dropout(ms.from_torch(x), 0.5, 3, 4).torch()
    assert bool((got[~kept] == 0).all()) and torch.equal(got[kept].isnan(), x[kept].isnan())
    assert torch.equal(got[kept & x.isinf()], x[kept & x.isinf()])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_dropout_layouts_count_in_c_order(ms, dtype):
    x = rand(40, 33, seed=1, dtype=dtype)
    kept, up = P.keep_mask((33, 40), 0.3, 9, 0, "cuda")
    want = torch.where(kept, x.t().float() * up, 0.0).to(x.dtype)
    assert torch.equal(ms.dropout(ms.transpose(ms.from_torch(x)), 0.3, 9).torch(), want)
    flat = rand(1003, seed=2, dtype=dtype)  # a start that no vector load may use
    kept, up = P.keep_mask((1000,), 0.3, 9, 1, "cuda")
    want = torch.where(kept, flat[3:].float() * up, 0.0).to(flat.dtype)
    out = ms.empty((1000,), dtype, "cuda:0")
    assert ms.dropout(ms.from_torch(flat[3:]), 0.3, 9, 1, out=out) is out and torch.equal(out.torch(), want)
    assert ms.dropout(ms.from_torch(x[:0]), 0.3, 9).shape == (0, 33)


def test_dropout_share_and_independence(ms):
    """Over 2^24 elements the dropped share is within 5 standard deviations of p; two offsets agree as independent
    masks do."""
    one = ms.ones((1 << 24,), "f32", "cuda:0")
    a = ms.dropout(one, 0.1, 1, 0).torch() != 0
    b = ms.dropout(one, 0.1, 1, 1).torch() != 0
    p = math.floor(0.1 * 65536 + 0.5) / 65536
    for share, q in (((~a).float().mean().item(), p), ((~a & ~b).float().mean().item(), p * p)):
        assert abs(share - q) < 5 * math.sqrt(q * (1 - q) / (1 << 24)) + 2.0 ** -24


def test_dropout_beyond_32_bits(ms):
    """2^32 + 24 elements: the last ones use counters above 2^29."""
    n = (1 << 32) + 24
    x = torch.ones(n, dtype=torch.float16, device="cuda")
    got = ms.dropout(ms.from_torch(x), 0.5, 5, 6).torch()
    for first in (0, (1 << 31) - 100, (1 << 32) - 100):
        m = min(200, n - first)
        want = torch.from_numpy(P.bits16(5, 6, first, m) >= 32768).cuda()
        assert torch.equal(got[first:first + m] != 0, want)


# ----------------------------------------------------------------- norms
def make_norm(R, D, dtype, kind, p, seed=0):
    shape = {"full": (R, D), "row": (R, 1), "channel": (D,), "none": None}[kind]
    t = {"x": rand(R, D, seed=seed + 1, dtype=dtype, std=2.0), "z": rand(R, D, seed=seed + 2, dtype=dtype, std=0.7),
         "w_post": rand(D, seed=seed + 3, std=0.1, mean=1.0), "w_pre": rand(D, seed=seed + 4, std=0.1, mean=1.0),
         "gate": None if shape is None else rand(*shape, seed=seed + 5, dtype=dtype),
         "dy": rand(R, D, seed=seed + 6, dtype=dtype), "du": rand(R, D, seed=seed + 7, dtype=dtype)}
    if p:
        kept, up = P.keep_mask((R, D), p, 11, 12, "cuda")
        t["m"] = torch.where(kept, up * 0.5, 0.0).double()
    else:
        t["m"] = torch.full((R, D), 0.5, dtype=torch.float64, device="cuda")
    return t


def check_norm(ms, t, activation, p, dy=True, du=True, lead=None):
    A = lambda v: None if v is None else ms.from_torch(v)
    d = lambda v: None if v is None else v.double()
    R, D = t["x"].shape
    how = dict(gate=A(t["gate"]), activation=activation, scale=0.5, dropout=p, seed=11, offset=12)
    y, u, rstd = ms.gated_residual_norm(A(t["x"]), A(t["z"]), A(t["w_post"]), A(t["w_pre"]), eps=1e-5, **how)
    (wy, wu, rz, ry), (ey, eu, er) = P.norm(d(t["x"]), d(t["z"]), d(t["w_post"]), d(t["w_pre"]), d(t["gate"]), activation,
                                            0.5, 1e-5, t["m"])
    P.close(y.torch(), wy, ey, "y")
    P.close(u.torch(), wu, eu, "u")
    P.close(rstd.torch()[0], rz[:, 0], (32 + D / 32) * P.EPS32 * rz[:, 0], "rstd of z")
    P.close(rstd.torch()[1], ry[:, 0], er[:, 0] * ry[:, 0], "rstd of y")
    gy, gu = t["dy"] if dy else None, t["du"] if du else None
    dx, dz, dg, dpost, dpre = ms.gated_residual_norm_backward(A(gy), A(gu), y, A(t["z"]), A(t["w_post"]), A(t["w_pre"]),
                                                              rstd, **how)
    r = rstd.torch().double()
    out, err = P.norm_backward(d(gy), d(gu), y.torch().double(), d(t["z"]), d(t["w_post"]), d(t["w_pre"]), r[0][:, None],
                               r[1][:, None], d(t["gate"]), activation, t["m"])
    P.close(dx.torch(), out["dx"], err["dx"], "dx")
    P.close(dz.torch(), out["dz"], err["dz"], "dz")
    col = lambda k: (out[k].sum(0), err[k].sum(0) + (R + 8) * P.EPS32 * out[k].abs().sum(0))
    P.close(dpost.torch(), *col("post"), "dw_post")
    P.close(dpre.torch(), *col("pre"), "dw_pre")
    if t["gate"] is None:
        assert dg is None
    elif t["gate"].shape == t["x"].shape:
        P.close(dg.torch(), out["gate"], err["gate"], "dgate")
    elif t["gate"].shape == (R, 1):
        P.close(dg.torch(), out["gate"].sum(1, keepdim=True),
                err["gate"].sum(1, keepdim=True) + (D + 8) * P.EPS32 * out["gate"].abs().sum(1, keepdim=True), "dgate")
    else:
        P.close(dg.torch(), *col("gate"), "dgate")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind,activation,p", [("full", "silu", 0.0), ("full", "sigmoid", 0.1), ("row", "silu", 0.3),
                                               ("channel", "linear", 0.0), ("channel", "silu", 0.5), ("none", "linear", 0.1),
                                               ("row", "linear", 0.0)])
@pytest.mark.parametrize("R,D", [(1, 1), (3, 7), (1, 64), (5, 100), (300, 128), (37, 1031), (9, 2048), (2, 4096), (700, 40),
                                 (3, 8192), (2, 9001), (1, 20000), (1, 40004)])
def test_norm(ms, R, D, dtype, kind, activation, p):
    check_norm(ms, make_norm(R, D, dtype, kind, p), activation, p)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["row gap", "odd start", "transposed", "one row for all", "channels apart"])
def test_norm_layouts(ms, dtype, layout):
    R, D = 21, 264
    t = make_norm(R, D, dtype, "full", 0.2)

    def view(v):
        if layout == "row gap":
            w = torch.zeros(R, D + 24, dtype=v.dtype, device="cuda")
            w[:, :D] = v
            return w[:, :D]
        if layout == "odd start":
            w = torch.zeros(R, D + 3, dtype=v.dtype, device="cuda")
            w[:, 1:D + 1] = v
            return w[:, 1:D + 1]
        if layout == "transposed":
            return v.t().contiguous().t()
        if layout == "channels apart":
            w = torch.zeros(R, 2 * D, dtype=v.dtype, device="cuda")
            w[:, ::2] = v
            return w[:, ::2]
        return v[:1].expand(R, D)

    for k in ("x", "z", "gate", "dy", "du"):
        t[k] = view(t[k])
    check_norm(ms, t, "silu", 0.2)


@pytest.mark.parametrize("dy,du", [(True, False), (False, True)])
def test_norm_with_one_gradient(ms, dy, du):
    check_norm(ms, make_norm(33, 520, "f32", "full", 0.1), "sigmoid", 0.1, dy, du)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(5, 7, 48), (1000, 33), (64,), (2, 3, 1), (4, 12000)])
def test_rms_norm(ms, dtype, shape):
    D = shape[-1]
    x, du, dy = (rand(*shape, seed=i, dtype=dtype) for i in range(3))
    w = rand(D, seed=5, mean=1.0, std=0.2)
    A = ms.from_torch
    u, rstd = ms.rms_norm(A(x), A(w), eps=1e-5)
    assert u.shape == shape and rstd.shape == shape[:-1]
    flat = lambda v: v.double().reshape(-1, D)
    (_, wu, _, ry), (_, eu, er) = P.norm(flat(x), None, None, w.double(), None, "linear", 1.0, 1e-5, None)
    P.close(u.torch().reshape(-1, D), wu, eu, "u")
    r = rstd.torch().reshape(-1)
    P.close(r, ry[:, 0], er[:, 0] * ry[:, 0], "rstd")
    for add in (None, dy):
        dx, dw = ms.rms_norm_backward(A(du), A(x), A(w), rstd, None if add is None else A(add))
        out, err = P.norm_backward(None if add is None else flat(add), flat(du), flat(x), None, None, w.double(), None,
                                   r.double()[:, None], None, "linear", None)
        P.close(dx.torch().reshape(-1, D), out["dx"], err["dx"], "dx")
        n = out["pre"].shape[0]
        P.close(dw.torch(), out["pre"].sum(0), err["pre"].sum(0) + (n + 8) * P.EPS32 * out["pre"].abs().sum(0), "dw")


def test_norm_empty_and_zero_rows(ms):
    A = ms.from_torch
    w = rand(8, seed=1)
    y, u, rstd = ms.gated_residual_norm(A(rand(0, 8, seed=1)), A(rand(0, 8, seed=1)), A(w), A(w))
    assert y.shape == u.shape == (0, 8) and rstd.shape == (2, 0)
    z = rand(0, 8, seed=1)
    out = ms.gated_residual_norm_backward(A(z), A(z), y, A(z), A(w), A(w), rstd, gate=A(w))
    assert out[0].shape == (0, 8) and all(bool((v.torch() == 0).all()) for v in out[2:])
    e = rand(3, 0, seed=1)
    w0 = rand(0, seed=1)
    y, u, rstd = ms.gated_residual_norm(A(e), A(e), A(w0), A(w0))
    out = ms.gated_residual_norm_backward(A(e), A(e), y, A(e), A(w0), A(w0), rstd, gate=A(rand(3, 1, seed=1)))
    assert out[0].shape == (3, 0) and out[2].shape == (3, 1) and bool((out[2].torch() == 0).all())
    zero = torch.zeros(4, 64, device="cuda")
    u, rstd = ms.rms_norm(A(zero), A(rand(64, seed=2)), eps=1e-6)
    assert bool((u.torch() == 0).all()) and torch.allclose(rstd.torch(), torch.full((4,), 1e3, device="cuda"))


def test_norm_dropped_branch_is_not_read(ms):
    """An infinity or a NaN of the gate in a dropped place does not reach the stream nor the gradients of the gate."""
    t = make_norm(4, 96, "f32", "full", 0.5)
    dropped = t["m"] == 0
    t["gate"][dropped] = math.nan
    A = ms.from_torch
    how = dict(gate=A(t["gate"]), activation="linear", scale=0.5, dropout=0.5, seed=11, offset=12)
    y, u, rstd = ms.gated_residual_norm(A(t["x"]), A(t["z"]), A(t["w_post"]), A(t["w_pre"]), **how)
    assert torch.equal(y.torch()[dropped], t["x"][dropped]) and not bool(u.torch().isnan().any())
    out = ms.gated_residual_norm_backward(A(t["dy"]), A(t["du"]), y, A(t["z"]), A(t["w_post"]), A(t["w_pre"]), rstd, **how)
    assert bool((out[2].torch()[dropped] == 0).all()) and not any(bool(v.torch().isnan().any()) for v in out)


def test_norm_is_repeatable(ms):
    t = make_norm(5000, 1000, "bf16", "channel", 0.1)
    A = ms.from_torch
    how = dict(gate=A(t["gate"]), activation="silu", scale=0.5, dropout=0.1, seed=11, offset=12)
    y, u, rstd = ms.gated_residual_norm(A(t["x"]), A(t["z"]), A(t["w_post"]), A(t["w_pre"]), **how)
    runs = [ms.gated_residual_norm_backward(A(t["dy"]), A(t["du"]), y, A(t["z"]), A(t["w_post"]), A(t["w_pre"]), rstd, **how)
            for _ in range(4)]
    for other in runs[1:]:
        assert all(torch.equal(a.torch(), b.torch()) for a, b in zip(runs[0], other))


def test_norm_gradient_is_differences(ms):
    R, D = 6, 50
    t = make_norm(R, D, "f32", "full", 0.3)
    A = ms.from_torch
    how = dict(gate=A(t["gate"]), activation="silu", scale=0.5, dropout=0.3, seed=11, offset=12)
    y, u, rstd = ms.gated_residual_norm(A(t["x"]), A(t["z"]), A(t["w_post"]), A(t["w_pre"]), eps=1e-6, **how)
    dx, dz, dg, dpost, dpre = ms.gated_residual_norm_backward(A(t["dy"]), A(t["du"]), y, A(t["z"]), A(t["w_post"]),
                                                              A(t["w_pre"]), rstd, **how)
    names = ("x", "z", "gate", "w_post", "w_pre")
    dirs = {k: rand(*t[k].shape, seed=40 + i).double() for i, k in enumerate(names)}

    def loss(s):
        v = {k: t[k].double() + s * dirs[k] for k in names}
        (yy, uu, _, _), _ = P.norm(v["x"], v["z"], v["w_post"], v["w_pre"], v["gate"], "silu", 0.5, 1e-6, t["m"])
        return float((yy * t["dy"].double()).sum() + (uu * t["du"].double()).sum())

    want = (loss(1e-4) - loss(-1e-4)) / 2e-4
    parts = [a.torch().double() * dirs[k] for a, k in zip((dx, dz, dg, dpost, dpre), names)]
    assert abs(float(sum(q.sum() for q in parts)) - want) < 1.1e-5 * float(sum(q.abs().sum() for q in parts))


# ---------------------------------------------------------------- policy
def make_policy(N, V, dtype, masked, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + 100)
    z = rand(N, V, seed=seed + 1, dtype=dtype, std=2.0)
    t = torch.randint(0, V, (N,), device="cuda", generator=g)
    z[torch.arange(N, device="cuda"), t] += 4.0
    now = torch.log_softmax(z.double(), 1)[torch.arange(N, device="cuda"), t]
    # ratios away from the ends of the clip, where the last bit would decide
    ratio = torch.tensor([0.5, 0.75, 0.9, 1.0, 1.1, 1.2, 1.5, 3.0], device="cuda")[torch.randint(0, 8, (N,), device="cuda", generator=g)]
    adv = rand(N, seed=seed + 2)
    adv[::7] = 0.0
    mask = torch.rand(N, device="cuda", generator=g) >= masked
    return {"z": z, "t": t, "old": (now - ratio.log()).float(), "adv": adv,
            "ref": (now + rand(N, seed=seed + 3, std=0.3)).float(), "mask": mask}


def check_policy(ms, c, beta=0.1, use_mask=True, grad_scale=1.0, what=""):
    A = ms.from_torch
    ones = torch.ones_like(c["mask"])
    r = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(c["ref"]) if beta else None,
                       A(c["mask"]) if use_mask else None, clip_low=0.2, clip_high=0.3, kl_coef=beta, grad_scale=grad_scale)
    want, err = P.policy(c["z"].double(), c["t"].long(), c["old"].double(), c["adv"].double(),
                         c["ref"].double() if beta else None, c["mask"] if use_mask else ones, 0.2, 0.3, beta, grad_scale)
    assert torch.equal(r.clipped.torch(), want["clipped"]), what
    for k in ("logp", "kl", "loss", "dlogits"):
        P.close(getattr(r, k).torch(), want[k], err[k], f"{what} {k}")
    only = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(c["ref"]) if beta else None,
                          A(c["mask"]) if use_mask else None, clip_low=0.2, clip_high=0.3, kl_coef=beta, grad=False)
    assert only.dlogits is None and torch.equal(only.clipped.torch(), r.clipped.torch())
    P.close(only.loss.torch(), want["loss"], err["loss"], f"{what} loss alone")
    P.close(only.logp.torch(), want["logp"], err["logp"], f"{what} logp alone")
    return r


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("N,V,masked", [(1, 1, 0.0), (3, 2, 0.0), (5, 31, 0.3), (2, 1000, 0.5), (64, 1003, 0.2), (700, 129, 0.2),
                                        (9, 32003, 0.2), (4, 65536, 0.0), (3, 131072, 0.3), (2, 200001, 0.0),
                                        (1, 1000003, 0.0)])
def test_policy(ms, dtype, N, V, masked):
    check_policy(ms, make_policy(N, V, dtype, masked), use_mask=masked > 0)


def test_policy_without_kl_and_scaled(ms):
    check_policy(ms, make_policy(50, 700, "f32", 0.2), beta=0.0)
    check_policy(ms, make_policy(50, 700, "f16", 0.2), grad_scale=1024.0)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", ["row gap", "odd start", "transposed", "batched", "int32"])
def test_policy_layouts(ms, dtype, layout):
    N, V = 12, 520
    c = make_policy(N, V, dtype, 0.25)
    if layout == "row gap":
        w = torch.zeros(N, V + 8, dtype=c["z"].dtype, device="cuda")
        w[:, :V] = c["z"]
        c["z"] = w[:, :V]
    elif layout == "odd start":
        w = torch.zeros(N, V + 3, dtype=c["z"].dtype, device="cuda")
        w[:, 3:] = c["z"]
        c["z"] = w[:, 3:]
    elif layout == "transposed":
        c["z"] = c["z"].t().contiguous().t()
    elif layout == "int32":
        c["t"] = c["t"].int()
    else:
        A = ms.from_torch
        flat = check_policy(ms, c)
        b = ms.policy_loss(A(c["z"].view(3, 4, V)), A(c["t"].view(3, 4)), A(c["old"].view(3, 4)), A(c["adv"].view(3, 4)),
                           A(c["ref"].view(3, 4)), A(c["mask"].view(3, 4)), clip_low=0.2, clip_high=0.3, kl_coef=0.1)
        assert b.dlogits.shape == (3, 4, V) and b.logp.shape == (3, 4) and b.loss.shape == ()
        assert torch.equal(b.dlogits.torch().view(N, V), flat.dlogits.torch()) and torch.equal(b.loss.torch(), flat.loss.torch())
        return
    check_policy(ms, c, what=layout)


@pytest.mark.parametrize("V", [300, 70001])
def test_policy_masked_tokens_are_not_read(ms, V):
    """NaN and infinite logits, targets outside the vocabulary: nothing of a masked token comes through; all tokens
    masked give zeros."""
    c = make_policy(6, V, "f32", 0.0)
    c["mask"][1::2] = False
    c["z"][1], c["z"][3], c["t"][3], c["t"][5] = math.nan, math.inf, -100, V
    c["old"][1], c["adv"][3], c["ref"][5] = math.nan, math.inf, math.nan
    r = check_policy(ms, {k: torch.nan_to_num(v, 0.0, 0.0, 0.0) if v.is_floating_point() else v for k, v in c.items()} | {
        "t": torch.where(c["mask"], c["t"], 0)})
    A = ms.from_torch
    raw = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(c["ref"]), A(c["mask"]), clip_low=0.2, clip_high=0.3,
                         kl_coef=0.1)
    for a, b in zip(raw, r):
        assert torch.equal(a.torch(), b.torch())
    none = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(c["ref"]), A(torch.zeros_like(c["mask"])), kl_coef=0.1)
    assert float(none.loss.torch()) == 0.0 and not bool(none.dlogits.torch().any()) and not bool(none.clipped.torch().any())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [40, 1027, 66000])
def test_policy_banned_words(ms, V, dtype):
    """Logits of -inf and of the type's lowest value take no probability; a row of the lowest value alone is an even
    distribution; a target that is banned, or outside the vocabulary, or a row of -inf gives what the formula gives."""
    c = make_policy(8, V, dtype, 0.0)
    low = torch.finfo(TORCH[dtype]).min
    keep = c["z"][torch.arange(8), c["t"]]
    c["z"][:, V // 2:] = -math.inf
    c["z"][:4, :8] = low
    c["z"][torch.arange(8), c["t"]] = keep
    check_policy(ms, c)
    c["z"][0] = low
    c["old"][0] = c["ref"][0] = -math.log(V)
    check_policy(ms, c, what="even row")
    c["t"][2] = V
    c["t"][3] = -1
    A = ms.from_torch
    r = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(c["ref"]), kl_coef=0.1)
    assert r.logp.torch().isnan().tolist() == [False, False, True, True] + [False] * 4 and bool(r.loss.torch().isnan())
    c["z"][5] = -math.inf
    r = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(c["ref"]), kl_coef=0.1)
    assert bool(r.logp.torch()[5].isnan()) and not bool(r.logp.torch()[6].isnan())
    c["z"][6, 3] = math.nan
    r = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(c["ref"]), kl_coef=0.1)
    assert bool(r.logp.torch()[6].isnan()) and bool(r.dlogits.torch()[6].isnan().all())


def test_policy_of_no_tokens(ms):
    A = ms.from_torch
    f = rand(0, seed=1)
    r = ms.policy_loss(A(rand(0, 50, seed=1)), A(torch.zeros(0, dtype=torch.int64, device="cuda")), A(f), A(f))
    assert float(r.loss.torch()) == 0.0 and r.dlogits.shape == (0, 50)


def test_policy_gradient_is_differences(ms):
    c = make_policy(7, 90, "f32", 0.2)
    A = ms.from_torch
    r = ms.policy_loss(A(c["z"]), A(c["t"]), A(c["old"]), A(c["adv"]), A(c["ref"]), A(c["mask"]), clip_low=0.2, clip_high=0.3,
                       kl_coef=0.1)
    v = rand(7, 90, seed=9).double()

    def loss(s):
        return float(P.policy(c["z"].double() + s * v, c["t"], c["old"].double(), c["adv"].double(), c["ref"].double(), c["mask"],
                              0.2, 0.3, 0.1, 1.0)[0]["loss"])

    want, part = (loss(1e-5) - loss(-1e-5)) / 2e-5, r.dlogits.torch().double() * v
    assert abs(float(part.sum()) - want) < 1.1e-5 * float(part.abs().sum())


# --------------------------------------------------------------- streams
def test_operators_on_another_stream_than_their_inputs(ms):
    """A long write on one stream, the operators on another: they wait for it, and the first stream's next write to an
    input waits for them."""
    n = 1 << 24
    s1, s2 = ms.Stream("cuda:0"), ms.Stream("cuda:0")
    with ms.stream(s1):
        one, x, y = ms.ones((n,), "f32"), ms.zeros((n,), "f32"), ms.empty((n,), "f32")
        for _ in range(20):
            ms.add(x, one, out=y)
            x, y = y, x
    with ms.stream(s2):
        d = ms.dropout(x, 0.5, 1)
        g = ms.full((1, 4096, 4096), 0.5, "f32")
        h = ms.gated_scan(ms.reshape(x, (1, 4096, 4096)), g)
    with ms.stream(s1):
        ms.mul(one, one, out=x)
    s1.synchronize()
    s2.synchronize()
    kept, up = P.keep_mask((n,), 0.5, 1, 0, "cuda")
    assert torch.equal(d.torch(), torch.where(kept, 20.0 * up, 0.0).float())
    assert float(h.torch()[0, 0, 5]) == 20.0 and abs(float(h.torch()[0, 4095, 7]) - 40.0) < 1e-4


def test_operators_in_a_cuda_graph(ms):
    """Captured once and replayed on new contents of the same buffers."""
    A = ms.from_torch
    x, g, h0 = rand(2, 600, 40, seed=1), gates(2, 600, 40, "linear", "f32", 2), rand(2, 40, seed=3)
    c = make_policy(20, 300, "f32", 0.2)
    t = make_norm(20, 300, "f32", "full", 0.1)
    arr = [A(v) for v in (x, g, h0, c["z"], c["t"], c["old"], c["adv"], t["x"], t["z"], t["w_post"], t["w_pre"], t["gate"])]

    def work():
        h, last = ms.gated_scan(arr[0], arr[1], arr[2], return_state=True)
        y, u, _ = ms.gated_residual_norm(*arr[7:11], gate=arr[11], dropout=0.1, seed=1)
        r = ms.policy_loss(*arr[3:7])
        return [v.torch() for v in (h, last, y, u, r.loss, r.dlogits)]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    x.mul_(2.0)
    t["x"].add_(1.0)
    c["z"].mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, work()):
        assert torch.equal(a, b)
