"""The block operators on the GPU on the kernels' paths that large calls take, against their formulas in 64 bits:
scans that walk chains of several tiles, norms whose blocks take several rows, rows too long for registers, losses whose
masked tokens are counted by a kernel of their own. Tolerances are the bounds that blocks_plain derives."""
import pytest
import torch

from . import blocks_plain as P
from .test_blocks_gpu import _odd_views, check_norm, check_policy, check_scan, gates, make_norm, make_policy, rand

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")]


# 80 chains (of 32 or 64 channels) and more, each of several tiles, the last one ragged
@pytest.mark.parametrize("mode", ["linear", "sigmoid"])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("B,T,D,H", [
    (4, 300, 1344, 1344), (3, 517, 2048, 32), (100, 261, 33, 33), (160, 300, 130, 130),  # more chains than blocks
    (3, 400, 1536, 32), (2, 290, 3200, 20), (90, 270, 24, 12), (80, 129, 64, 1), (81, 1025, 31, 31),
])
def test_scan_walks_several_tiles(ms, B, T, D, H, dtype, gate_dtype, mode):
    check_scan(ms, rand(B, T, D, seed=1, dtype=dtype), gates(B, T, H, mode, gate_dtype, 2), rand(B, D, seed=3), mode)


@pytest.mark.parametrize("kind", ["time first", "odd offset", "channels outside", "every second step", "broadcast"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H", [264, 4])
def test_scan_walk_layouts(ms, kind, dtype, H):
    x, gate = _odd_views(20, 300, 264, H, dtype, kind)
    check_scan(ms, x, gate, rand(20, 264, seed=3), "sigmoid", kind)


def test_scan_walk_without_an_initial_state(ms):
    A = ms.from_torch
    x, gate, dh = rand(90, 300, 40, seed=1), gates(90, 300, 40, "linear", "f32", 2), rand(90, 300, 40, seed=3)
    h, last = ms.gated_scan(A(x), A(gate), return_state=True)
    wh, wl, eh, el = P.scan(x.double(), gate.double(), None, "linear")
    P.close(h.torch(), wh, eh)
    P.close(last.torch(), wl, el)
    got = ms.gated_scan_backward(A(dh), A(x), A(gate), h)
    want, err = P.scan_backward(dh.double(), x.double(), gate.double(), h.torch().double(), None, None, "linear")
    for g, w, e in zip(got, want, err):
        P.close(g.torch(), w, e)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scan_walk_is_repeatable(ms, dtype):
    A = ms.from_torch
    x, gate = rand(6, 700, 1000, seed=1, dtype=dtype), gates(6, 700, 20, "sigmoid", dtype, 2)
    runs = []
    for _ in range(4):
        h = ms.gated_scan(A(x), A(gate), mode="sigmoid")
        runs.append((h.torch(),) + tuple(v.torch() for v in ms.gated_scan_backward(A(x), A(x), A(gate), h, mode="sigmoid")))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


# every width of the kernels' packs, at as many rows as give each block several
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,activation,p", [("full", "silu", 0.1), ("row", "sigmoid", 0.0), ("channel", "silu", 0.3),
                                               ("none", "linear", 0.0)])
@pytest.mark.parametrize("R,D", [(20000, 40), (9001, 128), (6000, 258), (4000, 520), (3001, 1031), (1500, 1000), (1501, 2046),
                                 (1500, 4096), (700, 4095), (650, 8192), (400, 9001), (320, 16384), (310, 16382),
                                 (305, 16383)])
def test_norm_of_many_rows(ms, R, D, dtype, kind, activation, p):
    check_norm(ms, make_norm(R, D, dtype, kind, p), activation, p)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind,activation,p", [("full", "silu", 0.1), ("row", "sigmoid", 0.3), ("channel", "silu", 0.0),
                                               ("none", "linear", 0.1)])
@pytest.mark.parametrize("R,D", [(5, 20000), (3, 16391), (40, 16385)])
def test_norm_of_long_rows(ms, R, D, dtype, kind, activation, p):
    check_norm(ms, make_norm(R, D, dtype, kind, p), activation, p)


@pytest.mark.parametrize("D", [520, 17000])
def test_norm_of_strided_rows(ms, D):
    t = make_norm(300 if D < 1000 else 6, D, "bf16", "full", 0.2)
    for k in ("x", "z", "gate", "dy", "du"):
        w = torch.zeros(t[k].shape[0], 2, D + 5, dtype=t[k].dtype, device="cuda")
        w[:, 1, 2:D + 2] = t[k]
        t[k] = w[:, 1, 2:D + 2]
    check_norm(ms, t, "sigmoid", 0.2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_of_weights_and_gates_inside_other_arrays(ms, dtype):
    """Weights that start at any float, a gate per row that is a column of a matrix, a gate per channel inside a row."""
    for kind in ("row", "channel"):
        t = make_norm(700, 512, dtype, kind, 0.1)
        for k in ("w_post", "w_pre"):
            w = torch.zeros(520, device="cuda")
            w[3:515] = t[k]
            t[k] = w[3:515]
        w = torch.zeros(700, 7, dtype=t["gate"].dtype, device="cuda") if kind == "row" else torch.zeros(520, dtype=t["gate"].dtype,
                                                                                                      device="cuda")
        view = w[:, 4:5] if kind == "row" else w[5:517]
        view.copy_(t["gate"])
        t["gate"] = view
        check_norm(ms, t, "silu", 0.1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("R,D", [(4000, 520), (3001, 1031), (6, 20000)])
def test_rms_norm_of_many_rows(ms, R, D, dtype):
    x, du, dy = (rand(R, D, seed=i, dtype=dtype) for i in range(3))
    w = rand(D, seed=5, mean=1.0, std=0.2)
    A = ms.from_torch
    u, rstd = ms.rms_norm(A(x), A(w), eps=1e-5)
    (_, wu, _, ry), (_, eu, er) = P.norm(x.double(), None, None, w.double(), None, "linear", 1.0, 1e-5, None)
    P.close(u.torch(), wu, eu, "u")
    P.close(rstd.torch(), ry[:, 0], er[:, 0] * ry[:, 0], "rstd")
    for add in (None, dy):
        dx, dw = ms.rms_norm_backward(A(du), A(x), A(w), rstd, None if add is None else A(add))
        out, err = P.norm_backward(None if add is None else add.double(), du.double(), x.double(), None, None, w.double(), None,
                                   rstd.torch().double()[:, None], None, "linear", None)
        P.close(dx.torch(), out["dx"], err["dx"], "dx")
        P.close(dw.torch(), out["pre"].sum(0), err["pre"].sum(0) + (R + 8) * P.EPS32 * out["pre"].abs().sum(0), "dw")


# more masked tokens than a block counts for itself: by a warp per token, by clusters, by three passes
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N,V,start", [(9000, 129, 0), (1500, 2051, 0), (1100, 5003, 0), (8300, 20001, 0), (17000, 37, 3)])
def test_policy_of_many_masked_tokens(ms, N, V, start, dtype):
    if N * V > 1 << 26 and dtype == "f32":
        N = 8200
    c = make_policy(N, V, dtype, 0.3)
    if start:
        w = torch.zeros(N, V + start, dtype=c["z"].dtype, device="cuda")
        w[:, start:] = c["z"]
        c["z"] = w[:, start:]
    check_policy(ms, c)
