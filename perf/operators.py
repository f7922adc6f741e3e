"""The operators of a recurrent block in training and serving, as measured cases: the gated linear recurrence,
the norms around a block with its gate, dropout and residual scale, dropout itself, and the clipped policy loss.

Each case is one call as a program makes it: a forward pass, a backward pass, a decode step, a loss with its
gradient. ``run`` computes it in its plain form, elementary torch operations in 32 bits, or through
``musapy_b200`` where ``own`` is true; ``exact`` computes it in 64 bits from the definition.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-6
_SCALE = 0.5  # the residual branch's scale
_CLIP_LOW, _CLIP_HIGH = 0.2, 0.28
_MASK32 = 0xFFFFFFFF


# ------------------------------------------------------------------ cases
def _scan(direction, batch, time, dim, heads, dtype, gate_dtype, mode):
    return {"op": "scan", "pass": direction, "batch": batch, "time": time, "dim": dim, "heads": heads,
            "dtype": dtype, "gate_dtype": gate_dtype, "mode": mode}


def _norm(direction, rows, dim, dtype, gate, activation, dropout):
    return {"op": "norm", "pass": direction, "rows": rows, "dim": dim, "dtype": dtype, "gate": gate,
            "activation": activation, "dropout": dropout}


def _dropout(rows, dim, dtype, dropout):
    return {"op": "dropout", "rows": rows, "dim": dim, "dtype": dtype, "dropout": dropout}


def _policy(rows, vocab, dtype, kl, masked):
    return {"op": "policy", "rows": rows, "vocab": vocab, "dtype": dtype, "kl": kl, "masked": masked}


def listed():
    return [
        # one token for each of 64 running sequences: what serving calls for every layer and token
        {"name": "scan step 64x4096 bf16", **_scan("step", 64, 1, 4096, 4096, "bf16", "bf16", "sigmoid")},
        # a training batch with a gate per channel: forward, and backward
        {"name": "scan fwd 8x4096x2048 bf16", **_scan("forward", 8, 4096, 2048, 2048, "bf16", "bf16", "sigmoid")},
        {"name": "scan bwd 8x4096x2048 bf16", **_scan("backward", 8, 4096, 2048, 2048, "bf16", "bf16", "sigmoid")},
        # one long document with few channels: the sequence itself has to be split
        {"name": "scan fwd 1x65536x1000 f32", **_scan("forward", 1, 65536, 1000, 1000, "f32", "f32", "linear")},
        # one decay for each head of 64 channels, kept in 32 bits; an odd length; its gradient sums over the head
        {"name": "scan bwd 4x4095x32h64 bf16", **_scan("backward", 4, 4095, 2048, 32, "bf16", "f32", "linear")},
        # the norms around a block for a handful of decoded tokens
        {"name": "norm fwd 8x4096 bf16", **_norm("forward", 8, 4096, "bf16", "full", "silu", 0.0)},
        # a learned gate per channel in full precision, odd rows and an odd width
        {"name": "norm fwd 3001x1031 f32", **_norm("forward", 3001, 1031, "f32", "channel", "linear", 0.0)},
        # a training batch with dropout on the block's branch, backward
        {"name": "norm bwd 16384x4096 bf16", **_norm("backward", 16384, 4096, "bf16", "full", "sigmoid", 0.1)},
        # a small activation in full precision, and the activations of a large batch
        {"name": "dropout 257x1000 f32", **_dropout(257, 1000, "f32", 0.25)},
        {"name": "dropout 65536x4096 f16", **_dropout(65536, 4096, "f16", 0.1)},
        # a short rollout over an odd vocabulary in full precision, and a long one over a large vocabulary
        {"name": "policy 255x32003 f32", **_policy(255, 32003, "f32", 0.05, 0.2)},
        {"name": "policy 4096x131072 bf16", **_policy(4096, 131072, "bf16", 0.02, 0.1)},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm; one in three is made a multiple of 64 if it can be."""
    n = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    if n >= 64 and rng.random() < 1 / 3:
        n -= n % 64
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["scan", "scan", "norm", "norm", "dropout", "policy"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "scan":
        direction = rng.choice(["forward", "forward", "backward", "backward", "step"])
        mode, most = rng.choice(["linear", "sigmoid"]), 1 << 25
        gate_dtype = rng.choice([dtype, "f32"])
        if rng.random() < 0.3:  # gates shared by the channels of a head
            per, heads = rng.choice([16, 48, 64, 80, 128]), _log(rng, 1, 32)
            dim = per * heads
        else:
            dim = heads = _log(rng, 32, 4096)
        if dim == 3072:
            heads, dim = heads + 1, dim + dim // heads
        if direction == "step":
            return _scan("step", _log(rng, 1, 512), 1, dim, heads, dtype, gate_dtype, mode)
        time = _log(rng, 2, max(2, min(65536, most // dim)))
        batch = _log(rng, 1, max(1, min(32, most // (dim * time))))
        return _scan(direction, batch, time, dim, heads, dtype, gate_dtype, mode)
    if op == "norm":
        dim = _log(rng, 64, 8192)
        return _norm(rng.choice(["forward", "backward"]), _log(rng, 1, min(32768, (1 << 26) // dim)), dim, dtype,
                     rng.choice(["full", "full", "row", "channel", "none"]),
                     rng.choice(["linear", "sigmoid", "silu"]), rng.choice([0.0, 0.1, 0.3]))
    if op == "dropout":
        dim = _log(rng, 64, 8192)
        return _dropout(_log(rng, 1, min(65536, (1 << 27) // dim)), dim, dtype, rng.choice([0.05, 0.1, 0.5]))
    vocab = _log(rng, 1000, 131072)
    return _policy(_log(rng, 1, min(4096, (1 << 28) // vocab)), vocab, dtype, rng.choice([0.0, 0.04]),
                   rng.choice([0.0, 0.3]))


# ----------------------------------------------------------------- inputs
def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    rng = torch.Generator(device="cuda")
    rng.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.empty(shape, device="cuda").normal_(mean, std, generator=rng).to(dtype)

    if case["op"] == "scan":
        b, t, d, h = case["batch"], case["time"], case["dim"], case["heads"]
        gt = _DTYPES[case["gate_dtype"]]
        # gates as trained models have them: most of the state is kept, some channels forget quickly
        gate = normal(b, t, h, std=1.5, mean=2.0)
        gate = gate.to(gt) if case["mode"] == "sigmoid" else torch.sigmoid(gate + 1.0).to(gt)
        s = {"x": normal(b, t, d, dtype=dt), "gate": gate, "state": normal(b, d)}
        if case["pass"] == "step":
            s["x"], s["gate"] = s["x"][:, 0], s["gate"][:, 0]
        if case["pass"] == "backward":
            h, _ = _plain_scan(s["x"].float(), s["gate"].float(), s["state"], case["mode"])
            s["h"] = h.to(dt)  # as the forward pass left it
            s["dh"], s["dstate"] = normal(b, t, d, dtype=dt), normal(b, d)
        return s
    if case["op"] == "norm":
        r, d = case["rows"], case["dim"]
        shape = {"full": (r, d), "row": (r, 1), "channel": (d,), "none": None}[case["gate"]]
        s = {"x": normal(r, d, std=2.0, dtype=dt), "z": (normal(r, d) * normal(r, 1).exp()).to(dt),
             "w_post": normal(d, std=0.1, mean=1.0), "w_pre": normal(d, std=0.1, mean=1.0),
             "gate": None if shape is None else normal(*shape, dtype=dt)}
        s["seed"], s["offset"] = 1000003 * seed + 17, (seed << 33) + 5
        if case["pass"] == "backward":
            y, _, rstd = _plain_norm(case, s)
            s["y"], s["rstd"] = y.to(dt), rstd  # as the forward pass left them
            s["dy"], s["du"] = normal(r, d, dtype=dt), normal(r, d, dtype=dt)
            del s["x"]
        return s
    if case["op"] == "dropout":
        return {"x": normal(case["rows"], case["dim"], dtype=dt), "seed": 1000003 * seed + 17, "offset": seed}
    n, v = case["rows"], case["vocab"]
    logits = normal(n, v, std=2.0, dtype=dt)
    targets = torch.randint(0, v - 4, (n,), device="cuda", generator=rng)
    rows = torch.arange(n, device="cuda")
    logits[rows, targets] += 8.0  # a sampled token is a likely one
    logits[:, v - 3:] = -math.inf  # the padding of the vocabulary
    now = _logp(logits.float(), targets)
    ratio = normal(n, std=0.3).exp()  # away from the two ends of the clip, where the last bit decides
    near = ((ratio - (1 - _CLIP_LOW)).abs() < 1e-3) | ((ratio - (1 + _CLIP_HIGH)).abs() < 1e-3)
    ratio = torch.where(near, ratio + 4e-3, ratio)
    return {"logits": logits, "targets": targets, "old_logp": now - ratio.log(),
            "ref_logp": now + normal(n, std=0.3), "advantages": normal(n),
            "mask": torch.rand(n, device="cuda", generator=rng) >= case["masked"]}


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # a program that uses the framework holds its Arrays: views of the same memory
        import musapy_b200 as ms

        s = {k: ms.from_torch(v) if isinstance(v, torch.Tensor) else v for k, v in s.items()}
        s["ms"] = ms
    return {"case": case, **s}


# -------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"]](case, state)
    return _PLAIN[case["op"]](case, state)


def _own_scan(case, s):
    ms, mode = s["ms"], case["mode"]
    if case["pass"] == "step":
        h = ms.gated_scan_step(s["state"], s["x"], s["gate"], mode=mode)
        return {"h": h.torch(), "state": s["state"].torch()}
    if case["pass"] == "forward":
        h, last = ms.gated_scan(s["x"], s["gate"], s["state"], mode=mode, return_state=True)
        return {"h": h.torch(), "state": last.torch()}
    dx, dgate, dh0 = ms.gated_scan_backward(s["dh"], s["x"], s["gate"], s["h"], s["state"], s["dstate"], mode=mode)
    return {"dx": dx.torch(), "dgate": dgate.torch(), "dstate": dh0.torch()}


def _own_norm(case, s):
    ms = s["ms"]
    how = {"gate": s["gate"], "activation": case["activation"], "scale": _SCALE, "dropout": case["dropout"],
           "seed": s["seed"], "offset": s["offset"]}
    if case["pass"] == "forward":
        y, u, rstd = ms.gated_residual_norm(s["x"], s["z"], s["w_post"], s["w_pre"], eps=_EPS, **how)
        return {"y": y.torch(), "u": u.torch(), "rstd": rstd.torch()}
    dx, dz, dgate, dpost, dpre = ms.gated_residual_norm_backward(s["dy"], s["du"], s["y"], s["z"], s["w_post"],
                                                                 s["w_pre"], s["rstd"], **how)
    out = {"dx": dx.torch(), "dz": dz.torch(), "dw_post": dpost.torch(), "dw_pre": dpre.torch()}
    if dgate is not None:
        out["dgate"] = dgate.torch()
    return out


def _own_dropout(case, s):
    return s["ms"].dropout(s["x"], case["dropout"], s["seed"], s["offset"]).torch()


def _own_policy(case, s):
    r = s["ms"].policy_loss(s["logits"], s["targets"], s["old_logp"], s["advantages"], s["ref_logp"], s["mask"],
                            clip_low=_CLIP_LOW, clip_high=_CLIP_HIGH, kl_coef=case["kl"], grad=True)
    return {"loss": r.loss.torch(), "logp": r.logp.torch(), "kl": r.kl.torch(), "clipped": r.clipped.torch(),
            "dlogits": r.dlogits.torch()}


_OWN = {"scan": _own_scan, "norm": _own_norm, "dropout": _own_dropout, "policy": _own_policy}


# ------------------------------------------------------------ plain forms
def _recur(a, b):
    """h[t] = a[t] h[t-1] + b[t] with h[-1] = 0 along dim 1: neighbours are joined, the half as long recurrence of
    the pairs is solved, and the steps between are filled in."""
    t = b.shape[1]
    if t == 1:
        return b
    n = t // 2
    a1, b1 = a[:, 1:2 * n:2], b[:, 1:2 * n:2]
    odd = _recur(a1 * a[:, 0:2 * n:2], a1 * b[:, 0:2 * n:2] + b1)
    h = torch.empty_like(b)
    h[:, 1::2] = odd
    h[:, 0] = b[:, 0]
    h[:, 2::2] = a[:, 2::2] * odd[:, :(t - 1) // 2] + b[:, 2::2]
    return h


def _spread(gate, d):
    """(b, t, heads) gates to (b, t, d): one for every channel."""
    b, t, h = gate.shape
    return gate if h == d else gate[..., None].expand(b, t, h, d // h).reshape(b, t, d)


def _plain_scan(x, gate, h0, mode):
    a = 1 / (1 + torch.exp(-gate)) if mode == "sigmoid" else gate
    a = _spread(a, x.shape[2])
    b = (1 - a) * x if mode == "sigmoid" else x.clone()
    b[:, 0] += a[:, 0] * h0
    h = _recur(a, b)
    return h, h[:, -1].clone()


def _do_scan(case, s):
    dt, gt, mode = _DTYPES[case["dtype"]], _DTYPES[case["gate_dtype"]], case["mode"]
    x, gate = s["x"].float(), s["gate"].float()
    if case["pass"] == "step":
        h, last = _plain_scan(x[:, None], gate[:, None], s["state"], mode)
        s["state"].copy_(last)
        return {"h": h[:, 0].to(dt), "state": s["state"]}
    if case["pass"] == "forward":
        h, last = _plain_scan(x, gate, s["state"], mode)
        return {"h": h.to(dt), "state": last}
    b, t, d = x.shape
    dh, h = s["dh"].float(), s["h"].float()
    narrow = 1 / (1 + torch.exp(-gate)) if mode == "sigmoid" else gate
    a = _spread(narrow, d)
    # the gradient of h[t] is dh[t] + a[t + 1] times that of h[t + 1]
    after = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1).flip(1)
    src = dh.clone()
    src[:, -1] += s["dstate"]
    g = _recur(after, src.flip(1)).flip(1)
    before = torch.cat([s["state"][:, None], h[:, :-1]], 1)
    if mode == "sigmoid":
        dx, dgate = g * (1 - a), g * (before - x) * a * (1 - a)
    else:
        dx, dgate = g, g * before
    heads = gate.shape[2]
    if heads != d:
        dgate = dgate.reshape(b, t, heads, d // heads).sum(3)
    return {"dx": dx.to(dt), "dgate": dgate.to(gt), "dstate": a[:, 0] * g[:, 0]}


def _philox(seed, offset, block):
    """Eight 16-bit numbers for each of the counters `block` (int64): Philox-4x32 with ten rounds (Salmon, Moraes,
    Dror and Shaw, 2011), counter {block, offset}, key `seed`, the low half of each word first."""
    c0, c1 = block & _MASK32, (block >> 32) & _MASK32
    c2, c3 = torch.full_like(block, offset & _MASK32), torch.full_like(block, (offset >> 32) & _MASK32)
    k0, k1 = seed & _MASK32, (seed >> 32) & _MASK32
    for _ in range(10):  # the cipher's rounds
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # the low 64 bits, which the sign does not change
        c0, c1, c2, c3 = (((p1 >> 32) & _MASK32) ^ c1 ^ k0, p1 & _MASK32,
                          ((p0 >> 32) & _MASK32) ^ c3 ^ k1, p0 & _MASK32)
        k0, k1 = (k0 + 0x9E3779B9) & _MASK32, (k1 + 0xBB67AE85) & _MASK32
    w = torch.stack([c0, c1, c2, c3], -1)
    return torch.stack([w & 0xFFFF, w >> 16], -1).reshape(-1, 8)


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _keep(shape, p, seed, offset, draw16=_philox):
    """Which elements (in C order) dropout keeps, and what it multiplies them with."""
    n, drop = math.prod(shape), _threshold(p)
    bits = draw16(seed, offset, torch.arange((n + 7) // 8, device="cuda"))
    return (bits.reshape(-1)[:n] >= drop).reshape(shape), 65536 / (65536 - drop)


def _do_dropout(case, s):
    keep, up = _keep(s["x"].shape, case["dropout"], s["seed"], s["offset"])
    return torch.where(keep, s["x"].float() * up, 0.0).to(_DTYPES[case["dtype"]])


def _act(case, gate):
    """The gate's value and its derivative."""
    if gate is None:
        return 1.0, None
    g = gate.float()
    if case["activation"] == "linear":
        return g, torch.ones_like(g)
    sig = 1 / (1 + torch.exp(-g))
    if case["activation"] == "sigmoid":
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


def _branch(case, s, shape):
    """What dropout and the residual scale multiply the branch with."""
    if case["dropout"] == 0.0:
        return _SCALE
    keep, up = _keep(shape, case["dropout"], s["seed"], s["offset"])
    return torch.where(keep, up * _SCALE, 0.0)


def _plain_norm(case, s):
    x, z = s["x"].float(), s["z"].float()
    r_z = 1 / torch.sqrt((z * z).mean(1, keepdim=True) + _EPS)
    value, _ = _act(case, s["gate"])
    y = x + _branch(case, s, z.shape) * value * (z * r_z * s["w_post"])
    r_y = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + _EPS)
    return y, y * r_y * s["w_pre"], torch.stack([r_z[:, 0], r_y[:, 0]])


def _do_norm(case, s):
    dt = _DTYPES[case["dtype"]]
    if case["pass"] == "forward":
        y, u, rstd = _plain_norm(case, s)
        return {"y": y.to(dt), "u": u.to(dt), "rstd": rstd}
    dy, du, y, z = s["dy"].float(), s["du"].float(), s["y"].float(), s["z"].float()
    r_z, r_y = s["rstd"][0][:, None], s["rstd"][1][:, None]
    y_hat, z_hat = y * r_y, z * r_z
    wu = du * s["w_pre"]
    dx = dy + r_y * (wu - y_hat * (wu * y_hat).mean(1, keepdim=True))
    value, slope = _act(case, s["gate"])
    d = dx * _branch(case, s, z.shape)
    dn = d * value
    wn = dn * s["w_post"]
    out = {"dx": dx.to(dt), "dz": (r_z * (wn - z_hat * (wn * z_hat).mean(1, keepdim=True))).to(dt),
           "dw_post": (dn * z_hat).sum(0), "dw_pre": (du * y_hat).sum(0)}
    if slope is not None:
        dg = d * z_hat * s["w_post"] * slope
        dg = dg.sum(1, keepdim=True) if case["gate"] == "row" else dg.sum(0) if case["gate"] == "channel" else dg
        out["dgate"] = dg.to(dt)
    return out


def _logp(z, targets):
    top = z.amax(1, keepdim=True)
    lse = top + torch.exp(z - top).sum(1, keepdim=True).log()
    return (z.gather(1, targets[:, None]) - lse)[:, 0]


def _do_policy(case, s):
    z, mask = s["logits"].float(), s["mask"]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    at = s["targets"][:, None]
    logp = (z.gather(1, at) - top - total.log())[:, 0]
    ratio, a = torch.exp(logp - s["old_logp"]), s["advantages"]
    clipped = ((a > 0) & (ratio > 1 + _CLIP_HIGH) | (a < 0) & (ratio < 1 - _CLIP_LOW)) & mask
    bound = torch.where(a > 0, 1 + _CLIP_HIGH, 1 - _CLIP_LOW)
    apart = s["ref_logp"] - logp
    kl = torch.exp(apart) - apart - 1
    each = -torch.where(clipped, bound, ratio) * a + case["kl"] * kl
    count = mask.sum().clamp(min=1)
    slope = (torch.where(clipped, 0.0, -ratio * a) + case["kl"] * (1 - torch.exp(apart))) / count
    slope = torch.where(mask, slope, 0.0)[:, None]
    grad = e * (-slope / total)
    grad.scatter_add_(1, at, slope)
    return {"loss": torch.where(mask, each, 0.0).sum() / count, "logp": torch.where(mask, logp, 0.0),
            "kl": torch.where(mask, kl, 0.0), "clipped": clipped, "dlogits": grad.to(_DTYPES[case["dtype"]])}


_PLAIN = {"scan": _do_scan, "norm": _do_norm, "dropout": _do_dropout, "policy": _do_policy}


# ------------------------------------------------------------------- work
def work(case):
    """Each input read once and each output written once; the operations that the formulas ask for."""
    e = _BYTES[case["dtype"]]
    if case["op"] == "scan":
        b, t, d, h, g = case["batch"], case["time"], case["dim"], case["heads"], _BYTES[case["gate_dtype"]]
        n, ng, extra = b * t * d, b * t * h, 4 if case["mode"] == "sigmoid" else 0
        if case["pass"] == "backward":  # dh, h, (x), gate, dstate, h0 -> dx, dgate, dh0
            reads = 3 if case["mode"] == "sigmoid" else 2
            return {"bytes": n * e * (reads + 1) + ng * g * 2 + 12 * b * d, "flops": n * (4 + extra)}
        return {"bytes": n * e * 2 + ng * g + 8 * b * d, "flops": n * (2 + extra)}
    n = case["rows"] * (case["vocab"] if case["op"] == "policy" else case["dim"])
    if case["op"] == "norm":
        r, d = case["rows"], case["dim"]
        gate = {"full": n, "row": r, "channel": d, "none": 0}[case["gate"]]
        if case["pass"] == "backward":  # dy, du, y, z, gate -> dx, dz, dgate
            return {"bytes": (6 * n + 2 * gate) * e + 8 * r + 16 * d, "flops": 24 * n}
        return {"bytes": (4 * n + gate) * e + 8 * r + 8 * d, "flops": 12 * n}
    if case["op"] == "dropout":
        return {"bytes": 2 * n * e, "flops": n}
    return {"bytes": 2 * n * e + 34 * case["rows"], "flops": 6 * n}


# -------------------------------------------------------- 64-bit versions
def _exact_philox(seed, offset, block):
    """The generator again, its 32 x 32 bit products put together from 16-bit halves."""
    def product(x, m):
        lo, hi = x & 0xFFFF, x >> 16
        low = lo * (m & 0xFFFF)
        mid = hi * (m & 0xFFFF) + (low >> 16)
        mid2 = lo * (m >> 16) + (mid & 0xFFFF)
        return hi * (m >> 16) + (mid >> 16) + (mid2 >> 16), ((mid2 & 0xFFFF) << 16) | (low & 0xFFFF)

    word = [block % 2**32, block // 2**32, torch.full_like(block, offset % 2**32),
            torch.full_like(block, offset // 2**32 % 2**32)]
    for i in range(10):
        h0, l0 = product(word[0], 0xD2511F53)
        h1, l1 = product(word[2], 0xCD9E8D57)
        word = [h1 ^ word[1] ^ ((seed + i * 0x9E3779B9) % 2**32), l1,
                h0 ^ word[3] ^ ((seed // 2**32 + i * 0xBB67AE85) % 2**32), l0]
    out = torch.empty(block.numel(), 8, dtype=torch.int64, device=block.device)
    for i, w in enumerate(word):
        out[:, 2 * i], out[:, 2 * i + 1] = w % 65536, w // 65536
    return out


def _exact_scan(case, s):
    x, gate, state = s["x"].double(), s["gate"].double(), s["state"].double()
    if case["pass"] == "step":
        x, gate = x[:, None], gate[:, None]
    b, t, d = x.shape
    sig = case["mode"] == "sigmoid"
    a = torch.sigmoid(gate) if sig else gate
    a = a.repeat_interleave(d // gate.shape[2], dim=2)
    if case["pass"] != "backward":
        out, h = torch.empty_like(x), state
        for i in range(t):
            h = torch.lerp(x[:, i], h, a[:, i]) if sig else torch.addcmul(x[:, i], a[:, i], h)
            out[:, i] = h
        return {"h": out[:, 0] if case["pass"] == "step" else out, "state": h}
    dh, h = s["dh"].double(), s["h"].double()
    g, carry = torch.empty_like(x), s["dstate"].double()
    for i in reversed(range(t)):
        g[:, i] = dh[:, i] + carry
        carry = g[:, i] * a[:, i]
    da = g.clone()
    da[:, 0] *= state - x[:, 0] if sig else state
    da[:, 1:] *= h[:, :-1] - x[:, 1:] if sig else h[:, :-1]
    if sig:
        da *= a - a * a
        g = g - g * a
    return {"dx": g, "dgate": da.unflatten(2, (gate.shape[2], -1)).sum(-1), "dstate": carry}


def _exact_norm(case, s):
    d = case["dim"]
    z, post, pre = s["z"].double(), s["w_post"].double(), s["w_pre"].double()
    acts = {"linear": lambda v: v, "sigmoid": torch.sigmoid, "silu": torch.nn.functional.silu}
    gate = None if s["gate"] is None else s["gate"].double().requires_grad_(case["pass"] == "backward")
    value = torch.ones((), dtype=torch.float64, device="cuda") if gate is None else acts[case["activation"]](gate)
    factor = _SCALE
    if case["dropout"]:
        keep, up = _keep(z.shape, case["dropout"], s["seed"], s["offset"], _exact_philox)
        factor = keep.double() * (up * _SCALE)
    if case["pass"] == "forward":
        r_z = ((z * z).sum(1) / d + _EPS).rsqrt()
        y = s["x"].double() + torch.einsum("rc,r,c->rc", z, r_z, post) * value * factor
        r_y = ((y * y).sum(1) / d + _EPS).rsqrt()
        return {"y": y, "u": torch.einsum("rc,r,c->rc", y, r_y, pre), "rstd": torch.stack([r_z, r_y])}
    dy, du, y = s["dy"].double(), s["du"].double(), s["y"].double()
    r_z, r_y = s["rstd"].double()
    dot = torch.einsum("rc,rc,c->r", du, y, pre)
    dx = dy + torch.einsum("rc,c,r->rc", du, pre, r_y) - y * (r_y**3 * dot / d)[:, None]
    n = torch.einsum("rc,r,c->rc", z, r_z, post)
    branch = dx * factor
    dn = branch * value.detach()
    dot = torch.einsum("rc,rc,c->r", dn, z, post)
    out = {"dx": dx, "dz": torch.einsum("rc,c,r->rc", dn, post, r_z) - z * (r_z**3 * dot / d)[:, None],
           "dw_post": torch.einsum("rc,rc,r->c", dn, z, r_z), "dw_pre": torch.einsum("rc,rc,r->c", du, y, r_y)}
    if gate is not None:
        out["dgate"], = torch.autograd.grad((branch * n * value).sum(), gate)
    return out


def _exact_policy(case, s):
    z = s["logits"].double().requires_grad_()
    mask, a = s["mask"], s["advantages"].double()
    logp = z[torch.arange(z.shape[0], device="cuda"), s["targets"]] - torch.logsumexp(z, 1)
    ratio = torch.exp(logp - s["old_logp"].double())
    surrogate = torch.minimum(ratio * a, ratio.clamp(1 - _CLIP_LOW, 1 + _CLIP_HIGH) * a)
    kl = torch.expm1(s["ref_logp"].double() - logp) - (s["ref_logp"].double() - logp)
    loss = ((case["kl"] * kl - surrogate) * mask).sum() / max(1, int(mask.sum()))
    grad, = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "logp": logp.detach() * mask, "kl": kl.detach() * mask, "clipped": None,
            "dlogits": grad}


def _exact_dropout(case, s):
    keep, up = _keep(s["x"].shape, case["dropout"], s["seed"], s["offset"], _exact_philox)
    return s["x"].double() * keep * up


def exact(case, seed):
    of = {"scan": _exact_scan, "norm": _exact_norm, "dropout": _exact_dropout, "policy": _exact_policy}
    return of[case["op"]](case, _inputs(case, seed))
