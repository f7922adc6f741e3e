"""The block operators in 64 bits (torch float64), straight from their formulas, and bounds on what float arithmetic
may make of them.

A bound is K * 2^-24 times a majorant, the same formula with every term taken by its magnitude, where K counts the
roundings on the longest way to the result; the rounding of a 16-bit result is added. K is set from the
formulas and the lengths, not from measured errors."""
import math

import torch

EPS32 = 2.0 ** -24
# half a unit in the last place of a result, relative, and half the smallest subnormal
ROUND = {t: (torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2)
         for t in (torch.float32, torch.float16, torch.bfloat16)}


def close(got, want, slack, what=""):
    """|got - want| <= slack + the rounding of got's type, NaN where and only where `want` has it."""
    rel, tiny = ROUND[got.dtype]
    g = got.double().to(want.device)
    assert g.shape == want.shape, f"{what}: {tuple(g.shape)} != {tuple(want.shape)}"
    assert torch.equal(g.isnan(), want.isnan()), f"{what}: NaN in other places"
    # a value that rounds to the type's infinity may come out as either side of it
    top = torch.finfo(got.dtype).max
    both_big = (g.abs() >= top) & (want.abs() >= top) & (g.sign() == want.sign())
    off = (g - want).abs() - slack - rel * (want.abs() + slack) - tiny
    bad = (off > 0) & ~both_big & ~want.isnan() & ~(g == want)
    if bad.any():
        i = int(torch.nonzero(bad.reshape(-1))[0])
        s = slack.reshape(-1)[i] if isinstance(slack, torch.Tensor) and slack.shape == want.shape else slack
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: "
                             f"{g.reshape(-1)[i].item()!r} want {want.reshape(-1)[i].item()!r} slack {s}")


# ------------------------------------------------------------------ scan
def spread(gate, D):
    return gate.repeat_interleave(D // gate.shape[-1], dim=-1) if gate.shape[-1] else gate


def scan(x, gate, h0, mode):
    """(h, last state, majorant of h, error bound of h). float64."""
    B, T, D = x.shape
    a = spread(torch.sigmoid(gate) if mode == "sigmoid" else gate, D)
    om = spread(torch.sigmoid(-gate), D) if mode == "sigmoid" else torch.ones_like(a)
    h = h0.clone() if h0 is not None else torch.zeros(B, D, dtype=torch.float64, device=x.device)
    # each step adds the roundings of its products, of the decay (a sigmoid: a few units) and of
    # the decays' products where a long sequence is joined from pieces: 16 units together
    M, E = h.abs(), h.abs() * EPS32
    hs, Es = [], []
    for t in range(T):
        h = a[:, t] * h + om[:, t] * x[:, t]
        M = a[:, t].abs() * M + (om[:, t] * x[:, t]).abs()
        E = a[:, t].abs() * E + 16 * EPS32 * M
        hs.append(h)
        Es.append(E)
    stack = (lambda v: torch.stack(v, 1)) if T else (lambda v: torch.zeros(B, 0, D, dtype=torch.float64, device=x.device))
    return stack(hs), h, stack(Es), E


def scan_backward(dh, x, gate, h, h0, dstate, mode):
    """(dx, dgate, dh0) and their error bounds, float64."""
    B, T, D = x.shape
    H = gate.shape[-1]
    sig = mode == "sigmoid"
    a = spread(torch.sigmoid(gate) if sig else gate, D)
    om = spread(torch.sigmoid(-gate), D) if sig else torch.ones_like(a)
    zero = torch.zeros(B, D, dtype=torch.float64, device=x.device)
    u = dstate.clone() if dstate is not None else zero
    before0 = h0 if h0 is not None else zero
    M, E = u.abs(), u.abs() * EPS32
    dx, dg = torch.empty_like(x), torch.empty_like(x)
    edx, edg = torch.empty_like(x), torch.empty_like(x)
    for t in reversed(range(T)):
        s = dh[:, t] + u
        M = dh[:, t].abs() + M
        E = E + 4 * EPS32 * M
        before = h[:, t - 1] if t else before0
        low = (before - x[:, t]) if sig else before
        lowm = before.abs() + x[:, t].abs() if sig else before.abs()
        slope = a[:, t] * om[:, t] if sig else 1.0
        dx[:, t] = om[:, t] * s
        edx[:, t] = om[:, t].abs() * (E + 16 * EPS32 * M)
        dg[:, t] = s * low * slope
        edg[:, t] = (E * low.abs() + 24 * EPS32 * M * lowm) * (slope if sig else 1.0)
        u = a[:, t] * s
        E = a[:, t].abs() * (E + 16 * EPS32 * M)
        M = a[:, t].abs() * M
    P = D // H if H else 1
    shape = (B, T, H, P)
    total = dg.reshape(shape).sum(-1)
    # the sum over a head's channels: at most P roundings of it in any order
    each = dg.abs().reshape(shape).sum(-1)
    return (dx, total, u), (edx, edg.reshape(shape).sum(-1) + P * EPS32 * each, E)


# --------------------------------------------------------------- dropout
def philox(key, counter):
    """Philox-4x32-10 on Python integers: four words from {k0, k1} and {c0..c3}."""
    k, c = list(key), list(counter)
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k[1], p0 & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def bits16(seed, offset, first, n):
    """The 16-bit numbers of elements first .. first + n - 1 (numpy uint32)."""
    import numpy as np

    lo, hi = first // 8, (first + n + 7) // 8
    blk = np.arange(lo, hi, dtype=np.uint64)
    m = np.uint64(0xFFFFFFFF)
    s = np.uint64(32)
    c = [blk & m, blk >> s, np.full_like(blk, offset & 0xFFFFFFFF), np.full_like(blk, (offset >> 32) & 0xFFFFFFFF)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> s) ^ c[1] ^ np.uint64(k[0]), p1 & m, (p0 >> s) ^ c[3] ^ np.uint64(k[1]), p0 & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    w = np.stack(c, -1)
    h = np.stack([w & np.uint64(0xFFFF), w >> np.uint64(16)], -1).reshape(-1)
    return h[first - lo * 8:first - lo * 8 + n].astype(np.uint32)


def keep_mask(shape, p, seed, offset, device="cpu"):
    """(kept, factor): what dropout keeps of an array of `shape`, and what it multiplies it with."""
    k = math.floor(p * 65536 + 0.5)
    n = math.prod(shape)
    kept = torch.from_numpy(bits16(seed, offset, 0, n) >= k).reshape(shape).to(device)
    return kept, (65536 / (65536 - k) if k < 65536 else 0.0)


# ----------------------------------------------------------------- norms
def act(name, g):
    """The gate's value and slope."""
    if name == "linear":
        return g, torch.ones_like(g)
    s, om = torch.sigmoid(g), torch.sigmoid(-g)
    return (s, s * om) if name == "sigmoid" else (g * s, s * (1 + g * om))


def norm(x, z, w_post, w_pre, gate, activation, scale, eps, m):
    """(y, u, r_z, r_y) and the error bounds of y and u; m: the branch's factor (dropout and scale) per element."""
    D = x.shape[1]
    K = 32 + D / 32  # a thread's run of a row, the joining of threads, and the steps of an element
    if z is None:
        y, r_z, ey = x, None, torch.zeros_like(x)
    else:
        r_z = 1 / torch.sqrt((z * z).mean(1, keepdim=True) + eps)
        v = act(activation, gate)[0] if gate is not None else 1.0
        branch = torch.where(m != 0, m * v * (z * r_z * w_post), 0.0)
        y = x + branch
        ey = K * EPS32 * branch.abs() + EPS32 * (x.abs() + branch.abs())
    r_y = 1 / torch.sqrt((y * y).mean(1, keepdim=True) + eps)
    # the norm of a row with errors ey: its own error and the row's, through the mean of y * ey
    drift = (y.abs() * ey).mean(1, keepdim=True) * r_y ** 2
    eu = (ey + y.abs() * (drift + K * EPS32)) * r_y * w_pre.abs()
    return (y, y * r_y * w_pre, r_z, r_y), (ey, eu, drift + K * EPS32)


def norm_backward(dy, du, y, z, w_post, w_pre, r_z, r_y, gate, activation, m):
    """(dx, dz, dg per element, dw_post per element, dw_pre per element) and their error bounds."""
    R, D = y.shape
    K = 48 + D / 32
    zero = torch.zeros_like(y)
    dy, du = dy if dy is not None else zero, du if du is not None else zero
    yh, wu = y * r_y, du * w_pre
    dx = dy + r_y * (wu - yh * (wu * yh).mean(1, keepdim=True))
    mx = dy.abs() + r_y * (wu.abs() + yh.abs() * (wu * yh).abs().mean(1, keepdim=True))
    out, err = {"dx": dx, "pre": du * yh}, {"dx": K * EPS32 * mx, "pre": 4 * EPS32 * (du * yh).abs()}
    if z is None:
        return out, err
    v, slope = act(activation, gate) if gate is not None else (torch.ones_like(y), None)
    zh = z * r_z
    d, md = torch.where(m != 0, dx * m, 0.0), mx * m.abs()
    dn, mn = d * v, md * v.abs()
    wn, mw = dn * w_post, mn * w_post.abs()
    out["dz"] = r_z * (wn - zh * (wn * zh).mean(1, keepdim=True))
    err["dz"] = 3 * K * EPS32 * r_z * (mw + zh.abs() * (mw * zh.abs()).mean(1, keepdim=True))
    out["post"], err["post"] = dn * zh, 2 * K * EPS32 * mn * zh.abs()
    if slope is not None:
        out["gate"] = d * (zh * w_post) * slope
        # silu's slope 1 + g (1 - s) may cancel: by magnitude it is 1 + |g|
        ms = (1 + gate.abs()) * (torch.sigmoid(gate) if activation == "silu" else 1.0) if activation == "silu" else slope.abs()
        err["gate"] = 2 * K * EPS32 * md * (zh * w_post).abs() * ms
    return out, err


# ---------------------------------------------------------------- policy
def policy(z, targets, old, adv, ref, mask, lo, hi, beta, grad_scale):
    """loss, logp, kl, clipped, dlogits and the error bounds of loss, logp, kl and dlogits."""
    N, V = z.shape
    top = z.max(1, keepdim=True).values
    base = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(z - base)
    total = e.sum(1, keepdim=True)
    ok = (targets >= 0) & (targets < V)
    at = targets.clamp(0, max(V - 1, 0))[:, None]
    logp = torch.where(ok, (z.gather(1, at) - base - total.log())[:, 0], math.nan)
    rho = torch.exp(logp - old)
    clipped = ((adv > 0) & (rho > 1 + hi) | (adv < 0) & (rho < 1 - lo)) & mask
    bound = torch.where(adv > 0, 1 + hi, 1 - lo)
    value = -torch.where(clipped, bound, rho) * adv
    slope = torch.where(clipped, 0.0, -rho * adv)
    q = ref - logp if ref is not None else torch.zeros_like(logp)
    kl = torch.expm1(q) - q
    value, slope = value + beta * kl, slope - beta * torch.expm1(q)
    count = max(1, int(mask.sum()))
    factor = grad_scale / count
    inside = mask[:, None]
    onehot = torch.zeros_like(z)
    onehot.scatter_(1, at, 1.0)
    grad = torch.where(inside, factor * slope[:, None] * (onehot - e / total), 0.0)
    loss = torch.where(mask, value, 0.0).sum() / count
    # the exponent's argument is rounded to a part of its size; the sum runs over V in any order of at
    # least 256 parts
    span = torch.where(z == -math.inf, 0.0, (z - base).abs()).max(1).values
    K = 64 + V / 256
    el = EPS32 * (2 * span + K + 4 * (logp.abs() + base[:, 0].abs()))
    em = EPS32 * (4 * (logp.abs() + old.abs()) + 8)  # of rho's argument, beside that of logp
    er = (el + em) * rho * adv.abs() * (1 + el)
    ek = (el + 4 * EPS32 * (logp.abs() + q.abs())) * torch.expm1(q).abs() + 8 * EPS32 * (torch.expm1(q).abs() + q.abs())
    ev = er + beta * ek + 4 * EPS32 * (value.abs() + rho * adv.abs() + beta * kl)
    es = er + beta * (el + 4 * EPS32 * (logp.abs() + q.abs()) + 8 * EPS32) * torch.exp(q) + 4 * EPS32 * ((rho * adv).abs() + beta * torch.expm1(q).abs())
    p = e / total
    ms = (rho * adv).abs() * ~clipped + beta * torch.expm1(q).abs()
    eg = abs(factor) * (es[:, None] * (onehot + p) + ms[:, None] * p * EPS32 * (2 * span[:, None] + K + 16)
                        + 4 * EPS32 * ms[:, None] * (onehot + p))
    zero = torch.zeros_like(logp)
    eloss = torch.where(mask, ev + EPS32 * (16 + N / 256) * value.abs(), 0.0).sum() / count
    return ({"loss": loss, "logp": torch.where(mask, logp, 0.0), "kl": torch.where(mask, kl, 0.0), "clipped": clipped,
             "dlogits": grad},
            {"loss": eloss, "logp": torch.where(mask, el, zero), "kl": torch.where(mask, ek, zero),
             "dlogits": torch.where(inside, eg, 0.0)})
