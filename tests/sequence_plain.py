"""The operators of a recurrent language model in 64 bits (torch float64), straight from their formulas, and bounds on
what the kernels' arithmetic may make of them.

A bound is a number of roundings times a majorant, the same formula with every term taken by its magnitude; the
rounding of a 16-bit result is added by blocks_plain.close. The numbers come from the formulas and the lengths."""
import math

import torch

EPS32 = 2.0 ** -24
# what scores lose before they meet values: bf16 keeps 8 bits of them, float16 16 bits in two numbers (their
# rounding, and twice the product of two second numbers that is left out), float 24
SCORES = {torch.bfloat16: 2.0 ** -8, torch.float16: 3 * 2.0 ** -16, torch.float32: 3 * EPS32}
CHUNK = 64


def spread(x, heads):
    return x.repeat_interleave(heads // x.shape[2], dim=2)


def attention(q, k, v, g, state, scale):
    """(o, last state) step by step; q, k (B, T, Hq, DK), v (B, T, H, DV), g (B, T, H) or (H,), state or None."""
    B, T, H, DV = v.shape
    q, k = spread(q, H), spread(k, H)
    a = g.expand(B, T, H).exp()
    S = torch.zeros(B, H, q.shape[3], DV, dtype=v.dtype, device=v.device) if state is None else state
    o = []
    for t in range(T):
        S = S * a[:, t, :, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :]
        o.append((q[:, t, :, :, None] * S).sum(2) * scale)
    return (torch.stack(o, 1) if T else torch.zeros_like(v)), S


def attention_backward(do, q, k, v, g, state, dstate, scale):
    """(dq, dk, dv, dg per step, dstate0) step by step."""
    B, T, H, DV = v.shape
    Hq, DK = q.shape[2:]
    q, k = spread(q, H), spread(k, H)
    a = g.expand(B, T, H).exp()
    zero = torch.zeros(B, H, DK, DV, dtype=v.dtype, device=v.device)
    S = [zero if state is None else state]
    for t in range(T):
        S.append(S[-1] * a[:, t, :, None, None] + k[:, t, :, :, None] * v[:, t, :, None, :])
    U = zero if dstate is None else dstate
    dq, dk, dv, dg = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), torch.empty_like(a)
    for t in reversed(range(T)):
        dq[:, t] = (S[t + 1] * do[:, t, :, None, :]).sum(3) * scale
        U = U + q[:, t, :, :, None] * do[:, t, :, None, :] * scale
        dk[:, t] = (U * v[:, t, :, None, :]).sum(3)
        dv[:, t] = (U * k[:, t, :, :, None]).sum(2)
        U = U * a[:, t, :, None, None]
        dg[:, t] = (U * S[t]).sum((2, 3))
    join = lambda x: x.reshape(B, T, Hq, H // Hq, DK).sum(3)
    return join(dq), join(dk), dv, dg, U


def roundings(T, DK, DV):
    """On the longest way to a result: a decay's exponent (up to 104, and a few), the sums over channels and a chunk, 16
    terms to a tensor core step that may cut instead of round, and one for every chunk that a state passes."""
    return 2 * (110 + (DK + DV) / 8 + CHUNK / 4 + 4 * math.ceil(T / CHUNK))


def attention_bounds(q, k, v, g, state, scale, dtype):
    """Bounds of o and the last state."""
    mag = lambda x: None if x is None else x.abs()
    o, S = attention(q.abs(), k.abs(), v.abs(), g, mag(state), abs(scale))
    n = roundings(v.shape[1], q.shape[3], v.shape[3]) * EPS32
    return (n + SCORES[dtype]) * o, n * S


def attention_backward_bounds(do, q, k, v, g, state, dstate, scale, dtype):
    """Bounds of (dq, dk, dv, dg per step, dstate0)."""
    mag = lambda x: None if x is None else x.abs()
    dq, dk, dv, dg, U = attention_backward(do.abs(), q.abs(), k.abs(), v.abs(), g, mag(state), mag(dstate), abs(scale))
    T, DK, DV = v.shape[1], q.shape[3], v.shape[3]
    n = roundings(T, DK, DV) * EPS32
    u = n + SCORES[dtype]
    # a decay's gradient is joined from the sums of a chunk's rows and columns: as large as all of the chunk's
    H = v.shape[2]
    share = (spread(q.abs(), H) * attention_backward(do.abs(), spread(q.abs(), H), spread(k.abs(), H), v.abs(), g, mag(state),
                                                     mag(dstate), abs(scale))[0]).sum(3)
    pad = -T % CHUNK
    whole = torch.nn.functional.pad(share, (0, 0, 0, pad)).unflatten(1, (-1, CHUNK)).sum(2, keepdim=True)
    whole = whole.expand(-1, -1, CHUNK, -1).flatten(1, 2)[:, :T]
    return u * dq, u * dk, u * dv, n * (dg + 2 * whole), n * U


# ---------------------------------------------------------- distillation
def distill(z, ids, teacher, mask, tau, grad_scale):
    """(loss, kl, dlogits) and their bounds; z (N, V), ids and teacher (N, K), float64."""
    N, V = z.shape
    kl, ekl = z.new_zeros(N), z.new_zeros(N)
    grad, egrad = torch.zeros_like(z), torch.zeros_like(z)
    count = max(1, int(mask.sum()))
    for i in range(N):
        if not mask[i]:
            continue
        on = teacher[i] != -math.inf
        x, at = teacher[i][on] / tau, ids[i][on]
        if x.numel() == 0:
            continue
        if bool(x.isnan().any()) or bool(((at < 0) | (at >= V)).any()):
            kl[i], grad[i] = math.nan, math.nan
            continue
        logp, logq = torch.log_softmax(x, 0), torch.log_softmax(z[i] / tau, 0)
        p, q = logp.exp(), logq.exp()
        kl[i] = (p * (logp - logq[at])).sum()
        # each log: its value's rounding, its argument's (taken from the row's maximum) and that of the sum below it
        ekl[i] = (p * (64 + 8 * logp.abs() + 8 * logq[at].abs()) * (1 + (logp - logq[at]).abs())).sum() * EPS32
        by = grad_scale * tau / count
        part = torch.zeros_like(q).index_add_(0, at, p)
        slip = torch.zeros_like(q).index_add_(0, at, p * (64 + 8 * logp.abs()))
        grad[i] = by * (q - part)
        finite = torch.where(logq > -math.inf, logq.abs(), 0.0)
        egrad[i] = abs(by) * (q * (64 + 8 * finite) + slip) * EPS32
    loss = tau * tau * kl.sum() / count
    return (loss, kl, grad), (tau * tau * (ekl.sum() + 64 * EPS32 * kl.abs().sum()) / count, ekl, egrad)


# ------------------------------------------------------------- embedding
def embedding_gradient(dout, tokens, V, scale):
    """(dtable, its bound), float64; tokens outside have no part."""
    on = (tokens >= 0) & (tokens < V)
    zero = torch.zeros(V, dout.shape[1], dtype=torch.float64, device=dout.device)
    at = tokens[on].long()
    count = torch.bincount(at, minlength=V).to(torch.float64)[:, None]
    table = zero.index_add(0, at, dout[on]) * scale
    return table, (count + 2) * EPS32 * zero.index_add(0, at, dout[on].abs()) * abs(scale)
