"""The operators around a recurrent language model, as measured cases: linear attention with a decay for each head,
distillation from a teacher's top logits, and the embedding with its gradient.

Each case is one call as a program makes it: a prompt or training batch forward or backward, one token of running
sequences, a loss with its gradient, a lookup, a table's gradient. ``run`` computes it in its plain form, elementary
torch operations in 32 bits (running sums of log-decays in 64), or through ``musapy_b200`` where ``own`` is true;
``exact`` computes it in 64 bits from the definition.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_CHUNK = 64  # of the plain form of linear attention


# ------------------------------------------------------------------ cases
def _attention(direction, batch, time, heads, q_heads, dk, dv, dtype, decay, packed):
    return {"op": "attention", "pass": direction, "batch": batch, "time": time, "heads": heads, "q_heads": q_heads,
            "dk": dk, "dv": dv, "dtype": dtype, "decay": decay, "packed": packed}


def _distill(rows, vocab, top, dtype, teacher, temperature, masked):
    return {"op": "distill", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype, "teacher": teacher,
            "temperature": temperature, "masked": masked}


def _embed(direction, tokens, vocab, dim, dtype, into):
    return {"op": "embed", "pass": direction, "tokens": tokens, "vocab": vocab, "dim": dim, "dtype": dtype,
            "into": into}


def listed():
    return [
        # one token for each of 64 running sequences: what serving calls for every layer and token
        {"name": "attention step 64x16h128 bf16", **_attention("step", 64, 1, 16, 16, 128, 128, "bf16", "token", 0)},
        # a training batch, forward and backward
        {"name": "attention fwd 8x4096x16h128 bf16",
         **_attention("forward", 8, 4096, 16, 16, 128, 128, "bf16", "token", 0)},
        {"name": "attention bwd 4x4096x16h128 bf16",
         **_attention("backward", 4, 4096, 16, 16, 128, 128, "bf16", "token", 0)},
        # documents packed into one long row, few heads: the row itself has to be split
        {"name": "attention fwd 1x32768x8h64 bf16", **_attention("forward", 1, 32768, 8, 8, 64, 64, "bf16", "token", 20)},
        # one fixed decay for each head, odd lengths and widths: prompts of a small model
        {"name": "attention fwd 3x777x6h40 f16", **_attention("forward", 3, 777, 6, 6, 40, 72, "f16", "head", 0)},
        # full precision, keys and queries shared by two heads each: its gradients sum over them
        {"name": "attention bwd 2x1000x4h96 f32", **_attention("backward", 2, 1000, 4, 2, 96, 80, "f32", "token", 0)},
        # a small batch over an odd vocabulary in full precision, and a large one over a large vocabulary
        {"name": "distill 511x32003 k20 f32", **_distill(511, 32003, 20, "f32", "f32", 2.0, 0.2)},
        {"name": "distill 4096x131072 k64 bf16", **_distill(4096, 131072, 64, "bf16", "bf16", 1.0, 0.1)},
        # the tokens of a decode step, and those of a training batch
        {"name": "embed 64 of 131072x4096 bf16", **_embed("forward", 64, 131072, 4096, "bf16", False)},
        {"name": "embed 32768 of 32000x4096 bf16", **_embed("forward", 32768, 32000, 4096, "bf16", False)},
        # a training batch's gradient, a new table of it; an odd one added to a tied table's
        {"name": "embed grad 32768 of 32000x2048 bf16", **_embed("backward", 32768, 32000, 2048, "bf16", False)},
        {"name": "embed grad 4097 of 50257x769 f32", **_embed("backward", 4097, 50257, 769, "f32", True)},
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over its logarithm; one in three is made a multiple of 64 if it can be."""
    n = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    if n >= 64 and rng.random() < 1 / 3:
        n -= n % 64
    return n


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "distill", "embed", "embed"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    if op == "attention":
        direction = rng.choice(["forward", "forward", "backward", "backward", "step"])
        dk, dv = rng.choice([16, 32, 64, 64, 80, 128, 128, 192, 256]), rng.choice([16, 24, 64, 64, 100, 128, 128, 256])
        q_heads = _log(rng, 1, 16)
        heads = q_heads * rng.choice([1, 1, 1, 2, 4])
        decay = rng.choice(["token", "token", "head"])
        if direction == "step":
            return _attention("step", _log(rng, 1, max(1, min(256, (1 << 24) // (heads * dk * dv)))), 1, heads, q_heads,
                              dk, dv, dtype, decay, 0)
        most = (1 << 24) // (heads * (dk + dv))  # tokens
        time = _log(rng, 1, max(1, min(32768, most)))
        batch = _log(rng, 1, max(1, min(16, most // time)))
        packed = rng.choice([0, 0, 1 + time // 700]) if decay == "token" else 0
        return _attention(direction, batch, time, heads, q_heads, dk, dv, dtype, decay, packed)
    if op == "distill":
        vocab = _log(rng, 1000, 131072)
        return _distill(_log(rng, 1, min(4096, (1 << 28) // vocab)), vocab, _log(rng, 1, 128), dtype,
                        rng.choice([dtype, "f32"]), rng.choice([1.0, 2.0, 0.7]), rng.choice([0.0, 0.3]))
    direction = rng.choice(["forward", "backward", "backward"])
    dim = _log(rng, 64, 8192)
    vocab = _log(rng, 100, min(262144, (1 << 27) // dim))
    tokens = _log(rng, 1, min(131072, (1 << 26) // dim))
    return _embed(direction, tokens, vocab, dim, dtype, direction == "backward" and rng.random() < 0.4)


# ----------------------------------------------------------------- inputs
def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    rng = torch.Generator(device="cuda")
    rng.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return torch.empty(shape, device="cuda").normal_(mean, std, generator=rng).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, device="cuda", generator=rng)

    if case["op"] == "attention":
        b, t, h, hq, dk, dv = (case[k] for k in ("batch", "time", "heads", "q_heads", "dk", "dv"))
        s = {"q": normal(b, t, hq, dk, dtype=dt), "k": normal(b, t, hq, dk, dtype=dt), "v": normal(b, t, h, dv, dtype=dt),
             "state": normal(b, h, dk, dv)}
        if case["decay"] == "head":  # memories from a few tokens to some hundred
            s["log_decay"] = -torch.exp2(-1.0 - 6.0 * torch.arange(h, device="cuda") / h)
        else:  # as trained models have them: most steps keep nearly all, some forget
            s["log_decay"] = torch.log(torch.sigmoid(normal(b, t, h, std=1.5, mean=3.0)))
        if case["packed"]:  # the sequences' first tokens drop the state
            s["log_decay"][whole(0, b, case["packed"]), whole(0, t, case["packed"])] = -math.inf
        if case["pass"] == "step":
            for k in ("q", "k", "v"):
                s[k] = s[k][:, 0]
            if case["decay"] == "token":
                s["log_decay"] = s["log_decay"][:, 0]
        if case["pass"] == "backward":
            s["do"], s["dstate"] = normal(b, t, h, dv, dtype=dt), normal(b, h, dk, dv)
        return s
    if case["op"] == "distill":
        n, v, k = case["rows"], case["vocab"], case["top"]
        real = v - 3  # the vocabulary is padded
        logits = normal(n, v, std=2.0)
        ids = (whole(0, real, n, 1) + whole(1, real // k + 1, n, 1) * torch.arange(k, device="cuda")) % real
        teacher = 6.0 + normal(n, k, std=2.0).sort(dim=1, descending=True).values
        logits.scatter_add_(1, ids, 0.7 * teacher + normal(n, k))  # the student has learned some of it
        logits[:, real:] = -math.inf
        short = whole(1, k + 1, n, 1).clamp(min=k - k // 4)  # some lists are shorter
        teacher = torch.where(torch.arange(k, device="cuda") < short, teacher, -math.inf)
        return {"logits": logits.to(dt), "ids": ids, "teacher": teacher.to(_DTYPES[case["teacher"]]),
                "mask": torch.rand(n, device="cuda", generator=rng) >= case["masked"]}
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    u = torch.rand(n, device="cuda", generator=rng, dtype=torch.float64)
    s = {"tokens": (v * u**3).long().clamp(max=v - 1)}  # few tokens are frequent, many are rare
    if case["pass"] == "forward":
        s["table"] = normal(v, d, dtype=dt)
    else:
        s["dout"] = normal(n, d, dtype=dt)
        if case["into"]:
            s["into"] = normal(v, d)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # a program that uses the framework holds its Arrays: views of the same memory
        import musapy_b200 as ms

        s = {k: ms.from_torch(v) for k, v in s.items()}
        s["ms"] = ms
    return {"case": case, **s}


# -------------------------------------------------------------- one pass
def run(state):
    case = state["case"]
    if own:
        return _OWN[case["op"]](case, state)
    return _PLAIN[case["op"]](case, state)


def _own_attention(case, s):
    ms = s["ms"]
    if case["pass"] == "step":
        o = ms.linear_attention_step(s["state"], s["q"], s["k"], s["v"], s["log_decay"])
        return {"o": o.torch(), "state": s["state"].torch()}
    if case["pass"] == "forward":
        o, state = ms.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], s["state"], return_state=True)
        return {"o": o.torch(), "state": state.torch()}
    dq, dk, dv, dg, dstate = ms.linear_attention_backward(s["do"], s["q"], s["k"], s["v"], s["log_decay"], s["state"],
                                                          s["dstate"])
    return {"dq": dq.torch(), "dk": dk.torch(), "dv": dv.torch(), "dlog_decay": dg.torch(), "dstate": dstate.torch()}


def _own_distill(case, s):
    r = s["ms"].distill_loss(s["logits"], s["ids"], s["teacher"], s["mask"], temperature=case["temperature"])
    return {"loss": r.loss.torch(), "kl": r.kl.torch(), "dlogits": r.dlogits.torch()}


def _own_embed(case, s):
    ms = s["ms"]
    scale = math.sqrt(case["dim"])
    if case["pass"] == "forward":
        return ms.embedding(s["table"], s["tokens"], scale=scale).torch()
    if case["into"]:
        return ms.embedding_backward(s["dout"], s["tokens"], scale=scale, into=s["into"]).torch()
    return ms.embedding_backward(s["dout"], s["tokens"], rows=case["vocab"], scale=scale).torch()


_OWN = {"attention": _own_attention, "distill": _own_distill, "embed": _own_embed}


# ------------------------------------------------------------ plain forms
def _scale(case):
    return 1 / math.sqrt(case["dk"])


def _heads(x, heads):
    """(B, T, Hq, D) to (B, T, H, D): each head of x for the H / Hq heads that share it."""
    return x if x.shape[2] == heads else x.repeat_interleave(heads // x.shape[2], dim=2)


def _unshare(x, heads):
    """The sum over the heads that share one."""
    b, t, h, d = x.shape
    return x if h == heads else x.reshape(b, t, heads, h // heads, d).sum(3)


def _chunks(x, t):
    """(B, T, H, ...) to (B H, chunks, chunk, ...), zeros behind the last step."""
    n = -(-t // _CHUNK)
    x = torch.nn.functional.pad(x.flatten(3), (0, 0, 0, 0, 0, n * _CHUNK - t)) if x.dim() == 4 else \
        torch.nn.functional.pad(x, (0, 0, 0, n * _CHUNK - t))[..., None]
    b, _, h, d = x.shape
    return x.reshape(b, n, _CHUNK, h, d).permute(0, 3, 1, 2, 4).reshape(b * h, n, _CHUNK, d)


def _unchunk(x, b, t):
    bh, n, c, d = x.shape
    return x.reshape(b, bh // b, n * c, d)[:, :, :t].transpose(1, 2)


class _Decays:
    """What the log-decays (B, T, H) make of pairs of steps of a chunk, of steps and its ends, of pairs of chunks: from
    running sums in 64 bits. -inf is a number whose exponential is zero."""

    def __init__(self, g, t):
        g = _chunks(g.double().clamp(min=-1e4), t)[..., 0]
        within = g.cumsum(2)
        whole = within[:, :, -1].cumsum(1)
        self.pair = (within[..., :, None] - within[..., None, :]).tril().exp().tril().float()
        self.into = within.exp().float()[..., None]  # from the chunk's start to a step
        self.rest = (within[:, :, -1:] - within).exp().float()[..., None]  # from a step to the chunk's end
        self.all = within[:, :, -1].exp().float()
        before = torch.cat([torch.zeros_like(whole[:, :1]), whole[:, :-1]], 1)
        self.start = before.exp().float()  # from the row's start to a chunk
        self.end = (whole[:, -1:] - whole).exp().float()  # from a chunk's end to the row's end
        self.total = whole[:, -1].exp().float()
        self.between = (before[:, :, None] - whole[:, None, :]).tril(-1).exp().tril(-1).float()  # [later, earlier]


def _states(decays, parts, first):
    """The state at each chunk's start and the last one, from what each chunk adds (N, n, Dk, Dv)."""
    n, c = parts.shape[:2]
    flat = parts.reshape(n, c, -1)
    start = decays.between @ flat + decays.start[..., None] * first.reshape(n, 1, -1)
    last = (decays.end[..., None] * flat).sum(1) + decays.total[:, None] * first.reshape(n, -1)
    return start.reshape(parts.shape), last.reshape(first.shape)


def _do_attention(case, s):
    dt, scale, h = _DTYPES[case["dtype"]], _scale(case), case["heads"]
    b, t = case["batch"], case["time"]
    if case["pass"] == "step":
        q, k, v = _heads(s["q"][:, None].float(), h)[:, 0], _heads(s["k"][:, None].float(), h)[:, 0], s["v"].float()
        s["state"].mul_(s["log_decay"].exp()[..., None, None]).add_(k[..., :, None] * v[..., None, :])
        return {"o": ((q[..., :, None] * s["state"]).sum(2) * scale).to(dt), "state": s["state"]}
    q, k, v = _chunks(_heads(s["q"].float(), h), t), _chunks(_heads(s["k"].float(), h), t), _chunks(s["v"].float(), t)
    e = _Decays(s["log_decay"].expand(b, t, h), t)
    first = s["state"].reshape(b * h, case["dk"], case["dv"])
    start, last = _states(e, (k * e.rest).transpose(2, 3) @ v, first)
    qk = (q @ k.transpose(2, 3)) * e.pair * scale
    if case["pass"] == "forward":
        o = qk @ v + (q * e.into * scale) @ start
        return {"o": _unchunk(o, b, t).to(dt), "state": last.reshape(s["state"].shape)}
    do = _chunks(s["do"].float(), t)
    # the states' gradients run from the last chunk to the first
    parts = (q * e.into * scale).transpose(2, 3) @ do
    flat = parts.flatten(2)
    dlast = s["dstate"].reshape(b * h, -1)
    dend = (e.between.transpose(1, 2) @ flat + e.end[..., None] * dlast[:, None]).reshape(parts.shape)
    dfirst = (e.start[..., None] * flat).sum(1) + e.total[:, None] * dlast
    dov = do @ v.transpose(2, 3)
    r = dov * e.pair * scale
    dv = qk.transpose(2, 3) @ do + e.rest * (k @ dend)
    dq_far, dk_far = e.into * scale * (do @ start.transpose(2, 3)), e.rest * (v @ dend.transpose(2, 3))
    dq, dk = r @ k + dq_far, r.transpose(2, 3) @ q + dk_far
    # a decay's gradient: what passes through its step, from steps and states before it to steps and states after
    m = (qk * dov).flip(2).cumsum(2).flip(2).tril(-1).sum(3)
    after = (q * dq_far).sum(3).flip(2).cumsum(2).flip(2)
    passed = (k * dk_far).sum(3)
    dg = m + after + passed.cumsum(2) - passed + (e.all * (start * dend).sum((2, 3)))[..., None]
    dg = _unchunk(dg[..., None], b, t)[..., 0]
    hq = case["q_heads"]
    return {"dq": _unshare(_unchunk(dq, b, t), hq).to(dt), "dk": _unshare(_unchunk(dk, b, t), hq).to(dt),
            "dv": _unchunk(dv, b, t).to(dt), "dlog_decay": dg.sum((0, 1)) if case["decay"] == "head" else dg.contiguous(),
            "dstate": dfirst.reshape(s["dstate"].shape)}


def _do_distill(case, s):
    tau, mask, ids = case["temperature"], s["mask"], s["ids"]
    z, teacher = s["logits"].float() / tau, s["teacher"].float() / tau
    p = torch.exp(teacher - teacher.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    logq = z.gather(1, ids) - top - total.log()
    logp = torch.where(p > 0, p, 1.0).log()
    kl = torch.where(p > 0, p * (logp - logq), 0.0).sum(1)
    count = mask.sum().clamp(min=1)
    by = torch.where(mask, tau / count, 0.0)[:, None]
    grad = e * (by / total)
    grad.scatter_add_(1, ids, -by * p)
    return {"loss": tau * tau * torch.where(mask, kl, 0.0).sum() / count, "kl": torch.where(mask, kl, 0.0),
            "dlogits": grad.to(_DTYPES[case["dtype"]])}


def _do_embed(case, s):
    scale = math.sqrt(case["dim"])
    if case["pass"] == "forward":
        return (s["table"][s["tokens"]].float() * scale).to(_DTYPES[case["dtype"]])
    table = s["into"] if case["into"] else torch.zeros(case["vocab"], case["dim"], device="cuda")
    return table.index_add_(0, s["tokens"], s["dout"].float() * scale)


_PLAIN = {"attention": _do_attention, "distill": _do_distill, "embed": _do_embed}


# ------------------------------------------------------------------- work
def work(case):
    """Each input read once and each output written once; the operations that the formulas ask for, those of linear
    attention in their chunked form."""
    e = _BYTES[case["dtype"]]
    if case["op"] == "attention":
        b, t, h, hq, dk, dv = (case[k] for k in ("batch", "time", "heads", "q_heads", "dk", "dv"))
        n, nq, states = b * t * h, b * t * hq, b * h * dk * dv
        gates = 4 * (n if case["decay"] == "token" else h)
        if case["pass"] == "step":
            return {"bytes": (2 * nq * dk + 2 * n * dv) * e + gates + 8 * states, "flops": 5 * states}
        pairs = min(t, _CHUNK) / 2  # of earlier steps in a chunk, on average
        if case["pass"] == "forward":
            return {"bytes": (2 * nq * dk + 2 * n * dv) * e + gates + 8 * states,
                    "flops": n * (2 * pairs * (dk + dv) + 4 * dk * dv)}
        return {"bytes": (4 * nq * dk + 3 * n * dv) * e + 2 * gates + 12 * states,
                "flops": n * (2 * pairs * (3 * dk + 2 * dv) + 10 * dk * dv)}
    if case["op"] == "distill":
        n, k = case["rows"] * case["vocab"], case["top"]
        return {"bytes": 2 * n * e + case["rows"] * (5 + k * (8 + _BYTES[case["teacher"]])), "flops": 6 * n}
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    if case["pass"] == "forward":  # of the table, the rows that are asked for
        return {"bytes": n * (2 * d * e + 8), "flops": n * d}
    u = v * (1 - math.exp(-n / v))  # rows that are touched, roughly: the tokens are not spread evenly
    return {"bytes": n * (d * e + 8) + 4 * d * (2 * min(u, n, v) if case["into"] else v), "flops": n * d}


# -------------------------------------------------------- 64-bit versions
def _exact_attention(case, s):
    scale, h, hq = _scale(case), case["heads"], case["q_heads"]
    b, t = case["batch"], case["time"]
    if case["pass"] == "step":
        s = {k: v[:, None] if k in ("q", "k", "v") else v for k, v in s.items()}
    q, k = (s[x].double()[:, :, torch.arange(h, device="cuda") // (h // hq)] for x in ("q", "k"))
    v, state = s["v"].double(), s["state"].double()
    a = s["log_decay"].double().exp()
    a = a.reshape(1, 1, h).expand(b, t, h) if case["decay"] == "head" else a.reshape(b, t, h)

    def on(state, i):
        return torch.baddbmm(state.flatten(0, 1) * a[:, i].reshape(-1, 1, 1), k[:, i].flatten(0, 1)[:, :, None],
                             v[:, i].flatten(0, 1)[:, None, :]).reshape(state.shape)

    if case["pass"] != "backward":
        o = torch.empty_like(v)
        for i in range(t):
            state = on(state, i)
            o[:, i] = torch.einsum("bhk,bhkv->bhv", q[:, i], state) * scale
        return {"o": o[:, 0] if case["pass"] == "step" else o, "state": state}
    do, dstate = s["do"].double(), s["dstate"].double()
    every = max(1, math.isqrt(t))
    kept = []
    for i in range(t):
        if i % every == 0:
            kept.append(state)
        state = on(state, i)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    da = torch.empty_like(a)
    for piece in reversed(range(len(kept))):
        steps = range(piece * every, min(t, (piece + 1) * every))
        states = [kept[piece]]
        for i in steps:
            states.append(on(states[-1], i))
        for i in reversed(steps):
            before, now = states[i - steps[0]], states[i - steps[0] + 1]
            dq[:, i] = torch.einsum("bhkv,bhv->bhk", now, do[:, i]) * scale
            dstate = dstate + torch.einsum("bhk,bhv->bhkv", q[:, i] * scale, do[:, i])
            dk[:, i] = torch.einsum("bhkv,bhv->bhk", dstate, v[:, i])
            dv[:, i] = torch.einsum("bhkv,bhk->bhv", dstate, k[:, i])
            da[:, i] = (dstate * before).sum((2, 3))
            dstate = dstate * a[:, i, :, None, None]
    dg = da * a
    return {"dq": dq.unflatten(2, (hq, -1)).sum(3), "dk": dk.unflatten(2, (hq, -1)).sum(3), "dv": dv,
            "dlog_decay": dg.sum((0, 1)) if case["decay"] == "head" else dg, "dstate": dstate}


def _exact_distill(case, s):
    tau, mask = case["temperature"], s["mask"]
    z = s["logits"].double().requires_grad_()
    logp = torch.log_softmax(s["teacher"].double() / tau, 1)
    logq = torch.log_softmax(z / tau, 1).gather(1, s["ids"])
    kl = torch.where(logp > -math.inf, torch.nn.functional.kl_div(logq, logp.clamp(min=-1e30), reduction="none",
                                                                  log_target=True), 0.0).sum(1)
    loss = tau**2 * (kl * mask).sum() / max(1, int(mask.sum()))
    grad, = torch.autograd.grad(loss, z)
    return {"loss": loss.detach(), "kl": kl.detach() * mask, "dlogits": grad}


def _exact_embed(case, s):
    if case["pass"] == "forward":
        return torch.nn.functional.embedding(s["tokens"], s["table"]).double() * case["dim"]**0.5
    table = s["into"].double() if case["into"] else torch.zeros(case["vocab"], case["dim"], device="cuda").double()
    return table.index_put_((s["tokens"],), s["dout"].double() * case["dim"]**0.5, accumulate=True)


def exact(case, seed):
    of = {"attention": _exact_attention, "distill": _exact_distill, "embed": _exact_embed}
    return of[case["op"]](case, _inputs(case, seed))
