"""A small recurrent policy, sampled and trained with the block operators.

Two blocks, each: input norm -> projection to a value, a forget gate and an output gate -> gated scan over time ->
projection back -> norm, gate, dropout and residual add, fused with the next block's input norm. Tokens are sampled one
at a time from the running states (gated_scan_step), then the policy is trained on what it sampled (gated_scan,
gated_residual_norm and their backward passes) with the clipped policy loss and its KL term. The matrix products and
the optimiser are torch's, on the same memory (from_torch / Array.torch() copy nothing).

The task: each token should be the one after the token before it (modulo the vocabulary).

    python examples/recurrent_policy.py [updates]
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import musapy_b200 as ms  # noqa: E402

VOCAB, DIM, BLOCKS, BATCH, TIME = 32, 64, 2, 128, 16
DROPOUT, SCALE = 0.05, 0.7


def arr(t):
    return ms.from_torch(t)


def make_params(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def mat(*shape):
        return torch.randn(*shape, device="cuda", generator=g) * shape[0] ** -0.5

    p = {"embed": mat(VOCAB, DIM) * VOCAB ** 0.5, "head": mat(DIM, VOCAB) * 0.1, "pre0": torch.ones(DIM, device="cuda")}
    for i in range(BLOCKS):
        p[f"in{i}"], p[f"out{i}"] = mat(DIM, 3 * DIM), mat(DIM, DIM)
        p[f"post{i}"], p[f"pre{i + 1}"] = torch.ones(DIM, device="cuda"), torch.ones(DIM, device="cuda")
    return p


def split(proj):
    """The value, the forget gate and the output gate: views of one product, not copies."""
    return [arr(t) for t in proj.split(DIM, dim=-1)]


def block_norm(p, i, x, z, o, dropout=0.0, seed=0):
    return ms.gated_residual_norm(x, arr(z), arr(p[f"post{i}"]), arr(p[f"pre{i + 1}"]), gate=o, activation="silu",
                                  scale=SCALE, dropout=dropout, seed=seed, offset=i)


def sample(p, start, generator):
    """Tokens (BATCH, TIME) and the log-probabilities that they had, one step at a time."""
    states = [ms.zeros((BATCH, DIM), "f32", "cuda:0") for _ in range(BLOCKS)]
    token, tokens, logps = start, [], []
    for _ in range(TIME):
        x = arr(p["embed"][token])
        u, _ = ms.rms_norm(x, arr(p["pre0"]))
        for i in range(BLOCKS):
            v, g, o = split(u.torch() @ p[f"in{i}"])
            h = ms.gated_scan_step(states[i], v, g, mode="sigmoid")
            x, u, _ = block_norm(p, i, x, h.torch() @ p[f"out{i}"], o)
        logp = torch.log_softmax(u.torch() @ p["head"], -1)
        token = torch.multinomial(logp.exp(), 1, generator=generator)[:, 0]
        tokens.append(token)
        logps.append(logp.gather(1, token[:, None])[:, 0])
    return torch.stack(tokens, 1), torch.stack(logps, 1)


def logits_of(p, fed, dropout=0.0, seed=0):
    """Logits (BATCH, TIME, VOCAB) of whole sequences, and what the backward pass needs."""
    x = arr(p["embed"][fed])
    u, rstd0 = ms.rms_norm(x, arr(p["pre0"]))
    kept = [(x, rstd0)]
    for i in range(BLOCKS):
        v, g, o = split(u.torch() @ p[f"in{i}"])
        h = ms.gated_scan(v, g, mode="sigmoid")
        z = h.torch() @ p[f"out{i}"]
        y, u_next, rstd = block_norm(p, i, x, z, o, dropout, seed)
        kept.append((u, v, g, o, h, z, y, rstd))
        x, u = y, u_next
    return u.torch() @ p["head"], u, kept


def gradients(p, fed, dlogits, u, kept, dropout, seed):
    flat = lambda t: t.reshape(-1, t.shape[-1])
    grads = {"head": flat(u.torch()).t() @ flat(dlogits)}
    du, dy = dlogits @ p["head"].t(), None
    for i in reversed(range(BLOCKS)):
        u, v, g, o, h, z, y, rstd = kept[i + 1]
        dx, dz, do, dpost, dpre = ms.gated_residual_norm_backward(
            dy, arr(du.contiguous()), y, arr(z), arr(p[f"post{i}"]), arr(p[f"pre{i + 1}"]), rstd, gate=o, activation="silu",
            scale=SCALE, dropout=dropout, seed=seed, offset=i)
        grads[f"post{i}"], grads[f"pre{i + 1}"] = dpost.torch(), dpre.torch()
        grads[f"out{i}"] = flat(h.torch()).t() @ flat(dz.torch())
        dv, dg, _ = ms.gated_scan_backward(arr(dz.torch() @ p[f"out{i}"].t()), v, g, h, mode="sigmoid")
        dproj = torch.cat([dv.torch(), dg.torch(), do.torch()], -1)
        grads[f"in{i}"] = flat(u.torch()).t() @ flat(dproj)
        du, dy = dproj @ p[f"in{i}"].t(), dx
    x, rstd0 = kept[0]
    dx, dpre = ms.rms_norm_backward(arr(du), x, arr(p["pre0"]), rstd0, dy=dy)
    grads["pre0"] = dpre.torch()
    grads["embed"] = torch.zeros_like(p["embed"]).index_add_(0, fed.reshape(-1), flat(dx.torch()))
    return grads


def train(updates=60, seed=0, report=print):
    """Mean rewards, one for each update."""
    p = make_params(seed)
    reference = {k: v.clone() for k, v in p.items()}  # the KL term keeps the policy near it
    opt = torch.optim.Adam(list(p.values()), lr=1e-2)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    rewards = []
    for step in range(updates):
        start = torch.randint(0, VOCAB, (BATCH,), device="cuda", generator=g)
        tokens, old = sample(p, start, g)
        fed = torch.cat([start[:, None], tokens[:, :-1]], 1)
        reward = (tokens == (fed + 1) % VOCAB).float()
        advantage = (reward - reward.mean()) / (reward.std() + 1e-4)
        ref = torch.log_softmax(logits_of(reference, fed)[0], -1).gather(2, tokens[..., None])[..., 0].contiguous()
        for epoch in range(2):
            drop_seed = step * 2 + epoch
            logits, u, kept = logits_of(p, fed, DROPOUT, drop_seed)
            loss = ms.policy_loss(arr(logits), arr(tokens), arr(old), arr(advantage), arr(ref), clip_low=0.2, clip_high=0.3,
                                  kl_coef=1e-3)
            grads = gradients(p, fed, loss.dlogits.torch(), u, kept, DROPOUT, drop_seed)
            for k, t in p.items():
                t.grad = grads[k]
            opt.step()
        rewards.append(float(reward.mean()))
        if step % 10 == 0 or step == updates - 1:
            report(f"update {step:3d}  reward {rewards[-1]:.3f}  loss {float(loss.loss.torch()):+.4f}  "
                   f"clipped {float(loss.clipped.torch().float().mean()):.3f}  kl {float(loss.kl.torch().mean()):.4f}")
    return rewards


if __name__ == "__main__":
    train(int(sys.argv[1]) if len(sys.argv) > 1 else 60)
