"""The example that runs the block operators together: its gradients against autograd of the same model in torch, and
that it learns."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example(ms):
    spec = importlib.util.spec_from_file_location("recurrent_policy", os.path.join(ROOT, "examples", "recurrent_policy.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def _torch_logits(ex, p, fed):
    """The model again in torch float64, step by step."""
    norm = lambda v, w: v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w
    x = p["embed"][fed]
    u = norm(x, p["pre0"])
    for i in range(ex.BLOCKS):
        v, g, o = (u @ p[f"in{i}"]).split(ex.DIM, -1)
        a, h, hs = torch.sigmoid(g), torch.zeros_like(v[:, 0]), []
        for t in range(v.shape[1]):
            h = a[:, t] * h + (1 - a[:, t]) * v[:, t]
            hs.append(h)
        z = torch.stack(hs, 1) @ p[f"out{i}"]
        x = x + ex.SCALE * torch.nn.functional.silu(o) * norm(z, p[f"post{i}"])
        u = norm(x, p[f"pre{i + 1}"])
    return u @ p["head"]


def test_example_gradients_are_autograds(example, ms):
    ex = example
    p = ex.make_params(3)
    g = torch.Generator(device="cuda").manual_seed(4)
    fed = torch.randint(0, ex.VOCAB, (ex.BATCH, ex.TIME), device="cuda", generator=g)
    logits, u, kept = ex.logits_of(p, fed)
    d = torch.randn(logits.shape, device="cuda", generator=g)
    got = ex.gradients(p, fed, d, u, kept, 0.0, 0)
    p64 = {k: v.double().requires_grad_() for k, v in p.items()}
    want_logits = _torch_logits(ex, p64, fed)
    # float32 products of 64 to 192 terms through two blocks: 1e-4 of the largest value
    assert (logits.double() - want_logits).abs().max() < 1e-4 * want_logits.abs().max()
    want = torch.autograd.grad((want_logits * d).sum(), list(p64.values()))
    for (k, a), b in zip(p64.items(), want):
        assert (got[k].double() - b).abs().max() < 1e-3 * b.abs().max() + 1e-6, k


def test_example_sampling_agrees_with_the_sequence_form(example, ms):
    """The log-probabilities of tokens sampled step by step are those that the whole sequence gives."""
    ex = example
    p = ex.make_params(5)
    g = torch.Generator(device="cuda").manual_seed(6)
    start = torch.randint(0, ex.VOCAB, (ex.BATCH,), device="cuda", generator=g)
    tokens, logp = ex.sample(p, start, g)
    fed = torch.cat([start[:, None], tokens[:, :-1]], 1)
    whole = torch.log_softmax(ex.logits_of(p, fed)[0], -1).gather(2, tokens[..., None])[..., 0]
    assert (whole - logp).abs().max() < 1e-3


def test_example_learns(example, ms):
    rewards = example.train(40, report=lambda line: None)
    assert sum(rewards[-5:]) / 5 > 3 * sum(rewards[:5]) / 5 + 0.1, rewards
