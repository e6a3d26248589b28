"""The operators of a policy with memory together, as examples/hover_memory.py
has them: norm, linear attention over a rollout and step by step, log
probabilities, Muon and AdamW."""
import os
import sys

import pytest
import torch

from b3test import ROOT
from memorytest import attention_oracle, norm_oracle

sys.path.insert(0, os.path.join(ROOT, "examples"))


def plain(net, x, starts, state):
    """The network in 64 bits, by the definitions; [logits, values]."""
    w = {name: p.detach().double().requires_grad_() for name, p in net.named_parameters()}
    lin = lambda y, name: y @ w[name + ".weight"].t() + (w[name + ".bias"] if name + ".bias" in w else 0.0)  # noqa: E731
    h = lin(x.double(), "embed")
    y = norm_oracle64(h, w["norms.0"])
    q, k, v = (lin(y, name).unflatten(-1, (net.heads, net.head_width)) for name in "qkv")
    h, y = h, attention64(q, k, v, net.decay, state, starts, net.head_width ** -0.5)
    h = lin(y.flatten(-2), "mix") + h
    y = norm_oracle64(h, w["norms.1"])
    h = lin(torch.relu(lin(y, "up")), "down") + h
    y = lin(norm_oracle64(h, w["norms.2"]), "head")
    return y[..., :3], y[..., 3] * 20.0, w


def norm_oracle64(h, weight):
    return norm_oracle(h, weight, None, 1e-6)[0]


def attention64(q, k, v, decay, state, starts, scale):
    """attention_oracle, written so that autograd goes through."""
    by, s, out = decay.double()[:, None, None], state.double(), []
    for t in range(q.shape[0]):
        s = torch.where((starts[t] != 0)[:, None, None, None], 0.0, by * s) + k[t][..., :, None] * v[t][..., None, :]
        out.append(scale * (q[t][..., :, None] * s).sum(-2))
    got = torch.stack(out)
    assert torch.allclose(got.detach(), attention_oracle(q.detach(), k.detach(), v.detach(), decay, state, starts, scale)[0])
    return got


@pytest.mark.gpu
def test_network_and_gradients():
    """Forward, every gradient, and acting step by step, against 64 bits: a
    dozen operations of at most 128 terms each in 32 bits."""
    from hover_memory import Net
    from puffysics_amd import policy
    torch.manual_seed(3)
    steps, envs = 70, 5
    net = Net().cuda()
    x, starts = torch.randn(steps, envs, 2, device="cuda"), (torch.rand(steps, envs, device="cuda") < 0.05).float()
    state = torch.randn(envs, 2, 32, 32, device="cuda")
    taken = torch.randint(0, 3, (steps, envs), device="cuda")
    logits, values = net(x, starts, state)
    want_logits, want_values, w = plain(net, x, starts, state)
    assert (logits - want_logits).abs().max() < 1e-4 and (values - want_values).abs().max() < 1e-3
    up = torch.randn(steps, envs, device="cuda")
    got = policy.log_probs(logits, taken)
    ((got.log_prob * up).sum() + (values * up).sum() + got.entropy.sum()).backward()
    lp = torch.log_softmax(want_logits, -1)
    ((lp.gather(-1, taken[..., None])[..., 0] * up).sum() + (want_values * up).sum() - (lp.exp() * lp).sum()).backward()
    for name, p in net.named_parameters():
        most = w[name].grad.abs().max()
        assert (p.grad - w[name].grad).abs().max() < 1e-4 * most, name
    with torch.no_grad():
        for t in range(steps):
            step_logits, step_values = net.act(x[t], starts[t], state)
            assert (step_logits - want_logits[t]).abs().max() < 1e-4, t
            assert (step_values - want_values[t]).abs().max() < 1e-3, t


@pytest.mark.gpu
def test_example_runs():
    from hover_memory import train
    lines = []
    got = train(envs=64, steps=16, updates=3, report=lines.append)
    assert len(got) == 3 and all(-1.0 <= r <= 1.0 for r in got) and len(lines) == 4


@pytest.mark.gpu
def test_update_captured():
    """Rollout's forward pass, norm and Muon in one graph: every replay is what
    the eager calls give, with other work between."""
    from puffysics_amd import policy
    g = torch.Generator().manual_seed(1)
    made = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x, w, r = made(40, 6, 2, 32), torch.ones(32, device="cuda"), made(40, 6, 2, 32)
    decay, weights, twins = torch.tensor([0.9, 0.99], device="cuda"), [made(64, 64), made(200, 130)], []
    twins = [p.clone() for p in weights]
    grads = [made(64, 64), made(200, 130)]
    opt, twin = policy.Muon(weights), policy.Muon(twins)

    def once(opt):
        y, h = policy.rms_norm(x, w, residual=r)
        a = policy.linear_attention(y, h, y, decay, last=True)
        opt.step(grads)
        return y, h, a.out, a.state

    once(policy.Muon([p.clone() for p in weights]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once(opt)
    for i in range(3):
        x.mul_(0.5)
        grads[1].add_(0.1)
        graph.replay()
        want = once(twin)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        assert all(torch.equal(a, b) for a, b in zip(weights, twins)), i


class _Dropped(torch.autograd.Function):
    """x, which gets no gradient."""

    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, d):
        return None


@pytest.mark.gpu
def test_results_that_get_no_gradient():
    """The backward pass runs, and is given none."""
    from puffysics_amd import policy
    x, w = (torch.ones(*s, device="cuda", requires_grad=True) for s in ((4, 3, 2, 8), (8,)))
    _Dropped.apply(policy.rms_norm(x, w, residual=x).out).sum().backward()
    assert x.grad is None and w.grad is None
    _Dropped.apply(policy.linear_attention(x, x, x, torch.ones(2, device="cuda"), last=True).out).sum().backward()
    assert x.grad is None


def test_refusals_of_axes_and_scales():
    """Nothing is launched: this runs without a GPU."""
    from puffysics_amd import policy
    q, decay = torch.zeros(5, 3, 2, 8), torch.zeros(2)
    for v in (torch.zeros(()), torch.zeros(8), torch.zeros(1, 5, 3, 2, 8)):
        with pytest.raises(ValueError, match="one shape"):
            policy.linear_attention(q, q, v, decay)
    for scale in (1e39, -1e39):                  # infinite in 32 bits
        with pytest.raises(ValueError, match="finite"):
            policy.linear_attention(q, q, q, decay, scale=scale)
