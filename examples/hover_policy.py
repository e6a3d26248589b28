"""Train a small policy on the hover environment, all of it on the GPU.

    python examples/hover_policy.py [--envs 4096] [--steps 64] [--updates 60]

The environments step in libb3hover.so; the update around them is
puffysics_amd.policy: advantages of the rollout, log probabilities and
entropies of the taken actions with their gradient, and AdamW with the clip of
the gradients' norm.  The network itself is torch's.  The loss is the clipped
surrogate of a policy gradient, with a squared error on the value.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from puffysics_amd import policy  # noqa: E402
from puffysics_amd.hover import HoverEnvs  # noqa: E402

ACTIONS = 3                 # thrust levels 0, 1 and 2
VALUE = 20.0                # the size of returns: the head's value is in units of it


class Net(torch.nn.Module):
    def __init__(self, width=64):
        super().__init__()
        self.body = torch.nn.Sequential(torch.nn.Linear(3, width), torch.nn.Tanh(), torch.nn.Linear(width, width),
                                        torch.nn.Tanh())
        self.head = torch.nn.Linear(width, ACTIONS + 1)

    def forward(self, x):
        y = self.head(self.body(x))
        return y[..., :ACTIONS], y[..., ACTIONS] * VALUE


def train(envs=4096, steps=64, updates=60, seed=1, epochs=2, minibatches=4, state_bits=32, report=None):
    """The mean reward of each update's rollout (an episode is 256 steps)."""
    torch.manual_seed(seed)
    env = HoverEnvs(envs, seed=seed)
    net = Net().cuda()
    opt = policy.AdamW(net.parameters(), lr=3e-3, weight_decay=0.0, state_bits=state_bits, max_grad_norm=0.5, seed=seed)
    obs = torch.zeros(steps, envs, 3, device="cuda")
    taken = torch.zeros(steps, envs, dtype=torch.int64, device="cuda")
    rewards, terminals, values, old = (torch.zeros(steps, envs, device="cuda") for _ in range(4))
    env.reset()
    got = []
    for update in range(updates):
        with torch.no_grad():
            for t in range(steps):
                obs[t] = env.observations
                logits, values[t] = net(env.observations)
                # the largest of logits with Gumbel noise is drawn with their probabilities
                noise = -torch.empty_like(logits).exponential_().log()
                taken[t] = (logits + noise).argmax(-1)
                old[t] = policy.log_probs(logits, taken[t]).log_prob
                env.actions.copy_(taken[t])
                env.step()
                rewards[t], terminals[t] = env.rewards, env.terminals
            last = net(env.observations)[1]
        advantages, returns = policy.advantages(rewards, values, terminals, last, gamma=0.99, lam=0.95)
        flat = [x.reshape(steps * envs, *x.shape[2:]) for x in (obs, taken, old, advantages, returns)]
        for _ in range(epochs):
            for part in torch.randperm(steps * envs, device="cuda").chunk(minibatches):
                x, a, before, adv, ret = (y[part] for y in flat)
                adv = (adv - adv.mean()) / (adv.std() + 1e-8)
                logits, value = net(x)
                now = policy.log_probs(logits, a)
                ratio = (now.log_prob - before).exp()
                gain = torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv).mean()
                loss = -gain + 0.5 * ((value - ret) / VALUE).square().mean() - 0.01 * now.entropy.mean()
                for p in net.parameters():
                    p.grad = None
                loss.backward()
                norm = opt.step()
        got.append(float(rewards.mean()))
        if report:
            report("update %3d  mean reward %6.3f  entropy %.3f  gradient norm %.3f" % (
                update, got[-1], float(now.entropy.detach().mean()), float(norm)))
    if report:
        report("episodes: %s" % env.log())
    opt.close()
    env.close()
    return got


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--envs", type=int, default=4096)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--updates", type=int, default=60)
    ap.add_argument("--seed", type=int, default=1)
    ap.add_argument("--state-bits", type=int, default=32, choices=(8, 32))
    args = ap.parse_args()
    train(args.envs, args.steps, args.updates, args.seed, state_bits=args.state_bits, report=print)
