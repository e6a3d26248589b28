"""Train a policy with memory on the hover environment, all of it on the GPU.

    python examples/hover_memory.py [--envs 1024] [--steps 64] [--updates 60]

As hover_policy.py, but the policy does not see the velocity: it has to come
from what was seen before.  The network's block is a norm, linear attention
over the steps of the episode and a feed-forward layer; where it acts the
attention's state is carried from step to step, in the update a rollout is gone
over at once, from the state that it began with.  Muon moves the matrices of
the block, AdamW the rest.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from puffysics_amd import policy  # noqa: E402
from puffysics_amd.hover import HoverEnvs  # noqa: E402

ACTIONS = 3                 # thrust levels 0, 1 and 2
SEEN = (0, 2)               # of the observation: all but the velocity
VALUE = 20.0                # the size of returns: the head's value is in units of it


class Net(torch.nn.Module):
    def __init__(self, width=64, heads=2):
        super().__init__()
        self.heads, self.head_width = heads, width // heads
        linear = torch.nn.Linear
        self.embed, self.head = linear(len(SEEN), width), linear(width, ACTIONS + 1)
        self.q, self.k, self.v, self.mix = (linear(width, width, bias=False) for _ in range(4))
        self.up, self.down = linear(width, 2 * width, bias=False), linear(2 * width, width, bias=False)
        self.norms = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(width)) for _ in range(3))
        # heads that remember some 4 steps to some 64
        self.register_buffer("decay", 1 - 0.5 ** torch.linspace(2, 6, heads))

    def matrices(self):
        return [x.weight for x in (self.q, self.k, self.v, self.mix, self.up, self.down)]

    def others(self):
        return [*self.embed.parameters(), *self.head.parameters(), *self.norms]

    def new_state(self, envs):
        return torch.zeros(envs, self.heads, self.head_width, self.head_width, device=self.decay.device)

    def block(self, x, attend):
        """`attend` gets q, k and v by heads."""
        h = self.embed(x)
        y = policy.rms_norm(h, self.norms[0]).out
        a = attend(*(f(y).unflatten(-1, (self.heads, self.head_width)) for f in (self.q, self.k, self.v)))
        y, h = policy.rms_norm(self.mix(a.flatten(-2)), self.norms[1], residual=h)
        y = policy.rms_norm(self.down(torch.relu(self.up(y))), self.norms[2], residual=h).out
        y = self.head(y)
        return y[..., :ACTIONS], y[..., ACTIONS] * VALUE

    def forward(self, x, starts, state=None):
        """Logits and values of a rollout [steps, envs, seen]."""
        return self.block(x, lambda q, k, v: policy.linear_attention(
            q, k, v, self.decay, state=state, starts=starts, scale=self.head_width ** -0.5).out)

    def act(self, x, starts, state):
        """Of one step [envs, seen]; the state is updated."""
        return self.block(x, lambda q, k, v: policy.linear_attention_step(
            q, k, v, self.decay, state, starts=starts, scale=self.head_width ** -0.5))


def train(envs=1024, steps=64, updates=60, seed=1, epochs=2, minibatches=4, report=None):
    """The mean reward of each update's rollout (an episode is 256 steps)."""
    torch.manual_seed(seed)
    env = HoverEnvs(envs, seed=seed)
    net = Net().cuda()
    muon = policy.Muon(net.matrices(), lr=3e-3)
    adamw = policy.AdamW(net.others(), lr=3e-3, weight_decay=0.0, max_grad_norm=0.5, seed=seed)
    obs = torch.zeros(steps, envs, len(SEEN), device="cuda")
    taken = torch.zeros(steps, envs, dtype=torch.int64, device="cuda")
    rewards, terminals, starts, values, old = (torch.zeros(steps, envs, device="cuda") for _ in range(5))
    state = net.new_state(envs)
    env.reset()
    env.terminals.fill_(1)                      # the first step begins an episode
    got = []
    for update in range(updates):
        began = state.clone()
        with torch.no_grad():
            for t in range(steps):
                obs[t], starts[t] = env.observations[:, SEEN], env.terminals
                logits, values[t] = net.act(obs[t], starts[t], state)
                # the largest of logits with Gumbel noise is drawn with their probabilities
                noise = -torch.empty_like(logits).exponential_().log()
                taken[t] = (logits + noise).argmax(-1)
                old[t] = policy.log_probs(logits, taken[t]).log_prob
                env.actions.copy_(taken[t])
                env.step()
                rewards[t], terminals[t] = env.rewards, env.terminals
            last = net.act(env.observations[:, SEEN], env.terminals, state.clone())[1]
        advantages, returns = policy.advantages(rewards, values, terminals, last, gamma=0.99, lam=0.95)
        advantages = (advantages - advantages.mean()) / (advantages.std() + 1e-8)
        for _ in range(epochs):
            for part in torch.randperm(envs, device="cuda").chunk(minibatches):
                x, begins, a, before, adv, ret = (y[:, part] for y in (obs, starts, taken, old, advantages, returns))
                logits, value = net(x, begins, began[part])
                now = policy.log_probs(logits, a)
                ratio = (now.log_prob - before).exp()
                gain = torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv).mean()
                loss = -gain + 0.5 * ((value - ret) / VALUE).square().mean() - 0.01 * now.entropy.mean()
                for p in net.parameters():
                    p.grad = None
                loss.backward()
                muon.step()
                norm = adamw.step()
        got.append(float(rewards.mean()))
        if report:
            report("update %3d  mean reward %6.3f  entropy %.3f  gradient norm %.3f" % (
                update, got[-1], float(now.entropy.detach().mean()), float(norm)))
    if report:
        report("episodes: %s" % env.log())
    muon.close()
    adamw.close()
    env.close()
    return got


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--envs", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--updates", type=int, default=60)
    ap.add_argument("--seed", type=int, default=1)
    args = ap.parse_args()
    train(args.envs, args.steps, args.updates, args.seed, report=print)
