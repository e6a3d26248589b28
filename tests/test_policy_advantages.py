"""Advantages and returns of a rollout (puffysics_amd.policy.advantages)
against the recurrence in 64 bits.

Tolerance: a step rounds its terms a few times (5 units of the largest of
them), and an error made at one step reaches the ones before it times gamma
lambda each: over min(steps, 1 / (1 - gamma lambda)) steps, whatever the order
in which the steps are composed; the weights' own roundings add as much
again."""
import numpy as np
import pytest
import torch

from policytest import EPS32, advantages_oracle

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rollout(steps, envs, type, seed, ends=1 / 30):
    g = torch.Generator().manual_seed(seed)
    r = torch.rand(steps, envs, generator=g) * 2 - 1
    v = (torch.randn(steps, envs, generator=g) * 3).to(TYPES[type])
    d = (torch.rand(steps, envs, generator=g) < ends).float()
    last = (torch.randn(envs, generator=g) * 3).to(TYPES[type])
    return r, v, d, last


def check(r, v, d, last, gamma=0.99, lam=0.95, place=lambda x: x.cuda()):
    from puffysics_amd import policy
    adv, ret = policy.advantages(place(r), place(v), place(d), last.cuda(), gamma, lam)
    assert adv.shape == r.shape and ret.dtype == torch.float32
    want, returns = advantages_oracle(r.double().numpy(), v.double().numpy(), d.double().numpy(), last.double().numpy(), gamma, lam)
    a = gamma * lam
    reach = min(r.shape[0], 1 / (1 - a) if a < 1 else np.inf)
    fine = np.isfinite(want)
    tol = 10 * EPS32 * (reach + 1) * (np.abs(want[fine]).max(initial=0) + np.abs(np.nan_to_num(v.double().numpy())).max(initial=0) + 1)
    for got, w in ((adv, want), (ret, returns)):
        got = got.cpu().double().numpy()
        assert (np.isnan(got) == np.isnan(w)).all()
        bad = ~np.isnan(w) & (np.abs(got - w) > tol)
        assert not bad.any(), (bad.sum(), np.argwhere(bad)[0], got[bad][0], w[bad][0], tol)
    return adv, ret


SHAPES = [(1, 1), (1, 5), (2, 1), (3, 64), (7, 65), (16, 300), (63, 17), (64, 64), (65, 1000), (127, 3), (128, 4096), (255, 129),
          (257, 33), (500, 2), (1000, 16), (1023, 15), (1025, 9), (2048, 1), (4097, 40), (16385, 2), (70001, 1), (5, 20000),
          (200, 9000)]


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("steps,envs", SHAPES)
def test_sizes(steps, envs, type):
    check(*rollout(steps, envs, type, steps))


@pytest.mark.gpu
@pytest.mark.parametrize("steps,envs", SHAPES)
def test_environment_after_environment(steps, envs):
    """[envs, steps] arrays, as views."""
    adv, _ = check(*rollout(steps, envs, "f32", envs), place=lambda x: x.t().contiguous().cuda().t())
    if steps > 1 and envs > 1:
        assert adv.stride() == (1, steps)


@pytest.mark.gpu
@pytest.mark.parametrize("steps,envs", [(33, 70), (300, 40), (9000, 5)])
def test_slices(steps, envs):
    """Every other step and environment of larger arrays."""
    def place(x):
        big = torch.full((2 * steps + 1, 2 * envs + 3), float("nan"), dtype=x.dtype).cuda()
        big[1::2, 3::2] = x.cuda()
        return big[1::2, 3::2]
    check(*rollout(steps, envs, "bf16", 3), place=place)


@pytest.mark.gpu
@pytest.mark.parametrize("gamma,lam", [(1, 1), (0, 0.5), (0.5, 0), (0.999, 0.5), (0.3, 0.2)])
def test_rates(gamma, lam):
    for steps, envs in ((300, 20), (5000, 3)):
        check(*rollout(steps, envs, "f32", 4), gamma, lam)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8, torch.float32])
def test_terminals(dtype):
    for steps, envs in ((50, 70), (3000, 4)):
        for ends in (0.0, 0.3, 1.0):
            r, v, d, last = rollout(steps, envs, "f32", 6, ends)
            d = d.to(dtype)
            if dtype == torch.uint8:
                d *= 200
            check(r, v, d, last)


@pytest.mark.gpu
@pytest.mark.parametrize("steps,envs", [(40, 9), (3000, 4), (20000, 2)])
def test_an_episode_keeps_its_nan(steps, envs):
    """A NaN or infinity lies in its own episode alone."""
    r, v, d, last = rollout(steps, envs, "f32", 7, 0)
    d[steps // 2 - 1] = 1
    v[steps // 2] = float("nan")              # the first value of the second episodes
    last[0] = float("inf")
    r[steps - 1, 1:] = float("nan")
    adv, _ = check(r, v, d, last)
    assert torch.isfinite(adv[:steps // 2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("by_env", [False, True])
def test_places_past_32_bits(by_env):
    """More than 2^31 steps in all: the last environments have what they have
    alone."""
    from puffysics_amd import policy
    steps, envs = 1024, 2 ** 21 + 3
    shape = (envs, steps) if by_env else (steps, envs)
    turn = (lambda x: x.t()) if by_env else (lambda x: x)
    r, v = turn(torch.zeros(shape, device="cuda")), turn(torch.zeros(shape, dtype=torch.bfloat16, device="cuda"))
    d = turn(torch.zeros(shape, dtype=torch.uint8, device="cuda"))
    few = rollout(steps, 5, "bf16", 12)
    for to, x in zip((r, v, d), few):
        to[:, -5:].copy_(x)
    last = torch.zeros(envs, dtype=torch.bfloat16, device="cuda")
    last[-5:] = few[3].cuda()
    adv, ret = policy.advantages(r, v, d, last)
    alone = check(*few)
    assert torch.allclose(adv[:, -5:], alone[0], rtol=1e-5, atol=1e-4) and torch.allclose(ret[:, -5:], alone[1], rtol=1e-5, atol=1e-4)
    assert int(torch.count_nonzero(adv[:, :1000])) == 0 and int(torch.count_nonzero(adv[-1, :-5])) == 0


@pytest.mark.gpu
def test_more_environments_than_a_launch_takes():
    """2^24 - 1 workgroups of 64 environments and some more; one step, so that
    A = r - V, + gamma V_1 where the episode goes on, of three roundings."""
    from puffysics_amd import policy
    envs = (2 ** 24 - 1) * 64 + 70
    last = (torch.arange(envs, dtype=torch.int32, device="cuda") % 251).to(torch.bfloat16)
    ends = (torch.arange(envs, dtype=torch.int32, device="cuda") % 7 == 3).view(1, envs)
    r, v = (torch.full((1, 1), x, device="cuda").expand(1, envs) for x in (0.5, 0.25))
    adv, ret = policy.advantages(r, v.to(torch.bfloat16), ends, last, gamma=0.75)
    want = torch.where(ends[0], 0.25, 0.75 * last.float() + 0.25)
    assert float((adv[0] - want).abs().max()) <= 256 * 2.0 ** -23
    assert float((ret[0] - adv[0] - 0.25).abs().max()) <= 256 * 2.0 ** -23


@pytest.mark.gpu
def test_nothing():
    from puffysics_amd import policy
    for steps, envs in ((0, 4), (4, 0), (0, 0)):
        r = torch.zeros(steps, envs, device="cuda")
        adv, ret = policy.advantages(r, r, r, torch.zeros(envs, device="cuda"))
        assert adv.shape == (steps, envs) == ret.shape


@pytest.mark.gpu
def test_same_results_every_time_on_another_stream_and_captured():
    from puffysics_amd import policy
    for steps, envs in ((128, 700), (30000, 2)):
        r, v, d, last = (x.cuda() for x in rollout(steps, envs, "f32", 8))
        a = policy.advantages(r, v, d, last)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            b = policy.advantages(r, v, d, last)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = policy.advantages(r, v, d, last)
        for k in range(4):
            r.copy_(torch.randn_like(r))
            graph.replay()
            torch.cuda.synchronize()
            want = policy.advantages(r, v, d, last)
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.gpu
def test_the_environments_own_buffers():
    """A rollout of HoverEnvs, its reward and terminal buffers as they are."""
    from puffysics_amd import policy
    from puffysics_amd.hover import HoverEnvs
    envs, steps = HoverEnvs(100, seed=3), 300
    envs.reset()
    rewards, terminals = torch.zeros(steps, 100, device="cuda"), torch.zeros(steps, 100, device="cuda")
    values = torch.randn(steps, 100, device="cuda")
    for t in range(steps):
        envs.actions.copy_(torch.randint(0, 3, (100,)).float())
        envs.step()
        rewards[t], terminals[t] = envs.rewards, envs.terminals
    assert terminals.sum() > 50
    last = torch.randn(100, device="cuda")
    check(rewards.cpu(), values.cpu(), terminals.cpu(), last.cpu())
    envs.close()


def test_refusals():
    from puffysics_amd import policy
    r, last = torch.zeros(4, 6), torch.zeros(6)
    good = dict(rewards=r, values=r, terminals=r, last_values=last)
    for change in (dict(rewards=r[0]), dict(rewards=r.half()), dict(values=r[:3]), dict(values=r.double()),
                   dict(terminals=r.long()), dict(terminals=r[:, :2]), dict(last_values=last[:5]), dict(last_values=last.half()),
                   dict(gamma=1.5), dict(gamma=float("nan")), dict(lam=-0.1), dict()):
        with pytest.raises(ValueError):
            policy.advantages(**{**good, **change})


def test_refusals_of_the_c_entry():
    from puffysics_amd import policy
    lib, two = policy.policy_lib(), policy._ll * 2
    good = dict(steps=4, envs=6, rewards=64, rewards_stride=two(6, 1), values=64, values_type=0, values_stride=two(6, 1),
                last_values=64, last_values_stride=1, terminals=64, terminals_type=0, terminals_stride=two(6, 1),
                advantages=64, returns=64, out_stride=two(6, 1))
    call = lambda gamma=0.9, lam=0.9, **k: lib.b3_advantages_gpu(policy.B3Rollout(**{**good, **k}), gamma, lam, None, 0, None)  # noqa: E731
    for k in (dict(steps=-1), dict(envs=-1), dict(values_type=3), dict(terminals_type=1), dict(rewards=None), dict(values=None),
              dict(last_values=None), dict(terminals=None), dict(advantages=None), dict(returns=None), dict(gamma=1.1),
              dict(lam=-1.0), dict(lam=float("nan"))):
        assert call(**k) == 1, k
    assert lib.b3_advantages_gpu(None, 0.9, 0.9, None, 0, None) == 1
    assert call(steps=0) == 0 and call(envs=0) == 0
