"""Tensors that puffysics_amd.policy has to read as torch does, or refuse."""
import pytest
import torch


def negated(x):
    """x as the imaginary part of a conjugate: marked as negated, every other
    number of the memory below."""
    return torch.complex(torch.zeros_like(x), -x).conj().imag


def test_negated_is_marked():
    x = negated(torch.tensor([1.0, -2.0]))
    assert x.is_neg() and x.tolist() == [1.0, -2.0] and x[:1].is_contiguous()


@pytest.mark.gpu
@pytest.mark.parametrize("actions", [1, 3, 300, 5000])
def test_log_probs_of_negated_logits(actions):
    """And of the gradient that comes in, of each output."""
    from puffysics_amd import policy
    g = torch.Generator().manual_seed(actions)
    x = torch.randn(7, actions, generator=g).cuda()
    taken = torch.randint(0, actions, (7,), generator=g).cuda()
    mask = (torch.rand(7, actions, generator=g) < 0.8).cuda()
    dl, dh = torch.randn(7, generator=g).cuda(), torch.randn(7, generator=g).cuda()
    for m in (None, mask):
        got, want = policy.log_probs(negated(x), taken, m, top=1), policy.log_probs(x, taken, m, top=1)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    want = torch.autograd.grad(policy.log_probs(x.requires_grad_(), taken)[:2], x, (dl, dh))[0]
    leaf = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(policy.log_probs(negated(leaf), taken)[:2], leaf, (dl, dh))[0], want)
    for pair in ((negated(dl), dh), (dl, negated(dh)), (negated(dl), negated(dh))):
        assert torch.equal(torch.autograd.grad(policy.log_probs(x, taken)[:2], x, pair)[0], want)
    # as autograd itself makes one
    z = torch.complex(torch.zeros_like(dl), policy.log_probs(x, taken).log_prob).conj() * torch.complex(dl, dh)
    d = torch.autograd.grad(z.real.sum(), x)[0]
    assert torch.equal(d, torch.autograd.grad(policy.log_probs(x, taken).log_prob, x, dh)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("steps,envs", [(1, 1), (1, 5), (200, 3), (40, 70)])
def test_advantages_of_negated_arrays(steps, envs):
    from puffysics_amd import policy
    g = torch.Generator().manual_seed(steps)
    r, v, d = (torch.randn(steps, envs, generator=g).cuda() for _ in range(3))
    d, last = (d > 1).float(), torch.randn(envs, generator=g).cuda()
    want = policy.advantages(r, v, d, last)
    for args in ((negated(r), v, d, last), (r, negated(v), d, last), (r, v, negated(d), last), (r, v, d, negated(last)),
                 [negated(x) for x in (r, v, d, last)]):
        got = policy.advantages(*args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_adamw_with_negated_gradients():
    from puffysics_amd import policy
    params, twins = ([torch.ones(n, device="cuda") for n in (1, 50, 1)] for _ in range(2))
    a, b = policy.AdamW(params), policy.AdamW(twins)
    g = torch.tensor([0.5, -0.25], device="cuda")
    long = torch.randn(50, device="cuda")
    for grads, marked in (([g[:1], long, g[1:]], [negated(g)[:1], long, negated(g)[1:]]),
                          ([None, long, g[1:]], [None, torch._neg_view(-long), negated(g)[1:]])):
        b.step(grads)
        a.step(marked)
        assert all(torch.equal(p, q) for p, q in zip(params, twins)) and torch.equal(a.moments()[0], b.moments()[0])
    assert [a.steps(i) for i in range(3)] == [1, 2, 2]


def test_negated_parameters_are_refused():
    from puffysics_amd import policy
    with pytest.raises(ValueError, match="negated"):
        policy.AdamW([negated(torch.ones(1))])


@pytest.mark.parametrize("needs", [False, True])
def test_tangents_are_refused(needs):
    """Nothing is launched: this runs without a GPU.  Without a tangent the
    next check is reached, also between the levels."""
    from puffysics_amd import policy
    from torch.autograd import forward_ad
    x, t = torch.randn(4, 6, requires_grad=needs), torch.zeros(4, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones(4, 6))
        for logits in (dual, dual * 2, dual[:, 1:3], dual.view(2, 2, 6)[0]):
            with pytest.raises(ValueError, match="forward-mode"):
                policy.log_probs(logits, t[:logits.shape[0]])
        with pytest.raises(ValueError, match="CUDA device"):
            policy.log_probs(x, t)
    with pytest.raises(ValueError, match="CUDA device"):
        policy.log_probs(dual, t)


@pytest.mark.gpu
def test_forward_mode_does_not_lose_the_tangent():
    from puffysics_amd import policy
    x, t = torch.randn(4, 6, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    with pytest.raises(Exception):
        torch.func.jvp(lambda y: policy.log_probs(y, t).log_prob, (x,), (torch.ones_like(x),))
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(ValueError):
            policy.log_probs(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), t)
        inside = policy.log_probs(x, t).log_prob
    assert torch.equal(inside, policy.log_probs(x, t).log_prob)


def test_sizes_past_the_limits_are_refused():
    """Nothing is launched: this runs without a GPU."""
    from puffysics_amd import policy
    one, none = torch.zeros(1), torch.zeros(1, dtype=torch.int64)
    for rows, actions in ((2, 2 ** 21 + 1), (2 ** 31, 3)):
        with pytest.raises(ValueError, match="at most 2"):
            policy.log_probs(one.expand(rows, actions), none.expand(rows))
    for steps, envs in ((2 ** 31, 1), (1, 2 ** 31)):
        x = one.expand(steps, envs)
        with pytest.raises(ValueError, match="at most 2"):
            policy.advantages(x, x, x, one.expand(envs))
    for rows, actions in ((2, 2 ** 21), (2 ** 31 - 1, 3)):
        with pytest.raises(ValueError, match="CUDA device"):          # the next check
            policy.log_probs(one.expand(rows, actions), none.expand(rows))


@pytest.mark.gpu
@pytest.mark.parametrize("lr", [-1e-3, float("nan")])
def test_rates_below_0_are_refused(lr):
    from puffysics_amd import policy
    p, g = torch.zeros(5, device="cuda"), torch.ones(5, device="cuda")
    opt = policy.AdamW([p], lr)
    with pytest.raises(ValueError):
        opt.step([g])
    with pytest.raises(ValueError):
        policy.AdamW([p]).step([g], lr=lr)
    assert opt.steps() == 0 and int(torch.count_nonzero(p)) == 0
    opt.step([g], lr=0.5)
    assert opt.steps() == 1 and (p < 0).all()


def test_rows_without_a_workspace():
    """The sizes for which log_probs does not ask are those that need none."""
    from puffysics_amd import policy
    lib = policy.policy_lib()
    for rows in (1, 16, 4096, 2 ** 20):
        for actions in (1, policy._SMALL - 1, policy._SMALL):
            assert lib.b3_log_probs_workspace(rows, actions, 32) == 0
        assert lib.b3_log_probs_workspace(rows, 2 ** 18, 32) > 0
    from b3test import ROOT
    text = open(ROOT + "/puffysics_amd/policy_csrc/b3_log_probs.hip").read()
    assert "kSmall = %d," % policy._SMALL in text
