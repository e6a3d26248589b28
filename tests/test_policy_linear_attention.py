"""puffysics_amd.policy.linear_attention and linear_attention_step against the
definition in 64 bits."""
import math

import pytest
import torch

from memorytest import STEP, attention_gradient_oracle, attention_oracle

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#        steps, envs, heads, key, value
SIZES = [(1, 1, 1, 1, 1), (1, 3, 2, 8, 5), (2, 1, 1, 16, 16), (15, 2, 3, 17, 33), (16, 1, 2, 32, 16), (31, 2, 1, 64, 64),
         (32, 1, 2, 48, 80), (33, 3, 1, 80, 48), (64, 2, 2, 64, 64), (65, 1, 3, 128, 128), (127, 2, 1, 100, 7),
         (200, 1, 2, 3, 128), (513, 1, 1, 33, 65)]


def made(steps, envs, heads, key, value, dtype, seed, rate=0.1):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(steps, envs, heads, d, generator=g).to(dtype) for d in (key, key, value))
    decay = 1 - torch.rand(heads, generator=g) ** 4            # from 0 to nearly 1
    starts = torch.rand(steps, envs, generator=g) < rate
    state = torch.randn(envs, heads, key, value, generator=g)
    return [x.cuda() for x in (q, k, v, decay, starts, state)]


def bounds(q, k, v, decay, state, starts, scale):
    """What the roundings of a step may add up to, relative to a step's own:
    the same sums of absolute values.  Weights decay^n come from a logarithm
    that is rounded: n |ln decay| decay^n is at most 2/e decay^(n / 2)."""
    state = None if state is None else state.abs()
    return attention_oracle(q.abs(), k.abs(), v.abs(), decay.sqrt(), state, starts, abs(scale))


def allowed(dtype, key, steps):
    """(factor of the sums of absolute values for out, for states): in 32 bits
    a term goes through the sums over `key` and over the steps, here or in
    blocks; in bfloat16 the scores are rounded once, and the state that they
    are multiplied with is two numbers, to 2^-16."""
    wide = (key + steps + 64) * 2.0 ** -24
    return (wide, wide) if dtype != torch.bfloat16 else (2.0 ** -8 + 2.0 ** -16 + wide, wide)


def close(got, want, bound, out_type):
    bad = (got.double() - want).abs() > bound + STEP[out_type] * want.abs() + 1e-30 + (
        2.0 ** -25 if out_type == torch.float16 else 0)                   # half a step of the least numbers
    assert not bad.any(), (got.double() - want)[bad].abs().max()
    assert torch.isfinite(got).all()


@pytest.mark.gpu
@pytest.mark.parametrize("given", ["nothing", "starts", "state", "both"])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward(size, type, given):
    from puffysics_amd import policy
    dtype, scale = TYPES[type], size[3] ** -0.5
    q, k, v, decay, starts, state = made(*size, dtype, sum(size))
    starts = starts if given in ("starts", "both") else None
    state = state if given in ("state", "both") else None
    got = policy.linear_attention(q, k, v, decay, state=state, starts=starts, scale=scale, last=True)
    want, states = attention_oracle(q, k, v, decay, state, starts, scale)
    most, most_states = bounds(q, k, v, decay, state, starts, scale)
    a, b = allowed(dtype, size[3], size[0])
    close(got.out, want, a * most, dtype)
    close(got.state, states[-1], b * most_states[-1], torch.float32)
    only = policy.linear_attention(q, k, v, decay, state=state, starts=starts, scale=scale)
    assert only.state is None and torch.equal(only.out, got.out)


@pytest.mark.gpu
@pytest.mark.parametrize("given", ["nothing", "both"])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_gradient(size, type, given):
    from puffysics_amd import policy
    dtype, scale = TYPES[type], size[3] ** -0.5
    q, k, v, decay, starts, state = made(*size, dtype, sum(size) + 1)
    g = torch.Generator().manual_seed(5)
    d_out = torch.randn(v.shape, generator=g).to(dtype).cuda()
    d_last = torch.randn(state.shape, generator=g).cuda()
    if given == "nothing":
        starts = state = d_last = None
    leaves = [x.requires_grad_() for x in (q, k, v, state) if x is not None]
    got = policy.linear_attention(q, k, v, decay, state=state, starts=starts, scale=scale, last=d_last is not None)
    outs, ups = ((got.out, got.state), (d_out, d_last)) if d_last is not None else ((got.out,), (d_out,))
    grads = torch.autograd.grad(outs, leaves, ups)
    with torch.no_grad():
        want = attention_gradient_oracle(q, k, v, decay, state, starts, scale, d_out, d_last)
        most = attention_gradient_oracle(q.abs(), k.abs(), v.abs(), decay.sqrt(), None if state is None else state.abs(),
                                         starts, scale, d_out.abs(), None if d_last is None else d_last.abs())
    a, b = allowed(dtype, max(size[3:]), size[0])
    for x, y, m in zip(grads[:3], want, most):
        close(x, y, a * m, dtype)
    if state is not None:
        close(grads[3], want[3], b * most[3], torch.float32)
    # one at a time: the same
    for i, leaf in enumerate(leaves):
        alone = policy.linear_attention(*(x.detach() if x is not leaf else x for x in (q, k, v)), decay,
                                        state=state if state is None or state is leaf else state.detach(), starts=starts,
                                        scale=scale, last=d_last is not None)
        assert torch.equal(torch.autograd.grad((alone.out, alone.state)[:len(ups)], leaf, ups)[0], grads[i])


@pytest.mark.gpu
def test_gradient_by_differences():
    from puffysics_amd import policy
    q, k, v, decay, starts, state = made(9, 2, 2, 4, 3, torch.float32, 3)
    g = torch.Generator().manual_seed(1)
    d_out, d_last = torch.randn(v.shape, generator=g).cuda(), torch.randn(state.shape, generator=g).cuda()
    leaves = [x.requires_grad_() for x in (q, k, v, state)]
    got = policy.linear_attention(q, k, v, decay, state=state, starts=starts, last=True)
    grads = torch.autograd.grad((got.out, got.state), leaves, (d_out, d_last))

    def loss(*xs):
        out, states = attention_oracle(*xs[:3], decay, xs[3], starts)
        return (out * d_out.double()).sum() + (states[-1] * d_last.double()).sum()

    base = [x.detach().double() for x in leaves]
    for i, (x, grad) in enumerate(zip(base, grads)):
        for at in range(0, x.numel(), max(1, x.numel() // 7)):
            up, down = x.clone(), x.clone()
            up.view(-1)[at] += 1e-4
            down.view(-1)[at] -= 1e-4
            # the loss is of the second degree in each: the difference is exact but for 64 bits' rounding
            d = (loss(*base[:i], up, *base[i + 1:]) - loss(*base[:i], down, *base[i + 1:])) / 2e-4
            assert abs(float(d) - float(grad.view(-1)[at])) < 1e-4 * (1 + abs(float(d)))


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (3, 2, 8, 5), (5, 3, 33, 17), (2, 2, 128, 128), (70, 4, 64, 64), (9, 1, 100, 30)])
def test_step(size, type):
    """Step after step it is the rollout's; the state is updated in place."""
    from puffysics_amd import policy
    dtype, steps = TYPES[type], 5
    q, k, v, decay, starts, state = made(steps, *size, dtype, sum(size), rate=0.4)
    want, states = attention_oracle(q, k, v, decay, state, starts, 0.5)
    most, most_states = bounds(q, k, v, decay, state, starts, 0.5)
    for t in range(steps):
        version = state._version
        out = policy.linear_attention_step(q[t], k[t], v[t], decay, state, starts=starts[t], scale=0.5)
        assert state._version > version
        wide = (size[2] + steps + 8) * 2.0 ** -24
        close(out, want[t], wide * most[t], dtype)
        close(state, states[t], wide * most_states[t], torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bool, torch.uint8])
def test_types_of_starts(dtype):
    from puffysics_amd import policy
    q, k, v, decay, starts, state = made(70, 3, 2, 16, 16, torch.float32, 2)
    want = policy.linear_attention(q, k, v, decay, state=state, starts=starts, last=True)
    got = policy.linear_attention(q, k, v, decay, state=state, starts=starts.to(dtype), last=True)
    turned = policy.linear_attention(q, k, v, decay, state=state, starts=starts.t().contiguous().t().to(dtype), last=True)
    for x in (got, turned):
        assert torch.equal(x.out, want.out) and torch.equal(x.state, want.state)
    a, b = state.clone(), state.clone()
    x = policy.linear_attention_step(q[0], k[0], v[0], decay, a, starts=starts[0])
    y = policy.linear_attention_step(q[0], k[0], v[0], decay, b, starts=starts[0].to(dtype))
    assert torch.equal(x, y) and torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
def test_strides(type):
    """Parts of a fused projection, environments first, broadcast heads, odd
    addresses: as contiguous copies of them."""
    from puffysics_amd import policy
    dtype, g = TYPES[type], torch.Generator().manual_seed(8)
    fused = torch.randn(3, 50, 2, 3 * 24 + 1, generator=g).to(dtype).cuda()      # environments, steps, heads
    parts = [fused[..., 24 * i + 1:24 * i + 25].transpose(0, 1) for i in range(3)]
    one = torch.randn(50, 3, 1, 24, generator=g).to(dtype).cuda().expand(50, 3, 2, 24)
    apart = torch.randn(50, 3, 2, 48, generator=g).to(dtype).cuda()[..., ::2]
    decay = torch.tensor([0.9, 0.97], device="cuda")
    d_out = torch.randn(2, 50, 3, 24, generator=g).to(dtype).cuda().permute(1, 2, 0, 3)
    for q, k, v in (parts, [parts[0], one, one], [apart, parts[1], apart]):
        xs = [x.detach().requires_grad_() for x in (q, k, v)]
        ys = [x.detach().contiguous().requires_grad_() for x in (q, k, v)]
        a, b = policy.linear_attention(*xs, decay).out, policy.linear_attention(*ys, decay).out
        assert a.is_contiguous() and torch.equal(a, b)
        for x, y in zip(torch.autograd.grad(a, xs, d_out), torch.autograd.grad(b, ys, d_out.contiguous())):
            assert torch.equal(x, y)
        for u, w in zip(xs, ys):
            u.requires_grad_(False), w.requires_grad_(False)
        sa, sb = torch.ones(3, 2, 24, 24, device="cuda"), torch.ones(3, 2, 24, 24, device="cuda")
        assert torch.equal(policy.linear_attention_step(*(x[7] for x in xs), decay, sa),
                           policy.linear_attention_step(*(x[7] for x in ys), decay, sb)) and torch.equal(sa, sb)


@pytest.mark.gpu
def test_gradient_of_shared_heads():
    """Keys that all heads share get the sum of the heads' gradients."""
    from puffysics_amd import policy
    q, k, v, decay, starts, _ = made(40, 2, 4, 16, 8, torch.float32, 4)
    shared = k[:, :, :1].clone().requires_grad_()
    each = shared.detach().expand(40, 2, 4, 16).contiguous().requires_grad_()
    up = torch.randn_like(v)
    a, = torch.autograd.grad(policy.linear_attention(q, shared.expand(40, 2, 4, 16), v, decay, starts=starts).out, shared, up)
    b, = torch.autograd.grad(policy.linear_attention(q, each, v, decay, starts=starts).out, each, up)
    assert torch.allclose(a, b.sum(2, keepdim=True), rtol=1e-6, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("key,value,steps", [(16, 16, 40), (64, 64, 100), (128, 40, 70)])
def test_what_an_episode_may_not_see(key, value, steps, type, bad):
    """NaN and infinities at a step are seen in the rest of its episode alone;
    back in time, in what came before it of the episode."""
    from puffysics_amd import policy
    q, k, v, decay, _, state = made(steps, 1, 1, key, value, TYPES[type], 6)
    decay = torch.tensor([0.9], device="cuda")
    starts = torch.zeros(steps, 1, device="cuda")
    first, at, after = steps // 3, steps // 2, steps // 2 + 3
    starts[first] = starts[after] = 1
    d_out = torch.randn_like(v)
    want_leaves = [x.detach().clone().requires_grad_() for x in (q, k, v)]
    want = policy.linear_attention(*want_leaves, decay, state=state, starts=starts, last=True)
    want_grads = torch.autograd.grad(want.out, want_leaves, d_out)
    for i in range(3):
        leaves = [x.detach().clone() for x in (q, k, v)]
        leaves[i][at] = bad
        leaves = [x.requires_grad_() for x in leaves]
        got = policy.linear_attention(*leaves, decay, state=state, starts=starts, last=True)
        out = got.out.detach()
        rest = torch.tensor([t < at or t >= after for t in range(steps)])
        assert torch.isfinite(out[rest]).all() and torch.isfinite(got.state).all()
        close(out[rest], want.out[rest].double(), 2.0 ** -7 * want.out.abs().max(), TYPES[type])
        assert not torch.isfinite(out[at]).all()
        episode = torch.tensor([t < first or t >= after for t in range(steps)])
        for x, y in zip(torch.autograd.grad(got.out, leaves, d_out), want_grads):
            assert torch.isfinite(x[episode]).all()
            close(x[episode], y[episode].double(), 2.0 ** -7 * y.abs().max(), TYPES[type])
    # of the upstream gradient
    d_bad = d_out.clone()
    d_bad[at] = bad
    for x in torch.autograd.grad(policy.linear_attention(*want_leaves, decay, state=state, starts=starts).out, want_leaves, d_bad):
        assert torch.isfinite(x[episode]).all() and not torch.isfinite(x[at]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_ends_of_the_decay(type):
    """0: each step alone.  1: plain sums.  Outside: NaN."""
    from puffysics_amd import policy
    q, k, v, _, _, state = made(100, 1, 4, 32, 32, TYPES[type], 7)
    decay = torch.tensor([0.0, 1.0, 1.5, -0.1], device="cuda")
    got = policy.linear_attention(q, k, v, decay, state=state, last=True)
    want, states = attention_oracle(q, k, v, decay, state)
    most, most_states = bounds(q[:, :, :2], k[:, :, :2], v[:, :, :2], decay[:2], state[:, :2], None, 1.0)
    a, b = allowed(TYPES[type], 32, 100)
    close(got.out[:, :, :2], want[:, :, :2], a * most, TYPES[type])
    close(got.state[:, :2], states[-1][:, :2], b * most_states[-1], torch.float32)
    assert got.out[1:, :, 2:].isnan().all() and got.state[:, 2:].isnan().all()
    s = state.clone()
    assert policy.linear_attention_step(q[0], k[0], v[0], decay, s)[:, 2:].isnan().all() and s[:, 2:].isnan().all()
    assert torch.allclose(s[:, 0], k[0, :, 0, :, None].float() * v[0, :, 0, None].float())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 3, 2), (5, 0, 2), (5, 3, 0)])
def test_nothing_to_do(shape):
    from puffysics_amd import policy
    steps, envs, heads = shape
    q, k, v, decay, starts, state = made(steps, envs, heads, 16, 8, torch.float32, 1)
    for x in (q, k, v, state):
        x.requires_grad_()
    got = policy.linear_attention(q, k, v, decay, state=state, starts=starts, last=True)
    assert got.out.shape == v.shape and torch.equal(got.state, state)
    d = torch.ones_like(got.state)
    grads = torch.autograd.grad((got.out, got.state), (q, k, v, state), (torch.ones_like(v), d))
    assert [g.shape for g in grads] == [x.shape for x in (q, k, v, state)] and torch.equal(grads[3], d)
    empty = policy.linear_attention(q, k, v, decay, last=True).state
    assert int(torch.count_nonzero(empty)) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(4000, 1, 2, 64, 64), (2500, 2, 1, 128, 96), (1500, 3, 1, 20, 33)])
def test_long(size, type):
    """Few sequences of many steps, which are cut into parts; starts far apart,
    so that memories cross the cuts."""
    from puffysics_amd import policy
    dtype, scale = TYPES[type], 0.2
    q, k, v, _, starts, state = made(*size, dtype, 9, rate=0.002)
    decay = 1 - 0.5 ** torch.linspace(3, 11, size[2], device="cuda")
    g = torch.Generator().manual_seed(2)
    d_out = torch.randn(v.shape, generator=g).to(dtype).cuda()
    d_last = torch.randn(state.shape, generator=g).cuda()
    leaves = [x.requires_grad_() for x in (q, k, v, state)]
    got = policy.linear_attention(q, k, v, decay, state=state, starts=starts, scale=scale, last=True)
    grads = torch.autograd.grad((got.out, got.state), leaves, (d_out, d_last))
    with torch.no_grad():
        want, states = attention_oracle(q, k, v, decay, state, starts, scale)
        most, most_states = bounds(q, k, v, decay, state, starts, scale)
        want_d = attention_gradient_oracle(q, k, v, decay, state, starts, scale, d_out, d_last)
        most_d = attention_gradient_oracle(q.abs(), k.abs(), v.abs(), decay.sqrt(), state.abs(), starts, scale, d_out.abs(),
                                           d_last.abs())
        a, b = allowed(dtype, max(size[3:]), size[0])
        close(got.out, want, a * most, dtype)
        close(got.state, states[-1], b * most_states[-1], torch.float32)
        for x, y, m in zip(grads[:3], want_d, most_d):
            close(x, y, a * m, dtype)
        close(grads[3], want_d[3], b * most_d[3], torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_a_rollout_in_two_halves(type):
    """The state that a first half leaves is what the second goes on from, and
    its gradient goes back through it."""
    from puffysics_amd import policy
    dtype = TYPES[type]
    q, k, v, decay, starts, state = made(90, 4, 2, 32, 32, dtype, 12)
    whole = policy.linear_attention(q, k, v, decay, state=state, starts=starts, last=True)
    first = policy.linear_attention(q[:41], k[:41], v[:41], decay, state=state, starts=starts[:41], last=True)
    second = policy.linear_attention(q[41:], k[41:], v[41:], decay, state=first.state, starts=starts[41:], last=True)
    most, most_states = bounds(q, k, v, decay, state, starts, 1.0)
    a, b = allowed(dtype, 32, 90)
    close(torch.cat([first.out, second.out]), whole.out.double(), 2 * a * most, dtype)
    close(second.state, whole.state.double(), 2 * b * most_states[-1], torch.float32)
    d_out = torch.randn_like(v)
    xs, ys = ([x.detach().clone().requires_grad_() for x in (q, k, v, state)] for _ in range(2))
    one = torch.autograd.grad(policy.linear_attention(*xs[:3], decay, state=xs[3], starts=starts).out, xs, d_out)
    h = policy.linear_attention(*(y[:41] for y in ys[:3]), decay, state=ys[3], starts=starts[:41], last=True)
    out = policy.linear_attention(*(y[41:] for y in ys[:3]), decay, state=h.state, starts=starts[41:]).out
    two = torch.autograd.grad((h.out, out), ys, (d_out[:41], d_out[41:]))
    with torch.no_grad():
        most = attention_gradient_oracle(q.abs(), k.abs(), v.abs(), decay.sqrt(), state.abs(), starts, 1.0, d_out.abs())
    for x, y, m, t in zip(one, two, most, (dtype, dtype, dtype, torch.float32)):
        close(x, y.double(), 2 * a * m, t)


@pytest.mark.gpu
def test_streams_and_replays():
    """On another stream than its tensors', and captured: every replay is the
    eager result of what the buffers hold then, with other work between."""
    from puffysics_amd import policy
    q, k, v, decay, starts, state = made(70, 8, 2, 32, 32, torch.bfloat16, 14)
    long = [torch.randn(3000, 1, 1, 64, device="cuda") for _ in range(3)]
    one = torch.tensor([0.99], device="cuda")
    side = torch.cuda.Stream()
    want = policy.linear_attention(q, k, v, decay, state=state, starts=starts, last=True)
    want_long = policy.linear_attention(*long, one, last=True)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = policy.linear_attention(q, k, v, decay, state=state, starts=starts, last=True)
    side.synchronize()
    assert torch.equal(got.out, want.out) and torch.equal(got.state, want.state)
    memory = state.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a = policy.linear_attention(q, k, v, decay, state=memory, starts=starts, last=True)
        b = policy.linear_attention(*long, one, last=True)
        c = policy.linear_attention_step(q[0], k[0], v[0], decay, memory, starts=starts[0])
    twin = state.clone()
    for i in range(3):
        v.add_(0.25)
        long[1].mul_(0.5)
        graph.replay()
        eager = policy.linear_attention(q, k, v, decay, state=twin, starts=starts, last=True)
        eager_long = policy.linear_attention(*long, one, last=True)
        step = policy.linear_attention_step(q[0], k[0], v[0], decay, twin, starts=starts[0])
        torch.cuda.synchronize()
        assert torch.equal(a.out, eager.out) and torch.equal(a.state, eager.state)
        assert torch.equal(b.out, eager_long.out) and torch.equal(b.state, eager_long.state)
        assert torch.equal(c, step) and torch.equal(memory, twin)
        torch.cuda.synchronize()
    assert torch.equal(want_long.out[:1], policy.linear_attention(*(x[:1] for x in long), one).out) or i == 2


@pytest.mark.gpu
def test_gradients_add_up_and_are_differentiable_once():
    from puffysics_amd import policy
    q, k, v, decay, starts, _ = made(20, 2, 2, 8, 8, torch.float32, 15)
    x = q.requires_grad_()
    out = policy.linear_attention(x, k, v, decay, starts=starts).out
    g, = torch.autograd.grad(out.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
    # q, k and v the same leaf
    leaf = torch.randn(20, 2, 2, 8, device="cuda", requires_grad=True)
    parts = [leaf.detach().clone().requires_grad_() for _ in range(3)]
    up = torch.randn(20, 2, 2, 8, device="cuda")
    total, = torch.autograd.grad(policy.linear_attention(leaf, leaf, leaf, decay).out, leaf, up)
    each = torch.autograd.grad(policy.linear_attention(*parts, decay).out, parts, up)
    assert torch.allclose(total, sum(each), rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(5, 2, 2, 64, 64), (40, 1, 2, 128, 128), (2000, 1, 1, 32, 32)])
def test_a_dropped_state_is_not_seen(size, type):
    """NaN in a state that an episode's start drops, forwards and back."""
    from puffysics_amd import policy
    q, k, v, decay, starts, state = made(*size, TYPES[type], 21, rate=0.0)
    starts[0] = True
    nan = torch.full_like(state, float("nan"))
    leaves = [x.requires_grad_() for x in (q, k, v, nan)]
    got = policy.linear_attention(q, k, v, decay, state=nan, starts=starts, last=True)
    want = policy.linear_attention(q.detach(), k.detach(), v.detach(), decay, starts=starts, last=True)
    assert torch.equal(got.state, want.state) and torch.equal(got.out, want.out)
    grads = torch.autograd.grad(got.out, leaves, torch.ones_like(v))
    assert all(torch.isfinite(g).all() for g in grads) and int(torch.count_nonzero(grads[3])) == 0
    s = nan.detach().clone()
    out = policy.linear_attention_step(q[0].detach(), k[0].detach(), v[0].detach(), decay, s, starts=starts[0])
    assert torch.isfinite(out).all() and torch.isfinite(s).all()


@pytest.mark.gpu
def test_negated_arrays():
    """Tensors that are only marked as negated are read as what they are."""
    from puffysics_amd import policy
    from test_policy_arguments import negated
    q, k, v, decay, starts, state = made(20, 2, 2, 8, 8, torch.float32, 22)
    d = torch.randn_like(v)
    want = policy.linear_attention(q, k, v, decay, state=state, last=True)
    got = policy.linear_attention(negated(q), negated(k), negated(v), negated(decay), state=negated(state), last=True)
    assert torch.equal(got.out, want.out) and torch.equal(got.state, want.state)
    x = q.clone().requires_grad_()
    a, = torch.autograd.grad(policy.linear_attention(x, k, v, decay).out, x, d)
    b, = torch.autograd.grad(policy.linear_attention(x, k, v, decay).out, x, negated(d))
    assert torch.equal(a, b)
    s, t = state.clone(), state.clone()
    assert torch.equal(policy.linear_attention_step(q[0], k[0], v[0], decay, s),
                       policy.linear_attention_step(negated(q[0]), negated(k[0]), negated(v[0]), decay, t)) and torch.equal(s, t)


@pytest.mark.gpu
def test_many_sequences():
    """The most there may be, of one step."""
    from puffysics_amd import policy
    envs, heads = 2 ** 20, 4
    q = torch.randn(1, envs, heads, 3, device="cuda")
    x = q.clone().requires_grad_()
    decay = torch.ones(heads, device="cuda")
    out = policy.linear_attention(x, x, x, decay).out
    want = (q * q).sum(-1, keepdim=True) * q
    assert torch.allclose(out, want, rtol=1e-5, atol=1e-5)
    d, = torch.autograd.grad(out, x, torch.ones_like(out))
    assert torch.allclose(d, (q * q).sum(-1, keepdim=True) + 2 * q * q.sum(-1, keepdim=True), rtol=1e-4, atol=1e-4)


def test_refusals():
    """Nothing is launched: this runs without a GPU."""
    from puffysics_amd import policy
    z = lambda *s, **kw: torch.zeros(*s, **kw)  # noqa: E731
    q, v, d, s = z(5, 3, 2, 8), z(5, 3, 2, 4), z(2), z(3, 2, 8, 4)
    ok = dict(q=q, k=q, v=v, decay=d)
    for what, change in (
            ("of one type", dict(k=q.half())), ("float32, float16", dict(q=q.double(), k=q.double(), v=v.double())),
            ("one shape", dict(k=z(5, 3, 2, 9))), ("one shape", dict(v=z(5, 3, 1, 4))), ("steps, envs", dict(q=q[0])),
            ("1 to 128", dict(q=z(5, 3, 2, 129), k=z(5, 3, 2, 129))), ("1 to 128", dict(v=z(5, 3, 2, 0))),
            ("1 to 128", dict(v=z(5, 3, 2, 129))), ("decay", dict(decay=z(3))), ("decay", dict(decay=d.double())),
            ("no gradient", dict(decay=z(2, requires_grad=True))), ("state", dict(state=s.half())),
            ("state", dict(state=s[:2])), ("starts", dict(starts=z(5, 2))), ("starts", dict(starts=z(5, 3).double())),
            ("finite", dict(scale=float("nan"))), ("finite", dict(scale=float("inf"))),
            ("2\\^22", dict(q=z(1).expand(1, 2 ** 21 + 1, 2, 8), k=z(1).expand(1, 2 ** 21 + 1, 2, 8),
                             v=z(1).expand(1, 2 ** 21 + 1, 2, 4))),
            ("2\\^31", dict(q=z(1).expand(2 ** 31, 1, 2, 8), k=z(1).expand(2 ** 31, 1, 2, 8), v=z(1).expand(2 ** 31, 1, 2, 4))),
            ("CUDA device", {})):
        with pytest.raises(ValueError, match=what):
            policy.linear_attention(**{**ok, **change})
    step = dict(q=q[0], k=q[0], v=v[0], decay=d, state=s)
    for what, change in (
            ("q has to be", dict(q=q)), ("state", dict(state=s.half())), ("state", dict(state=z(3, 2, 4, 8).transpose(2, 3))),
            ("starts", dict(starts=z(2))), ("no gradient", dict(state=s.clone().requires_grad_())),
            ("no gradient", dict(q=q[0].clone().requires_grad_())), ("CUDA device", {})):
        with pytest.raises(ValueError, match=what):
            policy.linear_attention_step(**{**step, **change})
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        for name in ("q", "k", "v"):
            with pytest.raises(ValueError, match="forward-mode"):
                policy.linear_attention(**{**ok, name: forward_ad.make_dual(ok[name], torch.ones_like(ok[name]))})


def test_c_refusals():
    """Of the C entries; no call reaches a launch."""
    import ctypes as C
    from puffysics_amd import policy
    lib = policy.policy_lib()
    one = (C.c_char * 64)()
    at = C.addressof(one)

    def call(**change):
        g = policy.B3Attention(1, 1, 1, 8, 8, 0, at, at, at, (8, 8, 8), (8, 8, 8), (8, 8, 8), at, None, 0, (0, 0), None, 1.0)
        for name, value in change.items():
            setattr(g, name, value)
        return lib.b3_linear_attention_gpu(C.byref(g), None if change.get("steps") != 0 else None, None, None, 0, None)

    for change in (dict(key=0), dict(key=129), dict(value=0), dict(value=129), dict(type=3), dict(steps=-1), dict(envs=-1),
                   dict(heads=-1), dict(q=None), dict(decay=None), dict(envs=(1 << 22) + 1), dict(steps=1 << 31), dict(),
                   dict(starts=at, starts_type=2), dict(scale=float("nan"))):
        assert call(**change) == 1, change
    assert call(envs=0) == 0 and call(heads=0) == 0 and call(steps=0) == 0
    assert lib.b3_linear_attention_gpu(None, None, None, None, 0, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
def test_columns_that_do_not_fill_vectors(type):
    """Every number of columns left over, of narrow and of wide heads; the
    last head's rows end the arrays."""
    from puffysics_amd import policy
    dtype = TYPES[type]
    for key in (*range(1, 18), 35, 39, 46, 62, 97, 109, 127):
        size = (40, 1, 2, key, 128 - key)
        q, k, v, decay, starts, state = made(*size, dtype, key)
        got = policy.linear_attention(q, k, v, decay, state=state, starts=starts, scale=0.1, last=True)
        want, states = attention_oracle(q, k, v, decay, state, starts, 0.1)
        most, most_states = bounds(q, k, v, decay, state, starts, 0.1)
        a, b = allowed(dtype, key, size[0])
        close(got.out, want, a * most, dtype)
        close(got.state, states[-1], b * most_states[-1], torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("type,size", [("f32", 2e34), ("f32", 3e38), ("f32", 1e-28), ("bf16", 1e37), ("bf16", 3e38),
                                       ("bf16", 1e-28), ("f16", 6e4)])
@pytest.mark.parametrize("key,value", [(1, 1), (64, 64), (128, 128), (17, 100)])
@pytest.mark.parametrize("decay", [0.9, 0.999, 1.0])
def test_sizes_of_numbers(type, size, key, value, decay):
    """States that 32 bits hold are right however large or small they are: of
    few sequences, in pieces, and of many, and step by step; the gradient of
    the state that was entered with alike."""
    from puffysics_amd import policy
    dtype, decay = TYPES[type], torch.tensor([decay], device="cuda")
    g = torch.Generator().manual_seed(key)
    steps = 300
    some = lambda d, size: ((torch.rand(steps, 1, 1, d, generator=g) + 0.5) * size).to(dtype).cuda()  # noqa: E731
    # one step of the size among small ones, or all of a small size
    at = slice(100, 101) if size > 1 else slice(0, steps)
    big = (torch.rand(steps, 1, 1, value, generator=g) * 0.5 + 0.5).mul(size).to(dtype).cuda()
    q, k, v = some(key, 1e-6 / key if size > 1e5 else 1e-3 if size > 1 else 1.0), some(key, 0.1), some(value, 1e-3)
    v[at] = big[at]

    def near(got, want, bound):
        assert ((got.double() - want).abs() <= bound + STEP[got.dtype] * want.abs() + (2.0 ** -25 if type == "f16" else 0)).all()

    want, states = attention_oracle(q, k, v, decay)
    a, b = allowed(dtype, key, steps)
    most, most_states = bounds(q, k, v, decay, None, None, 1.0)
    for envs in (1, 3000):
        got = policy.linear_attention(*(x.expand(steps, envs, 1, x.shape[-1]) for x in (q, k, v)), decay, last=True)
        for e in (0, envs - 1):
            near(got.out[:, e:e + 1], want, a * most)
            near(got.state[e:e + 1], states[-1], b * most_states[-1])
    s = torch.zeros(1, 1, key, value, device="cuda")
    for t in range(steps):
        policy.linear_attention_step(q[t], k[t], v[t], decay, s)
    near(s, states[-1], b * most_states[-1])
    # G grows by what comes in, as the state by v
    d_out, q, v = v, some(key, 0.1), some(value, 1e-3)
    for envs in (1, 3000):
        leaves = [x.expand(steps, envs, 1, x.shape[-1]).detach().requires_grad_() for x in (q, k, v)]
        leaves.append(torch.zeros(envs, 1, key, value, device="cuda", requires_grad=True))
        out = policy.linear_attention(*leaves[:3], decay, state=leaves[3]).out
        _, d_k, _, d_state = torch.autograd.grad(out, leaves, d_out.expand(steps, envs, 1, value))
        want = attention_gradient_oracle(q, k, v, decay, s, None, 1.0, d_out)
        most = attention_gradient_oracle(q, k, v, decay.sqrt(), s, None, 1.0, d_out)
        a, b = allowed(dtype, value, steps)
        for e in (0, envs - 1):
            near(d_state[e:e + 1], want[3], b * most[3])
            if type != "f16":
                near(d_k[:, e:e + 1], want[1], a * most[1])


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("decay,steps", [(1 - 2.0 ** -14, 16384), (1 - 2.0 ** -14, 1000), (1 - 2.0 ** -10, 30000),
                                         (0.97, 2000), (0.5, 100)])
def test_what_is_left_after_many_steps(decay, steps, type):
    """Of a state alone: decay^steps, forwards and back.  Its logarithm, to
    2^-23 of it, and the product with the steps are off by 1.5 2^-23 of the
    bits that the state falls by; a power and its product by 2^-22 each time
    that the state is gone over, which is once for 8 bits, or where pieces
    meet."""
    from puffysics_amd import policy
    decay = torch.tensor([decay], device="cuda")
    want = float(decay.double() ** steps)
    bits = -math.log2(want)
    for envs, pieces in ((3000, 0), (1, 64)):
        x = torch.zeros(1, 1, 1, 1, dtype=TYPES[type], device="cuda").expand(steps, envs, 1, 1)
        q, k, v = (x.detach().requires_grad_() for _ in range(3))
        state = torch.full((envs, 1, 1, 1), 3.0, device="cuda", requires_grad=True)
        got = policy.linear_attention(q, k, v, decay, state=state, last=True)
        d_state, = torch.autograd.grad(got.state, state, torch.full_like(state, 5.0))
        most = math.log(2) * bits * 1.5 * 2.0 ** -23 + (bits / 8 + 3 + pieces) * 2.0 ** -22
        assert float((got.state.detach().double() / (3 * want) - 1).abs().max()) <= most
        assert float((d_state.double() / (5 * want) - 1).abs().max()) <= most


@pytest.mark.gpu
@pytest.mark.parametrize("given", ["nothing", "both"])
@pytest.mark.parametrize("size", [*SIZES, (4000, 1, 2, 64, 64), (64, 300, 2, 64, 64)], ids=lambda s: "x".join(map(str, s)))
def test_sums_of_bfloat16(size, given):
    """Rounded once, at the end: scores and the state that bfloat16 numbers are
    multiplied with are two such numbers, to 2^-16 of them each (2^-18 where
    they lie evenly: the half step of a second number of 8 bits)."""
    from puffysics_amd import policy
    dtype, scale = torch.bfloat16, size[3] ** -0.5
    q, k, v, decay, starts, state = made(*size, dtype, sum(size))
    d_out = torch.randn(v.shape, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    starts, state = (starts, state) if given == "both" else (None, None)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    got = policy.linear_attention(q, k, v, decay, state=state, starts=starts, scale=scale).out
    grads = torch.autograd.grad(got, leaves, d_out)
    with torch.no_grad():
        want, _ = attention_oracle(q, k, v, decay, state, starts, scale)
        most, _ = bounds(q, k, v, decay, state, starts, scale)
        wants = attention_gradient_oracle(q, k, v, decay, state, starts, scale, d_out)
        mosts = attention_gradient_oracle(q.abs(), k.abs(), v.abs(), decay.sqrt(), None if state is None else state.abs(),
                                          starts, scale, d_out.abs())
        a = 2.0 ** -16 + (max(size[3:]) + size[0] + 64) * 2.0 ** -24
        for x, y, m in zip((got, *grads), (want, *wants), (most, *mosts)):
            close(x, y, a * m, dtype)
            # together: next to what the last rounding leaves, little
            far, least = (x.double() - y).norm(), (y.to(dtype).double() - y).norm()
            assert float(far) <= 1.01 * float(least) + 2.0 ** -16 * float(m.norm())


@pytest.mark.parametrize("name", ["q", "k", "v", "decay", "state"])
def test_tangents_are_refused(name):
    """Of every argument that a derivative could go through, the rollout's and
    the step's; without one the next check is reached.  Nothing is launched:
    this runs without a GPU."""
    from torch.autograd import forward_ad

    from puffysics_amd import policy
    z = torch.zeros
    rollout = dict(q=z(5, 3, 2, 8), k=z(5, 3, 2, 8), v=z(5, 3, 2, 4), decay=z(2), state=z(3, 2, 8, 4))
    step = {n: x[0] if n in "qkv" else x for n, x in rollout.items()}
    with forward_ad.dual_level():
        for call, args in ((policy.linear_attention, rollout), (policy.linear_attention_step, step)):
            with pytest.raises(ValueError, match="forward-mode"):
                call(**{**args, name: forward_ad.make_dual(args[name], torch.ones_like(args[name]))})
            with pytest.raises(ValueError, match="CUDA device"):
                call(**args)


def test_c_no_decay():
    """Where a launch reads the decay it has to be there, also for no steps; a
    call without work is none.  No call reaches a launch."""
    import ctypes as C
    from puffysics_amd import policy
    lib = policy.policy_lib()
    one = (C.c_char * 64)()
    at = C.addressof(one)
    g = policy.B3Attention(0, 1, 1, 8, 8, 0, None, None, None, (8, 8, 8), (8, 8, 8), (8, 8, 8), None, None, 0, (0, 0), None, 1.0)
    by = (C.c_int64 * 3)(8, 8, 8)

    def backward(d_v, d_state):
        return lib.b3_linear_attention_backward_gpu(C.byref(g), None, by, None, None, None, d_v, d_state, None, 0, None)

    assert lib.b3_linear_attention_gpu(C.byref(g), None, at, None, 0, None) == 1
    assert lib.b3_linear_attention_gpu(C.byref(g), None, None, None, 0, None) == 0
    assert backward(None, at) == 1 and backward(at, at) == 1
    assert backward(None, None) == 0 and backward(at, None) == 0
    g.steps, g.q, g.k, g.v = 1, at, at, at
    assert lib.b3_linear_attention_step_gpu(C.byref(g), at, at, None) == 1


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("key,value", [(128, 128), (100, 96), (70, 40), (128, 70), (64, 128)])
@pytest.mark.parametrize("steps,at", [(100, 45), (100, 32), (70, 69), (3000, 1500)])
def test_a_bad_column(steps, at, key, value, type, bad):
    """What is not finite in one column of v is in that column of out and of the
    state alone, from its step to the end of its episode: also where waves that
    share q and k have other columns, whichever of them finds it."""
    from puffysics_amd import policy
    q, k, v, _, _, state = made(steps, 2, 1, key, value, TYPES[type], 31)
    decay = torch.tensor([0.95], device="cuda")
    starts = torch.zeros(steps, 2, device="cuda")
    after = min(at + 5, steps - 1)
    starts[after, 0] = 1 if after > at else 0
    want = policy.linear_attention(q, k, v, decay, state=state, starts=starts, last=True)
    for col in (0, value // 2, value - 1):
        u = v.clone()
        u[at, :, 0, col] = bad
        got = policy.linear_attention(q, k, u, decay, state=state, starts=starts, last=True)
        seen = torch.zeros(v.shape, dtype=torch.bool, device="cuda")
        seen[at:, 1, 0, col] = True
        seen[at:after if after > at else steps, 0, 0, col] = True
        assert not torch.isfinite(got.out[seen]).any() and torch.isfinite(got.out[~seen]).all()
        clean = torch.where(seen, 0.0, got.out.float())
        close(clean.to(v.dtype), torch.where(seen, 0.0, want.out.float()).double(), 2.0 ** -7 * want.out.float().abs().max(), v.dtype)
        gone = torch.zeros(state.shape, dtype=torch.bool, device="cuda")
        gone[1, 0, :, col] = True
        gone[0, 0, :, col] = after == at
        assert not torch.isfinite(got.state[gone]).any() and torch.isfinite(got.state[~gone]).all()
        assert torch.allclose(got.state[~gone], want.state[~gone], rtol=1e-4, atol=1e-4)


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("size", [(70, 8, 2, 32, 32), (3000, 1, 1, 64, 64), (200, 2, 1, 128, 128)])
def test_gradient_replays(size, type):
    """A captured update, forwards and back, and a step of acting: every replay
    is the eager result of what the buffers hold then, the first one's too, with
    other work between."""
    from puffysics_amd import policy
    q, k, v, decay, starts, state = made(*size, TYPES[type], 14, rate=0.01)
    d = torch.randn_like(v)
    memory, twin = state.clone(), state.clone()

    def once(memory, *xs):
        leaves = [x.detach().requires_grad_() for x in xs]
        got = policy.linear_attention(*leaves[:3], decay, state=leaves[3], starts=starts, last=True)
        grads = torch.autograd.grad((got.out, got.state), leaves, (d, torch.ones_like(got.state)))
        step = policy.linear_attention_step(*(x[0] for x in xs[:3]), decay, memory, starts=starts[0])
        return [x.detach() for x in (got.out, got.state, *grads, step)]

    once(state.clone(), q, k, v, state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once(memory, q, k, v, state)
    for i in range(4):
        graph.replay()
        want = once(twin, *(x.clone() for x in (q, k, v, state)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(memory, twin), i
        q.mul_(0.5)
        v.add_(0.25)
        starts[i + 1] = ~starts[i + 1]
        torch.cuda.synchronize()
