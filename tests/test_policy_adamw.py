"""AdamW over many tensors (puffysics_amd.policy.AdamW) against the formulas
in 64 bits.

Tolerances, with u = 2^-24: a moment is two products and a sum of rounded
rates, 4 u of its terms; the update another ten operations, 16 u of itself
and 3 u of the weight; a weight in 16 bits half a unit of its type.  The norm
adds at most 64 squares one after the other in a thread and the rest pairwise:
100 u.  8-bit moments: the value of the grid below or above, by the random
bits that seed, step and place give; where these decide within 1e-5 of a step
of the grid, either."""
import numpy as np
import pytest
import torch

from policytest import adamw_oracle, grid_of, round_bits

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
U = 2.0 ** -24
LR, BETAS, EPS, DECAY = 0.01, (0.9, 0.999), 1e-8, 0.05
SIZES = [1, 3, 31, 32, 33, 255, 256, 257, 1000, 4095, 4096, 4097, 5001, 20000, 70003]


def tensors(sizes, type, seed, scale=1.0, offset=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n + offset, generator=g) * scale).to(TYPES[type]).cuda()[offset:] for n in sizes]


def f64(x):
    return x.detach().double().cpu().numpy()


class Moments32:
    def __init__(self, sizes):
        self.m, self.v = [np.zeros(n) for n in sizes], [np.zeros(n) for n in sizes]


def check_step(opt, params, grads, before, master_before, mom, type, decay, lr=LR, clip=1.0):
    """One step has been taken: weights and moments against the formulas on
    what was there before it."""
    avg, sq = opt.moments()
    for i, p in enumerate(params):
        if grads[i] is None:
            assert np.array_equal(f64(p), before[i])
            continue
        n, at = p.numel(), opt.offsets[i]
        w0 = before[i] if master_before is None else master_before[i]
        w, m, v = adamw_oracle(w0, f64(grads[i]), mom.m[i], mom.v[i], opt.steps(i), lr, *BETAS, EPS, decay, clip)
        gc = np.abs(f64(grads[i]) * clip)
        tm = (8 + 100 * (clip != 1)) * U * (BETAS[0] * np.abs(mom.m[i]) + (1 - BETAS[0]) * gc)
        tv = (8 + 200 * (clip != 1)) * U * v
        update = np.abs(w - w0 * (1 - lr * decay))
        root = np.sqrt(v / (1 - BETAS[1] ** opt.steps(i))) + EPS
        tw = 4 * U * np.abs(w0) + 24 * U * update + tm * lr / (1 - BETAS[0] ** opt.steps(i)) / root + 110 * U * update * (clip != 1)
        gm, gv = f64(avg[at:at + n]), f64(sq[at:at + n])
        assert (np.abs(gm - m) <= tm + 1e-44).all(), (i, np.abs(gm - m).max())
        assert (np.abs(gv - v) <= tv + 1e-44).all(), i
        if master_before is not None:
            kept = opt.master()[at:at + n]
            assert (np.abs(f64(kept) - w) <= tw).all(), i
            assert torch.equal(kept.to(p.dtype), p.detach().reshape(-1))
        else:
            assert (np.abs(f64(p) - w) <= tw + HALF_UNIT[type] * np.abs(w) * 1.01 + (2.0 ** -25 if type == "f16" else 0)).all(), i
        mom.m[i], mom.v[i] = gm, gv


def state_of(opt, params):
    master = opt.master()
    return [f64(p) for p in params], None if master is None else [
        f64(master[at:at + p.numel()]) for at, p in zip(opt.offsets, params)]


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1])
@pytest.mark.parametrize("master", [True, False])
@pytest.mark.parametrize("grad", ["own", "f32"])
@pytest.mark.parametrize("type", TYPES)
def test_steps(type, grad, master, offset):
    """Several steps, each against the formulas on the state before it;
    tensors that start anywhere their type may."""
    from puffysics_amd import policy
    params = tensors(SIZES, type, 1, offset=offset)
    opt = policy.AdamW(params, LR, BETAS, EPS, DECAY, master=master)
    mom = Moments32(SIZES)
    for t in range(1, 5):
        grads = tensors(SIZES, type if grad == "own" else "f32", 10 + t, 0.3, offset=offset)
        before, kept = state_of(opt, params)
        assert opt.step(grads) is None
        assert all(opt.steps(i) == t for i in range(len(params)))
        check_step(opt, params, grads, before, kept, mom, type, DECAY)
    if type == "f32" or not master:
        assert opt.master() is None
    opt.close()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """More tensors than one launch takes, empty ones and ones without a
    gradient among them, the norm over all that have one."""
    from puffysics_amd import policy
    sizes = [(i * 37) % 91 + (4096 if i % 50 == 0 else 0) for i in range(421)]
    params = tensors(sizes, "f32", 2)
    opt = policy.AdamW(params, LR, BETAS, EPS, [0.1 * (i % 3) for i in range(421)], state_bits=bits, max_grad_norm=1.0)
    grads = tensors(sizes, "f32", 3, 0.2)
    for i in range(0, 421, 7):
        grads[i] = None
    grads[160:320] = [None] * 160
    before, _ = state_of(opt, params)
    norm = opt.step(grads)
    want = np.sqrt(sum((f64(g) ** 2).sum() for g in grads if g is not None))
    assert abs(float(norm) - want) <= 100 * U * want
    clip = min(1.0, 1.0 / (want + 1e-6))
    for i, p in enumerate(params):
        assert opt.steps(i) == (grads[i] is not None)
        if grads[i] is None:
            assert np.array_equal(f64(p), before[i])
            continue
        w, m, v = adamw_oracle(before[i], f64(grads[i]), 0, 0, 1, LR, *BETAS, EPS, 0.1 * (i % 3), clip)
        # the first step's update is lr g / (|g| + eps / clip): nearly its sign
        assert (np.abs(f64(p) - w) <= 4 * U * np.abs(before[i]) + 300 * U * LR).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("most", [0.5, 1e9])
def test_clip(type, most):
    from puffysics_amd import policy
    params = tensors(SIZES, type, 4)
    opt = policy.AdamW(params, LR, BETAS, EPS, DECAY, max_grad_norm=most)
    mom = Moments32(SIZES)
    for t in range(3):
        grads = tensors(SIZES, type, 20 + t, 0.1)
        before, kept = state_of(opt, params)
        norm = float(opt.step(grads))
        want = np.sqrt(sum((f64(g) ** 2).sum() for g in grads))
        assert abs(norm - want) <= 100 * U * want
        check_step(opt, params, grads, before, kept, mom, type, DECAY, clip=min(1.0, most / (want + 1e-6)))


@pytest.mark.gpu
def test_zero_and_lost_gradients():
    from puffysics_amd import policy
    params = tensors([50, 300], "f32", 5)
    opt = policy.AdamW(params, LR, max_grad_norm=1.0, weight_decay=0.0)
    before = [p.clone() for p in params]
    assert float(opt.step([torch.zeros_like(p) for p in params])) == 0
    assert all(torch.equal(p, b) for p, b in zip(params, before))
    assert float(opt.step([None, None])) == 0
    g = [torch.ones_like(p) for p in params]
    g[0][3] = float("nan")
    assert np.isnan(float(opt.step(g)))
    assert all(torch.isnan(p).all() for p in params)           # a NaN norm is not passed over
    g[0][3] = float("inf")
    params = tensors([50, 300], "f32", 5)
    opt = policy.AdamW(params, LR, max_grad_norm=1.0, weight_decay=0.0)
    before = [p.clone() for p in params]
    assert float(opt.step(g)) == float("inf")                   # scales all that is finite to 0
    assert torch.isnan(params[0]).sum() == 1 and torch.equal(params[1], before[1])


def check_8_bits(opt, params, grads, before, old, seed):
    avg, sq = (f64(x) for x in opt.moments())
    t = opt.steps(0)
    for i, p in enumerate(params):
        at, n = opt.offsets[i], p.numel()
        padded = -(-n // 32) * 32
        g = np.zeros(padded)
        g[:n] = f64(grads[i])
        m0, v0 = old[0][at:at + padded], old[1][at:at + padded]
        m, v = BETAS[0] * m0 + (1 - BETAS[0]) * g, BETAS[1] * v0 + (1 - BETAS[1]) * g * g
        r = np.sqrt(v)
        um, ur = round_bits(padded, t, seed, at)
        for x, u, got, root in ((m, um, avg, False), (r, ur, sq, True)):
            got = got[at:at + padded]
            grid, least = grid_of(x)
            spread = 1e-5 + 16 * U * (BETAS[0] * np.abs(m0) + (1 - BETAS[0]) * np.abs(g)) / grid * (not root)
            lo, hi = (np.floor(np.abs(x) / grid + u + s * spread) * grid for s in (-1, 1))
            if root:
                lo, hi = (np.where(x > 0, np.maximum(y, least), y) ** 2 for y in (lo, hi))
            else:
                got = got * np.sign(x)
            # a group whose largest lies at the edge of two powers may go by either
            most = np.abs(x).reshape(-1, 32).max(1)
            edge = np.abs(np.log2(np.maximum(most, 1e-30) / 448.0) - np.round(np.log2(np.maximum(most, 1e-30) / 448.0))) < 1e-5
            ok = (got == lo) | (got == hi) | np.repeat(edge, 32)
            # exactly zero first moments carry no sign
            assert ok.all(), (i, root, np.flatnonzero(~ok)[:4], got[~ok][:4], lo[~ok][:4], hi[~ok][:4])
        w, *_ = adamw_oracle(before[i], g[:n], m0[:n], v0[:n], t, LR, *BETAS, EPS, DECAY)
        update = np.abs(w - before[i] * (1 - LR * DECAY))
        tm = 8 * U * (BETAS[0] * np.abs(m0) + (1 - BETAS[0]) * np.abs(g))[:n] * LR / (1 - BETAS[0] ** t) / (
            r[:n] / np.sqrt(1 - BETAS[1] ** t) + EPS)
        assert (np.abs(f64(p) - w) <= 4 * U * np.abs(before[i]) + 24 * U * update + tm).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, 1e-6, 1e5])
def test_8_bit_steps(scale):
    from puffysics_amd import policy
    params = tensors(SIZES, "f32", 6)
    opt = policy.AdamW(params, LR, BETAS, EPS, DECAY, state_bits=8, seed=12345)
    for t in range(6):
        grads = [g * torch.exp(3 * torch.randn_like(g)) for g in tensors(SIZES, "f32", 30 + t, scale)]
        old = [f64(x) for x in opt.moments()]
        before = [f64(p) for p in params]
        opt.step(grads)
        check_8_bits(opt, params, grads, before, old, 12345)


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["bf16", "f16"])
def test_8_bit_moments_of_16_bit_weights(type):
    """The same moments and 32-bit copies as 32-bit weights have on the same
    gradients."""
    from puffysics_amd import policy
    params = tensors(SIZES, type, 7)
    twins = [p.float() for p in params]
    a = policy.AdamW(params, LR, BETAS, EPS, DECAY, state_bits=8, seed=3)
    b = policy.AdamW(twins, LR, BETAS, EPS, DECAY, state_bits=8, seed=3)
    for t in range(3):
        grads = tensors(SIZES, type, 40 + t)
        a.step(grads)
        b.step([g.float() for g in grads])
    assert all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))
    for at, p, q in zip(a.offsets, params, twins):
        assert torch.equal(a.master()[at:at + p.numel()], q) and torch.equal(p, q.to(p.dtype))


@pytest.mark.gpu
def test_8_bit_second_moments_follow_small_changes():
    """From zero under a steady gradient, a thousandth a step: each step
    rounds the root up or down by at most an eighth of it, with the chance
    (at most 0.008) of the change, so the mean square is over the true second
    moment by at most 0.008 / 64 of it for each of the thousand steps that it
    remembers: 12.5%."""
    from puffysics_amd import policy
    p = torch.zeros(32768, device="cuda")
    opt = policy.AdamW([p], 0.0, BETAS, EPS, 0.0, state_bits=8)
    g = torch.full_like(p, 0.02)
    for t in range(2000):
        opt.step([g])
    m, v = opt.moments()
    want = 0.02 ** 2 * (1 - BETAS[1] ** 2000)
    assert 0.99 * want < float(v.float().mean()) < 1.13 * want
    # the first moment: a step of the grid is a twelfth of it on the average,
    # and 32768 places average the last ten steps' roundings to 0.1%
    assert abs(float(m.float().mean()) - 0.02) < 0.005 * 0.02


@pytest.mark.gpu
def test_8_bit_extremes():
    """Groups of zeros, of tiny and huge values, of one large value beside
    small ones, and lost gradients."""
    from puffysics_amd import policy
    n = 32 * 8
    g = torch.zeros(n)
    g[32:64] = 1e-30
    g[64:96] = 1e18
    g[96:128] = torch.logspace(-12, 0, 32)
    g[130], g[161], g[163] = float("nan"), float("inf"), 2.0
    g[192:224] = -0.0
    p = torch.zeros(n, device="cuda")
    opt = policy.AdamW([p], LR, BETAS, EPS, 0.0, state_bits=8, seed=9)
    opt.step([g.cuda()])
    m, v = (x.float().cpu() for x in opt.moments())
    lost = torch.zeros(n, dtype=torch.bool)
    lost[130] = lost[161] = True
    assert torch.equal(torch.isnan(m), lost) and torch.equal(torch.isnan(v), lost)
    assert (m[:32] == 0).all() and (v[:32] == 0).all() and (m[192:224] == 0).all()
    # a root over 0 stays over 0, unless its square is under the least of bf16
    assert (v[96:128] > 0).all()
    rel = lambda x, want: float(((x - want).abs() / want).max())  # noqa: E731
    assert rel(m[64:96], torch.tensor(1e17)) < 0.13 and rel(v[64:96].sqrt(), torch.tensor(0.001 ** 0.5 * 1e18)) < 0.13
    assert rel(m[163], torch.tensor(0.2)) < 0.13
    assert torch.isfinite(p.cpu()[~lost]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_moments_go_in_and_out(bits):
    """What moments() gives, load_moments() restores, to the bit: a run that
    is taken up again goes on as it would have."""
    from puffysics_amd import policy
    def views(opt, flat):
        return [flat[at:at + p.numel()].float() for at, p in zip(opt.offsets, opt.params)]
    sizes = [5, 300, 4097, 64]
    params = tensors(sizes, "bf16", 8)
    a = policy.AdamW(params, LR, state_bits=bits, seed=5)
    for t in range(3):
        a.step(tensors(sizes, "bf16", 50 + t))
    twins = [p.clone() for p in params]
    b = policy.AdamW(twins, LR, state_bits=bits, seed=5)
    m, v = a.moments()
    b.load_moments(views(a, m), views(a, v), 3, master=views(a, a.master()))
    assert all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))
    g = tensors(sizes, "bf16", 60)
    a.step(g)
    b.step(g)
    assert a.steps() == b.steps() == 4
    assert all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))
    assert all(torch.equal(x, y) for x, y in zip(params, twins))
    assert torch.equal(a.master(), b.master())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_same_results_every_time_and_on_another_stream(bits):
    from puffysics_amd import policy
    sizes = [70000, 3, 4096, 1000]
    runs = []
    for k in range(2):
        s = torch.cuda.current_stream() if k == 0 else torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            params = tensors(sizes, "f32", 9)
            opt = policy.AdamW(params, LR, state_bits=bits, max_grad_norm=0.5)
            for t in range(3):
                norm = opt.step(tensors(sizes, "f32", 70 + t))
        torch.cuda.current_stream().wait_stream(s)
        runs.append((*params, *opt.moments(), norm))
    assert all(torch.equal(x, y) for x, y in zip(*runs))


@pytest.mark.gpu
def test_captured():
    """A captured step repeats the corrections of the step that was captured,
    on whatever the gradients hold."""
    from puffysics_amd import policy
    params, grads = tensors([5000, 7], "f32", 10), tensors([5000, 7], "f32", 11)
    opt = policy.AdamW(params, LR, BETAS, EPS, DECAY, max_grad_norm=0.5)
    opt.step(grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = opt.step(grads)
    mom = Moments32([5000, 7])
    avg, sq = opt.moments()
    for i, at in enumerate(opt.offsets):
        mom.m[i], mom.v[i] = f64(avg[at:at + params[i].numel()]), f64(sq[at:at + params[i].numel()])
    for k in range(3):
        for g in grads:
            g.copy_(torch.randn_like(g))
        before, _ = state_of(opt, params)
        graph.replay()
        torch.cuda.synchronize()
        want = np.sqrt(sum((f64(g) ** 2).sum() for g in grads))
        assert abs(float(norm) - want) <= 100 * U * want
        check_step(opt, params, grads, before, None, mom, "f32", DECAY, clip=0.5 / (want + 1e-6))


@pytest.mark.gpu
def test_parameters_own_gradients():
    from puffysics_amd import policy
    layer = torch.nn.Linear(40, 30).cuda()
    twin = [p.detach().clone() for p in layer.parameters()]
    opt, same = policy.AdamW(layer.parameters(), LR), policy.AdamW(twin, LR)
    layer(torch.randn(5, 40, device="cuda")).square().sum().backward()
    opt.step()
    same.step([p.grad for p in layer.parameters()])
    assert all(torch.equal(p.detach(), q) for p, q in zip(layer.parameters(), twin))
    none = policy.AdamW([], LR, max_grad_norm=1.0)
    assert float(none.step([])) == 0 and none.size == 0


@pytest.mark.gpu
def test_refusals_of_gradients():
    from puffysics_amd import policy
    p = [torch.zeros(4, 6, device="cuda", dtype=torch.bfloat16)]
    opt = policy.AdamW(p, LR)
    for g in (torch.zeros(4, 5), torch.zeros(6, 4).t(), torch.zeros(4, 6).half(), torch.zeros(4, 6).double()):
        with pytest.raises(ValueError):
            opt.step([g.cuda()])
    for g in ([], [torch.zeros(4, 6)], [None, None]):
        with pytest.raises(ValueError):
            opt.step(g)
    assert opt.steps() == 0
    for bad in (dict(exp_avg=[], exp_avg_sq=[], step=1), dict(exp_avg=p, exp_avg_sq=p, step=-1),
                dict(exp_avg=[p[0][0]], exp_avg_sq=p, step=1)):
        with pytest.raises(ValueError):
            opt.load_moments(**bad)
    with pytest.raises(ValueError):
        policy.AdamW(p + p, LR)
    for bad in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(state_bits=4), dict(weight_decay=[0.1, 0.2]),
                dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            policy.AdamW(p, LR, **bad)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [8, 32])
def test_refused_moments_leave_the_state(bits):
    from puffysics_amd import policy
    p = [torch.zeros(40, device="cuda"), torch.zeros(7, device="cuda", dtype=torch.bfloat16)]
    opt = policy.AdamW(p, LR, state_bits=bits)
    good, bad = [torch.ones(40), torch.ones(7)], [torch.ones(40), torch.ones(8)]
    for args in ((bad, good, 3), (good, bad, 3), (good, good, 3, bad)):
        with pytest.raises(ValueError):
            opt.load_moments(*args)
    assert all(int(torch.count_nonzero(x)) == 0 for x in (*opt.moments(), opt.master())) and opt.steps() == 0


@pytest.mark.gpu
def test_a_clip_of_0_is_refused():
    """Also where it is set later: it would have meant no clip at all."""
    from puffysics_amd import policy
    p = torch.zeros(5, device="cuda")
    for most in (0.0, 0, -1.0, float("nan")):
        with pytest.raises(ValueError):
            policy.AdamW([p], LR, max_grad_norm=most)
        opt = policy.AdamW([p], LR, max_grad_norm=1.0)
        opt.max_grad_norm = most
        with pytest.raises(ValueError):
            opt.step([torch.ones(5, device="cuda")])
        assert opt.steps() == 0 and int(torch.count_nonzero(p)) == 0


@pytest.mark.gpu
def test_a_step_is_an_operation_in_place():
    """Autograd notices weights that were stepped between a forward pass and
    its backward; a parameter whose memory went elsewhere is refused."""
    from puffysics_amd import policy
    w = torch.randn(5, device="cuda", requires_grad=True)
    opt = policy.AdamW([w], LR)
    y = (w * w).sum()
    opt.step([torch.ones(5, device="cuda")])
    with pytest.raises(RuntimeError):
        y.backward()
    w.data = torch.randn(5, device="cuda")
    with pytest.raises(ValueError):
        opt.step([torch.ones(5, device="cuda")])


@pytest.mark.gpu
def test_places_past_32_bits():
    """The weights at the far end of more than 2^32."""
    from puffysics_amd import policy
    n = 2 ** 32 + 70_001
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-5:] = torch.tensor([1.0, -1.0, 0.5, 2.0, -3.0])
    g[2 ** 32] = 4.0
    opt = policy.AdamW([p], LR, weight_decay=0.0, state_bits=8, master=False, max_grad_norm=100.0)
    assert abs(float(opt.step([g])) - (1 + 1 + 0.25 + 4 + 9 + 16) ** 0.5) < 1e-5
    assert torch.equal(p[-5:].float().sign(), -g[-5:].float().sign()) and float(p[2 ** 32]) < 0
    assert int(torch.count_nonzero(p[-100_000:])) == 6 and int(torch.count_nonzero(p[:100_000])) == 0
    m, v = opt.moments()
    assert (m[2 ** 32:n][g[2 ** 32:] == 0] == 0).all() and abs(float(m[n - 1]) + 0.3) < 0.3 / 8
    assert abs(float(v[2 ** 32]) - 0.016) < 0.016 / 3


def test_refusals():
    from puffysics_amd import policy
    for p in (torch.zeros(3, dtype=torch.float64), torch.zeros(4, 6).t(), torch.zeros(4, dtype=torch.int64), torch.zeros(3)):
        with pytest.raises(ValueError):
            policy.AdamW([p], LR)


def test_refusals_of_the_c_entry():
    from puffysics_amd import policy
    C, lib = policy.C, policy.policy_lib()
    T, h = policy.B3AdamWTensor, C.c_void_p()
    one = (T * 1)(T(64, 0, 10, 0.0))
    state, config = policy.B3AdamWState(32, 64, 64, None, None, None), policy.B3AdamWConfig(0.9, 0.999, 1e-8, 0)
    assert lib.b3_adamw_size(one, 1) == 256 and lib.b3_adamw_size(one, 0) == 0 and lib.b3_adamw_size(None, 1) == -1
    bad_tensors = [T(None, 0, 10, 0.0), T(64, 3, 10, 0.0), T(64, 0, -1, 0.0), T(64, 0, 10, -1.0), T(64, 0, 2 ** 41, 0.0)]
    for t in bad_tensors:
        assert lib.b3_adamw_create(C.byref(h), (T * 1)(t), 1, state, config) == 1 and not h.value
        assert lib.b3_adamw_size((T * 1)(t), 1) == -1
    for s in (policy.B3AdamWState(16, 64, 64, None, None, None), policy.B3AdamWState(32, None, 64, None, None, None),
              policy.B3AdamWState(8, 64, 64, None, 64, None)):
        assert lib.b3_adamw_create(C.byref(h), one, 1, s, config) == 1
    for c in ((1.0, 0.9, 0.0), (0.9, -0.1, 0.0), (0.9, 0.9, -1.0), (float("nan"), 0.9, 0.0)):
        assert lib.b3_adamw_create(C.byref(h), one, 1, state, policy.B3AdamWConfig(*c, 0)) == 1
    assert lib.b3_adamw_create(None, one, 1, state, config) == 1
    assert lib.b3_adamw_step_gpu(None, None, None, 0.1, 0.0, None, None) == 1
    assert lib.b3_adamw_steps(None, 0) == -1 and lib.b3_adamw_set_steps(None, 0, 1) == 1
    assert lib.b3_adamw_moments_gpu(None, 64, 64, None) == 1 and lib.b3_adamw_load_moments_gpu(None, 64, 64, None) == 1
    assert lib.b3_adamw_destroy(None) == 0


def test_every_declared_symbol_is_exported():
    import re
    from b3test import ROOT
    from puffysics_amd import policy
    text = open(ROOT + "/include/b3_policy.h").read()
    names = set(re.findall(r"^(?:hipError_t|int64_t|size_t) (\w+)\(", text, re.M))
    assert names == {n for n, _, _ in policy.POLICY_SYMBOLS}
    assert all(hasattr(policy.policy_lib(), n) for n in names)
    assert int(re.search(r"B3_ADAMW_SEGMENT (\d+)", text).group(1)) == policy.SEGMENT
    assert int(re.search(r"B3_MAX_TOP (\d+)", text).group(1)) == policy.MAX_TOP


def test_grid_of_the_oracle():
    """Every e4m3 number is on the grid of its group, and 16 random bits of
    one in 2^16 have their mean."""
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    x = np.concatenate([codes, [448.0]]).reshape(4, 32)
    x[:, -1] = 448.0
    grid, least = grid_of(x)
    assert (x.reshape(-1) / grid % 1 == 0).all() and (least == 2.0 ** -9).all()
    a, b = round_bits(1 << 16, 7, 3)
    assert abs(a.mean() - 0.5) < 0.01 and abs(b.mean() - 0.5) < 0.01 and abs(np.corrcoef(a, b)[0, 1]) < 0.02
