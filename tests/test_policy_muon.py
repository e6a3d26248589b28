"""puffysics_amd.policy.Muon against the definition in 64 bits."""
import math

import pytest
import torch

from memorytest import STEP, orthogonalised_oracle

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [(1, 1), (3, 64), (64, 3), (64, 64), (4, 64), (1, 200), (33, 65), (128, 128), (100, 129), (130, 300), (300, 130),
          (257, 256), (512, 37), (17, 1000), (384, 640)]
LR, MU, DECAY = 0.05, 0.9, 0.1


def tensors(shapes, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(*s, generator=g) * scale).to(dtype).cuda() for s in shapes]


def views(opt, flat):
    return [flat[at:at + p.numel()].view(p.shape) for at, p in zip(opt.offsets, opt.params)]


def exactness(shape, steps=5):
    """How far x may be off, in its 2-norm, relative to 1 (the size of its
    singular values): x is off by some 2^-22 of its norm after each of the
    products' roundings (sums of up to the longer side of products exact to
    2^-22, in 32 bits), and the steps may carry on what is there by at most
    3.4445 each."""
    return 2.0 ** -22 * math.sqrt(max(shape)) * sum(3.4445 ** i for i in range(steps + 1))


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("type", TYPES)
def test_steps(type, nesterov):
    """Some steps over matrices of all shapes, 16-bit ones with and without
    copies; gradients of the matrices' type or in 32 bits, some left out."""
    from puffysics_amd import policy
    dtype = TYPES[type]
    for master in ((True, False) if dtype != torch.float32 else (True,)):
        params = tensors(SHAPES, dtype, 1, 0.1)
        opt = policy.Muon(params, LR, MU, weight_decay=DECAY, nesterov=nesterov, master=master)
        assert (opt.master() is None) == (dtype == torch.float32 or not master)
        w, m = [p.double() for p in params], [torch.zeros_like(p, dtype=torch.float64) for p in params]
        off, before = [0.0] * len(params), [p.clone() for p in params]
        for t in range(3):
            grads = tensors(SHAPES, dtype if t != 1 else torch.float32, 10 + t)
            grads = [None if t == 2 and i % 3 == 0 else g for i, g in enumerate(grads)]
            opt.step(grads)
            for i, g in enumerate(grads):
                if g is None:
                    continue
                m[i] = MU * m[i] + g.double()
                x = orthogonalised_oracle(g.double() + MU * m[i] if nesterov else m[i])
                rate = LR * math.sqrt(max(1.0, g.shape[0] / g.shape[1]))
                if dtype != torch.float32 and not master:
                    w[i] = before[i].double()
                    off[i] = 0.0
                w[i] = w[i] * (1 - LR * DECAY) - rate * x
                off[i] += rate * exactness(g.shape)
                got = params[i].double() if dtype == torch.float32 or not master else views(opt, opt.master())[i].double()
                most = float(w[i].abs().max())
                step = 2.0 ** -22 if dtype == torch.float32 or master else STEP[dtype] * 1.01
                far = (got - w[i]).norm() / math.sqrt(g.numel())
                assert float(far) <= off[i] + 4 * step * most, (g.shape, t)
                if dtype != torch.float32 and master:
                    assert torch.equal(params[i], views(opt, opt.master())[i].to(dtype))
                close = (views(opt, opt.momentum())[i].double() - m[i]).abs() <= 2.0 ** -22 * (m[i].abs() + 3)
                assert close.all()
            before = [p.clone() for p in params]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("kind", ["even", "low rank", "spike", "graded", "tiny", "huge"])
def test_orthogonalised(shape, kind):
    """x itself: the weights begin at 0, with a rate of 1 over the factor of
    tall matrices."""
    from puffysics_amd import policy
    g = torch.Generator().manual_seed(sum(shape))
    u = torch.randn(*shape, generator=g, dtype=torch.float64)
    if kind == "low rank":
        u = torch.randn(shape[0], 2, generator=g, dtype=torch.float64) @ torch.randn(2, shape[1], generator=g, dtype=torch.float64)
    elif kind == "spike":
        u = u * 1e-3
        u[0, 0] = 100.0
    elif kind == "graded":
        u = u * torch.logspace(0, -6, shape[0], dtype=torch.float64)[:, None]
    elif kind == "tiny":
        u = u * 1e-12
    elif kind == "huge":
        u = u * 1e15
    u = u.float().cuda()
    param = torch.zeros(shape, device="cuda")
    eps = 1e-7 if kind != "tiny" else 1e-20
    opt = policy.Muon([param], math.sqrt(min(1.0, shape[1] / shape[0])), momentum=0.0, eps=eps)
    opt.step([u])
    want = -orthogonalised_oracle(u, eps=eps)
    # 2-norm of the difference: all its singular values together
    assert float((param.double() - want).norm()) <= exactness(shape) * math.sqrt(min(shape)) * 2, kind
    assert torch.isfinite(param).all()


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 5, 6, 9, 16])
@pytest.mark.parametrize("shape", [(60, 90), (140, 200), (130, 300), (700, 129)])
def test_counts_of_newton_schulz(shape, steps):
    from puffysics_amd import policy
    u, = tensors([shape], torch.float32, 4)
    param = torch.zeros(shape, device="cuda")
    policy.Muon([param], math.sqrt(min(1.0, shape[1] / shape[0])), momentum=0.0, newton_schulz=steps).step([u])
    want = -orthogonalised_oracle(u, steps)
    # beyond 5 steps singular values are near 1, where a step's slope is between -1.6 and 2.5: what the first leave
    # grows by far less than their 3.4445 at each
    assert float((param.double() - want).norm()) <= exactness(shape, min(steps, 7)) * math.sqrt(min(shape)) * 2


@pytest.mark.gpu
def test_zero_and_bad_gradients():
    """A gradient of zeros moves nothing but the decay; NaN stay in their matrix."""
    from puffysics_amd import policy
    params = tensors([(40, 30), (40, 30), (200, 150), (200, 150)], torch.float32, 1)
    before = [p.clone() for p in params]
    opt = policy.Muon(params, LR, weight_decay=DECAY)
    grads = [torch.zeros_like(p) for p in params]
    grads[1][3, 4] = grads[3][7, 7] = float("nan")
    opt.step(grads)
    keep = torch.tensor(1 - LR * DECAY, dtype=torch.float64).float()
    for i in (0, 2):
        assert torch.equal(params[i], before[i] * keep.cuda())
    for i in (1, 3):
        assert params[i].isnan().all()


@pytest.mark.gpu
def test_groups_are_their_matrices():
    """A step over many matrices is each one's own step, bit for bit."""
    from puffysics_amd import policy
    shapes = SHAPES + [(64, 3)] * 200 + [(0, 5), (5, 0)]
    grads = tensors(shapes, torch.float32, 2)
    params, twins = tensors(shapes, torch.float32, 3), tensors(shapes, torch.float32, 3)
    policy.Muon(params, LR).step(grads)
    for i in list(range(len(SHAPES) + 3)) + [len(shapes) - 3, len(shapes) - 1]:
        policy.Muon([twins[i]], LR).step([grads[i]])
        assert torch.equal(params[i], twins[i]), shapes[i]


@pytest.mark.gpu
def test_written_weights_and_resumed_momentum():
    from puffysics_amd import policy
    shapes = [(20, 30), (200, 140)]
    params = tensors(shapes, torch.bfloat16, 1)
    opt = policy.Muon(params, LR)
    opt.step(tensors(shapes, torch.bfloat16, 2))
    twins = [p.clone() for p in params]
    twin = policy.Muon(twins, LR)
    twin.load_momentum(views(opt, opt.momentum()), master=views(opt, opt.master()))
    with torch.no_grad():
        params[1].add_(1.0)
        twins[1].copy_(params[1])
        views(twin, twin.master())[1].copy_(params[1])
    grads = tensors(shapes, torch.bfloat16, 3)
    opt.step(grads)
    twin.step(grads)
    assert all(torch.equal(a, b) for a, b in zip(params, twins))
    assert torch.equal(opt.master()[:600], twin.master()[:600])
    for p in params:
        p.requires_grad_()
        p.grad = torch.ones_like(p)
    version = params[0]._version
    opt.step()
    assert params[0]._version > version
    opt.close()
    opt.close()


@pytest.mark.gpu
def test_replays():
    """A captured step, replayed with other gradients and other work between,
    is the eager step."""
    from puffysics_amd import policy
    shapes = [(64, 64), (3, 64), (150, 200), (260, 128)]
    params, twins = tensors(shapes, torch.float32, 1), tensors(shapes, torch.float32, 1)
    opt, twin = policy.Muon(params, LR), policy.Muon(twins, LR)
    grads = tensors(shapes, torch.float32, 2)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(grads)
    for i in range(4):
        for g in grads:
            g.copy_(torch.randn(g.shape, generator=torch.Generator().manual_seed(i)).cuda())
        graph.replay()
        twin.step(grads)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(params, twins)), i
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_on_another_stream():
    from puffysics_amd import policy
    shapes = [(64, 64), (150, 200)]
    params, twins = tensors(shapes, torch.float32, 1), tensors(shapes, torch.float32, 1)
    grads = tensors(shapes, torch.float32, 2)
    opt, twin = policy.Muon(params, LR), policy.Muon(twins, LR)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        opt.step(grads)
    side.synchronize()
    twin.step(grads)
    assert all(torch.equal(a, b) for a, b in zip(params, twins))


def test_refusals():
    """Nothing is launched: this runs without a GPU."""
    from puffysics_amd import policy
    p = torch.zeros(3, 4)
    for what, args in (("contiguous", ([p.t()],)), ("float32, float16", ([p.double()],)), ("twice", ([p, p[1:]],))):
        with pytest.raises(ValueError, match=what):
            policy.Muon(*args)
    with pytest.raises(ValueError, match="CUDA device"):
        policy.Muon([p])
    for args in (dict(momentum=1.0), dict(momentum=-0.1), dict(eps=0.0), dict(newton_schulz=0), dict(newton_schulz=17),
                 dict(lr=-1.0), dict(lr=float("nan")), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            policy.Muon([], **args) if "weight_decay" not in args else policy.Muon([p], **args)


@pytest.mark.gpu
def test_refusals_of_a_step():
    from puffysics_amd import policy
    params = tensors([(3, 4), (5, 6)], torch.bfloat16, 1)
    before = [p.clone() for p in params]
    with pytest.raises(ValueError, match="matrices"):
        policy.Muon([torch.zeros(4, device="cuda")])
    opt = policy.Muon(params, LR)
    good = tensors([(3, 4), (5, 6)], torch.bfloat16, 2)
    for grads in (good[:1], [good[0], good[1].t()], [good[0].half(), good[1]], [good[0].cpu(), good[1]], [good[1], good[0]]):
        with pytest.raises(ValueError):
            opt.step(grads)
    with pytest.raises(ValueError):
        opt.step(good, lr=-1.0)
    with pytest.raises(ValueError):
        opt.load_momentum([good[0]])
    assert all(torch.equal(a, b) for a, b in zip(params, before)) and int(torch.count_nonzero(opt.momentum())) == 0
    policy.Muon([]).step([])


def in_32_bits(u, steps=5, eps=1e-7):
    """Muon's steps with torch's 32-bit products."""
    x = u.float()
    turned = x.shape[0] > x.shape[1]
    x = x.t() if turned else x
    x = x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        y = x @ x.t()
        x = 3.4445 * x + (-4.7750 * y + 2.0315 * (y @ y)) @ x
    return x.t() if turned else x


def far(x, want):
    return float((x.double() - want).norm())


def near_32_bits(u, want, steps=5):
    """What x may be off by, in the norm of all elements.  A number is kept to
    2^-22, a quarter as exactly as in 32 bits, of both sides of a product, and
    matrices that take their steps on the short side have twice as many
    products: 16 times what the steps in 32 bits are off by; or, where that
    happens to be little, as of few or simple numbers, a step of each number's
    for all that is formed in five steps, three products and z."""
    return 16 * far(in_32_bits(u, steps), want) + 4 * max(steps, 5) * 2.0 ** -22 * float(want.norm())


WIDE = [(1100, 1100), (1100, 1600), (1600, 1100), (130, 1500), (600, 1030), (256, 1024)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES + WIDE, ids=lambda s: "%dx%d" % s)
@pytest.mark.parametrize("kind", ["even", "low rank", "spike", "graded", "strong and weak"])
def test_as_exact_as_32_bits(shape, kind):
    """Next to the same steps with torch's 32-bit products, by the norm of the
    difference; sides of more than a square of tiles among them."""
    from puffysics_amd import policy
    g = torch.Generator().manual_seed(sum(shape))
    u = torch.randn(*shape, generator=g, dtype=torch.float64)
    two = torch.randn(shape[0], 2, generator=g, dtype=torch.float64) @ torch.randn(2, shape[1], generator=g, dtype=torch.float64)
    if kind == "low rank":
        u = two
    elif kind == "strong and weak":
        u = two + 1e-4 * u
    elif kind == "spike":
        u = u * 1e-3
        u[0, 0] = 100.0
    elif kind == "graded":
        u = u * torch.logspace(0, -6, shape[0], dtype=torch.float64)[:, None]
    u = u.float().cuda()
    param = torch.zeros(shape, device="cuda")
    policy.Muon([param], math.sqrt(min(1.0, shape[1] / shape[0])), momentum=0.0).step([u])
    want = -orthogonalised_oracle(u)
    assert far(param, want) <= near_32_bits(-u, want), (far(param, want), near_32_bits(-u, want), float(want.norm()))


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 4, 5, 6, 7, 11, 16])
@pytest.mark.parametrize("shape", [(60, 90), (130, 200), (250, 1000), (700, 129)])
def test_as_exact_after_any_steps(shape, steps):
    from puffysics_amd import policy
    g = torch.Generator().manual_seed(steps)
    u = (torch.randn(shape[0], 3, generator=g) @ torch.randn(3, shape[1], generator=g)).cuda()
    param = torch.zeros(shape, device="cuda")
    policy.Muon([param], math.sqrt(min(1.0, shape[1] / shape[0])), momentum=0.0, newton_schulz=steps).step([u])
    want = -orthogonalised_oracle(u, steps)
    assert far(param, want) <= near_32_bits(-u, want, steps)


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_weights_move_as_exactly(type):
    """Three steps with momentum over matrices of many shapes at once."""
    from puffysics_amd import policy
    dtype, shapes = TYPES[type], SHAPES + WIDE
    params = tensors(shapes, dtype, 1, 0.1)
    opt = policy.Muon(params, LR, MU, weight_decay=DECAY)
    w, m = [p.double() for p in params], [torch.zeros_like(p, dtype=torch.float64) for p in params]
    off = [0.0] * len(params)
    for t in range(3):
        grads = tensors(shapes, dtype, 20 + t)
        opt.step(grads)
        for i, g in enumerate(grads):
            m[i] = MU * m[i] + g.double()
            u = g.double() + MU * m[i]
            x = orthogonalised_oracle(u)
            rate = LR * math.sqrt(max(1.0, g.shape[0] / g.shape[1]))
            w[i] = w[i] * (1 - LR * DECAY) - rate * x
            # u is of 32 bits too: half a step, which the steps carry on as that of in_32_bits
            off[i] += rate * near_32_bits(u, x) + 2.0 ** -22 * float(w[i].norm())
            got = params[i] if dtype == torch.float32 else views(opt, opt.master())[i]
            assert far(got, w[i]) <= off[i], (g.shape, t)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [3, 5, 6, 8])
@pytest.mark.parametrize("shape", [(5, 510), (510, 5), (17, 1000), (60, 510), (100, 1000), (128, 700), (200, 1000), (513, 2048)])
@pytest.mark.parametrize("kind", ["all rows", "five rows"])
def test_as_exact_of_weak_directions(shape, kind, steps):
    """Two strong directions over others of a tenth, in all rows or in a few."""
    from puffysics_amd import policy
    g = torch.Generator().manual_seed(shape[0] + steps)
    some = lambda r: torch.randn(r, 2, generator=g) @ torch.randn(2, shape[1], generator=g) + 0.1 * torch.randn(r, shape[1], generator=g)  # noqa: E731
    u = some(shape[0])
    if kind == "five rows":
        u = 1e-2 * torch.randn(shape, generator=g)
        u[:5] = some(min(5, shape[0]))
    u = u.cuda()
    param = torch.zeros(shape, device="cuda")
    policy.Muon([param], math.sqrt(min(1.0, shape[1] / shape[0])), momentum=0.0, newton_schulz=steps).step([u])
    want = -orthogonalised_oracle(u, steps)
    assert far(param, want) <= near_32_bits(-u, want, steps)
