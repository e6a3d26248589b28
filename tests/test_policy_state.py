"""What puffysics_amd.policy.AdamW keeps between steps: 32-bit copies of
16-bit weights, moments, counts of steps."""
import numpy as np
import pytest
import torch

LR, BETAS, EPS, DECAY = 0.01, (0.9, 0.999), 1e-8, 0.05
SIZES = [1, 3, 31, 33, 256, 257, 4095, 4097, 20000]
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def tensors(sizes, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale).to(dtype).cuda() for n in sizes]


def views(opt, flat):
    return [flat[at:at + p.numel()].float().view(p.shape) for at, p in zip(opt.offsets, opt.params)]


def resumed(opt, params, bits, **how):
    """An optimizer made of `params` that goes on from opt's moments."""
    from puffysics_amd import policy
    got = policy.AdamW(params, LR, BETAS, EPS, DECAY, state_bits=bits, seed=4)
    m, v = opt.moments()
    got.load_moments(views(opt, m), views(opt, v), opt.steps(), **how)
    return got


def equal(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def write_copy(p, x):
    with torch.no_grad():
        p.copy_(x)


def write_data(p, x):
    p.data.copy_(x)


def write_state(p, x):
    holder = torch.nn.Module()
    holder.weight = p if isinstance(p, torch.nn.Parameter) else torch.nn.Parameter(p)
    holder.load_state_dict({"weight": x})


@pytest.mark.gpu
@pytest.mark.parametrize("write", [write_copy, write_data, write_state])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("type", TYPES)
def test_written_weights_count(type, bits, write):
    """16-bit weights that are loaded after the optimizer was made are what
    the next step goes on from, as if it had been made of them; the weights
    beside them keep their 32-bit copies."""
    from puffysics_amd import policy
    dtype = TYPES[type]
    params = [torch.nn.Parameter(p) for p in tensors(SIZES, dtype, 1)]
    opt = policy.AdamW(params, LR, BETAS, EPS, DECAY, state_bits=bits, seed=4)
    for t in range(3):
        opt.step(tensors(SIZES, dtype, 10 + t))
    new = [p.detach() + 4 if i % 2 else None for i, p in enumerate(params)]
    twins = [p.detach().clone() if x is None else x.clone() for p, x in zip(params, new)]
    twin = resumed(opt, twins, bits, master=[m if x is None else x.float() for m, x in zip(views(opt, opt.master()), new)])
    for p, x in zip(params, new):
        if x is not None:
            write(p, x)
    for t in range(2):
        grads = tensors(SIZES, dtype, 20 + t)
        opt.step(grads)
        twin.step(grads)
        assert equal([p.detach() for p in params], twins)
        assert equal(views(opt, opt.master()), views(twin, twin.master()))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_written_weights_count_in_replays(bits):
    """Also between the replays of a captured step, and weight by weight."""
    from puffysics_amd import policy
    p, = tensors([5000], torch.bfloat16, 2)
    g = torch.zeros_like(p)
    opt = policy.AdamW([p], LR, BETAS, EPS, 0.0, state_bits=bits)
    opt.step([g])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step([g])
    for k in range(3):
        p[k::7] = 3.0 + k                        # gradients and moments of 0: nothing else moves
        want = p.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(p, want) and torch.equal(opt.master()[:5000], want.float())


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
def test_copies_of_every_weight_are_kept(type):
    """Every 16-bit number, denormals and infinities among them, keeps a copy
    that differs from it by less than the rounding."""
    from puffysics_amd import policy
    bits = torch.arange(-2 ** 15, 2 ** 15, dtype=torch.int32).to(torch.int16)
    w = bits.view(TYPES[type])
    w = w[~torch.isnan(w)].cuda()
    copies = w.float() * (1 + 2.0 ** -13)
    assert torch.equal(copies.to(w.dtype).view(torch.int16), w.view(torch.int16)) and not torch.equal(copies, w.float())
    p = torch.zeros_like(w)
    opt = policy.AdamW([p], 0.0, weight_decay=0.0)
    zero = [torch.zeros_like(w)]
    opt.load_moments(zero, zero, 1, master=[copies])
    assert torch.equal(p.view(torch.int16), w.view(torch.int16))
    for _ in range(2):
        opt.step(zero)
        assert torch.equal(p, w) and torch.equal(opt.master()[:len(w)], copies)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_moments_without_copies(bits):
    """A run taken up from 16-bit weights and moments alone is the run of an
    optimizer that is made of these weights."""
    from puffysics_amd import policy
    params = tensors(SIZES, torch.bfloat16, 3)
    opt = policy.AdamW(params, LR, BETAS, EPS, DECAY, state_bits=bits, seed=4)
    for t in range(3):
        opt.step(tensors(SIZES, torch.bfloat16, 30 + t))
    twins = [p.clone() for p in params]
    twin = resumed(opt, twins, bits)
    m, v = opt.moments()
    opt.load_moments([x.clone() for x in views(opt, m)], [x.clone() for x in views(opt, v)], 3)
    assert equal(views(opt, opt.master()), [p.float() for p in params])
    grads = tensors(SIZES, torch.bfloat16, 40)
    opt.step(grads)
    twin.step(grads)
    assert equal(params, twins) and equal(views(opt, opt.master()), views(twin, twin.master()))


@pytest.mark.gpu
def test_written_copies_count():
    """master() is the state's own array: what is written there is gone on
    from, in the 16-bit weights alone."""
    from puffysics_amd import policy
    params = [tensors([300], torch.bfloat16, 5)[0], tensors([40], torch.float32, 6)[0]]
    other = params[1].clone()
    opt = policy.AdamW(params, 0.0, weight_decay=0.0)
    zero = [torch.zeros_like(p) for p in params]
    opt.step(zero)
    new = torch.randn(300, device="cuda")
    opt.master()[:300] = new
    opt.step(zero)
    assert torch.equal(opt.master()[:300], new) and torch.equal(params[0], new.bfloat16()) and torch.equal(params[1], other)
