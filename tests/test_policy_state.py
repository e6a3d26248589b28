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


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [1, 2])
def test_8_bit_moments_follow_in_replays(graphs):
    """A steady gradient through replays of captured steps: the second moment
    goes the way of the formula, from above and from below.  As in single
    steps, rounding raises its mean square by at most 12.5%.  Below, its root
    rises from a hundredth of the gradient; above, it falls from ten times."""
    from puffysics_amd import policy
    n, steps, g0 = 8192, 1000, 0.02
    p = torch.zeros(2 * n, device="cuda")
    g = torch.full_like(p, g0)
    opt = policy.AdamW([p], 0.0, BETAS, EPS, 0.0, state_bits=8)
    start = torch.full_like(p, (0.01 * g0) ** 2)
    start[n:] = (10 * g0) ** 2
    opt.load_moments([g], [start], 5)
    captured = [torch.cuda.CUDAGraph() for _ in range(graphs)]
    for graph in captured:
        with torch.cuda.graph(graph):
            opt.step([g])
    for k in range(steps):
        captured[k % graphs].replay()
        if k % 100 == 3:
            opt.step([g])
    steps += steps // 100
    assert opt.steps() == 5 + graphs + 10
    m, v = opt.moments()
    for part, v0 in ((slice(0, n), (0.01 * g0) ** 2), (slice(n, 2 * n), (10 * g0) ** 2)):
        want = g0 ** 2 + (v0 - g0 ** 2) * BETAS[1] ** steps
        assert 0.99 * want < float(v[part].float().mean()) < 1.13 * want
        assert len(v[part].unique()) > 1
    assert abs(float(m.float().mean()) - g0) < 0.005 * g0


@pytest.mark.gpu
def test_replays_round_by_other_bits_and_the_first_by_its_own():
    """The first run of a captured step is the step that was captured; every
    later one rounds the same values otherwise."""
    from puffysics_amd import policy
    g = torch.randn(4096, device="cuda") * 0.01
    zero = torch.zeros_like(g)

    def run(captured):
        opt = policy.AdamW([torch.zeros_like(g)], 0.0, BETAS, EPS, 0.0, state_bits=8, seed=11)
        if not captured:
            opt.step([g])
            return [opt.moments()]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step([g])
        got = []
        for _ in range(4):
            opt.load_moments([zero], [zero], 0)
            graph.replay()
            torch.cuda.synchronize()
            got.append(opt.moments())
        return got

    want, got = run(False)[0], run(True)
    assert equal(got[0], want)
    for i in range(4):
        for j in range(i):
            assert all(int((a != b).sum()) > 400 for a, b in zip(got[i], got[j]))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_every_tensor_resumes_from_its_own_count(bits):
    """Tensors that had no gradient in some steps go on with the corrections
    and the rounding of their own counts."""
    from puffysics_amd import policy
    params = tensors(SIZES, torch.float32, 7)
    opt = policy.AdamW(params, LR, BETAS, EPS, DECAY, state_bits=bits, seed=4)
    for t in range(4):
        opt.step([g if (i + t) % 3 or i == 0 else None for i, g in enumerate(tensors(SIZES, torch.float32, 50 + t))])
    counts = [opt.steps(i) for i in range(len(params))]
    assert len(set(counts)) > 1
    twins = [p.clone() for p in params]
    twin = policy.AdamW(twins, LR, BETAS, EPS, DECAY, state_bits=bits, seed=4)
    m, v = opt.moments()
    twin.load_moments(views(opt, m), views(opt, v), counts)
    assert [twin.steps(i) for i in range(len(params))] == counts
    for t in range(2):
        grads = tensors(SIZES, torch.float32, 60 + t)
        opt.step(grads)
        twin.step(grads)
    assert equal(params, twins) and equal(opt.moments(), twin.moments())
    assert [opt.steps(i) for i in range(len(params))] == [k + 2 for k in counts]


@pytest.mark.gpu
@pytest.mark.parametrize("step", [-1, 2.5, [1], [1, -1], [1, 2, 3], [1, 2.0], "3", 2 ** 63])
def test_refused_counts_leave_the_state(step):
    from puffysics_amd import policy
    p = [torch.zeros(40, device="cuda"), torch.zeros(7, device="cuda")]
    opt = policy.AdamW(p, LR)
    one = [torch.ones(40), torch.ones(7)]
    with pytest.raises(ValueError):
        opt.load_moments(one, one, step)
    assert all(int(torch.count_nonzero(x)) == 0 for x in opt.moments()) and opt.steps(0) == opt.steps(1) == 0
    opt.load_moments(one, one, (np.int64(3), 4))
    assert opt.steps(0) == 3 and opt.steps(1) == 4


def grid_values(first, last, groups, seed):
    """e4m3 numbers in groups of 32 on every scale 2^(b - 127) from b = first
    to last: random ones of both signs and the largest, which pins the scale."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float().cuda()
    x = codes[torch.randint(0, 127, (last - first + 1, groups, 32), generator=g, device="cuda")]
    x[..., 0] = 448.0
    x *= torch.randint(0, 2, x.shape, generator=g, device="cuda") * 2 - 1
    scale = (torch.arange(first, last + 1, dtype=torch.int32, device="cuda") << 23).view(torch.float32)
    return (x * scale[:, None, None]).reshape(-1)


def same_where_held(got, x):
    """got, in bf16, is x wherever bf16 holds it, and for nearly all it does."""
    held = x.bfloat16().float() == x
    return float(held.float().mean()) > 0.95 and torch.equal(got[held].float(), x[held])


@pytest.mark.gpu
def test_values_on_the_grid_stay():
    """A moment that 8 bits can hold is not rounded, on every scale: with
    rates of 0 a step's moments are the gradient and its square.  Where the
    factor to the grid is a unit low, one in 2^16 random bits takes it a step
    of the grid down; 2^18 values a scale meet each four times.  A factor that
    is high would make the largest of a group NaN.  Squares stay within 32
    bits on the scales from 80 to 180."""
    from puffysics_amd import policy
    for first, last, square in ((1, 246, False), (80, 180, True)):
        x = grid_values(first, last, 2 ** 13, first)
        opt = policy.AdamW([torch.zeros_like(x)], 0.0, (0.0, 0.0), state_bits=8)
        opt.step([x])
        for got, want in zip(opt.moments(), (x, x * x) if square else (x,)):
            held = want.bfloat16().float() == want
            assert float(held.float().mean()) > 0.95 and torch.isfinite(got[held]).all()
            off = held & (got.float() != want)
            assert (off.view(last - first + 1, -1).sum(1) <= 40).all()
            down = (want[off].abs() - got[off].float().abs()) / want[off].abs()
            # a step of the grid is an eighth at most
            assert (down > 0).all() and (down <= (0.235 if square and want is not x else 0.126)).all()


@pytest.mark.gpu
def test_values_on_the_grid_are_read_in_and_out():
    from puffysics_amd import policy
    for first, last in ((1, 246), (80, 180)):
        x = grid_values(first, last, 16, first + 5)
        opt = policy.AdamW([torch.zeros_like(x)], state_bits=8)
        opt.load_moments([x], [x * x if first == 80 else torch.zeros_like(x)], 1)
        m, v = opt.moments()
        assert same_where_held(m, x)
        if first == 80:
            assert same_where_held(v, x * x)
            opt.load_moments([m], [v], 1)
            assert equal(opt.moments(), (m, v))


def test_overlapping_parameters_are_refused():
    """Before anything is done with them: this runs without a GPU."""
    from puffysics_amd import policy
    whole = torch.zeros(100)
    for params in ([whole[:60], whole[59:]], [whole[50:], whole[:51]], [whole, whole[99:]], [whole[10:20], whole],
                   [whole, whole.view(torch.bfloat16)[199:]], [whole, whole[:0], whole[5:6]]):
        with pytest.raises(ValueError, match="overlap"):
            policy.AdamW(params, LR)
    for params in ([whole[:60], whole[60:]], [whole, whole[:0], whole[7:7]], [whole.view(torch.float16)[:3], whole[2:]]):
        with pytest.raises(ValueError, match="CUDA device"):          # the next check
            policy.AdamW(params, LR)


def test_overlapping_tensors_are_refused_by_the_c_entry():
    from puffysics_amd import policy
    lib, C, T = policy.policy_lib(), policy.C, policy.B3AdamWTensor
    state, config = policy.B3AdamWState(32, 64, 64, None, None, None), policy.B3AdamWConfig(0.9, 0.999, 1e-8, 0)
    h = C.c_void_p()
    for tensors in ([(4096, 0, 10), (4132, 0, 3)], [(4132, 0, 3), (4096, 0, 10)], [(4096, 1, 10), (4114, 2, 1)],
                    [(4096, 0, 100), (8192, 0, 1), (4097, 2, 1)]):
        table = (T * len(tensors))(*[T(*t, 0.0) for t in tensors])
        assert lib.b3_adamw_create(C.byref(h), table, len(tensors), state, config) == 1 and not h.value


@pytest.mark.gpu
def test_8_bit_moments_lie_anywhere():
    """Codes and scales are bytes: a state at odd addresses goes the way of
    an aligned one, in steps, out and in again."""
    from puffysics_amd import policy
    lib, C = policy.policy_lib(), policy.C
    sizes = [1, 300, 4097, 20000]
    offsets = [0, 256, 768, 768 + 4352]
    total = 768 + 4352 + 20224
    runs = []
    for odd in ((0, 0, 0, 0), (1, 3, 1, 1), (2, 1, 3, 5)):
        params = tensors(sizes, torch.float32, 8)
        memory = [torch.zeros(n + 64, dtype=torch.uint8, device="cuda") for n in (total, total, total // 32, total // 32)]
        at = [x[16 + o:] for x, o in zip(memory, odd)]
        for x in at[2:]:
            x.fill_(1)
        table = (policy.B3AdamWTensor * 4)(*[policy.B3AdamWTensor(p.data_ptr(), 0, p.numel(), DECAY) for p in params])
        assert lib.b3_adamw_size(table, 4) == total
        state = policy.B3AdamWState(8, *[x.data_ptr() for x in at], None)
        h = C.c_void_p()
        torch.cuda.synchronize()
        assert lib.b3_adamw_create(C.byref(h), table, 4, state, policy.B3AdamWConfig(*BETAS, EPS, 4)) == 0
        out = torch.zeros((2, total), dtype=torch.bfloat16, device="cuda")
        for t in range(3):
            grads = tensors(sizes, torch.float32, 80 + t)
            pointers = (C.c_void_p * 4)(*[g.data_ptr() for g in grads])
            assert lib.b3_adamw_step_gpu(h, pointers, None, LR, 0.0, None, None) == 0
            torch.cuda.synchronize()
        for _ in range(2):
            assert lib.b3_adamw_moments_gpu(h, out[0].data_ptr(), out[1].data_ptr(), None) == 0
            torch.cuda.synchronize()
            runs.append((*params, out.clone()))
            flat = out.float()
            assert lib.b3_adamw_load_moments_gpu(h, flat[0].data_ptr(), flat[1].data_ptr(), None) == 0
            torch.cuda.synchronize()
        assert all(int(torch.count_nonzero(x[:16 + o])) == 0 for x, o in zip(memory[:2], odd))
        assert lib.b3_adamw_destroy(h) == 0
    assert offsets[3] + 20224 == total and all(equal(r, runs[0]) for r in runs[1:])


def test_workspaces_are_aligned():
    """Nothing is launched: this runs without a GPU."""
    from puffysics_amd import policy
    lib, C = policy.policy_lib(), policy.C
    need = lib.b3_log_probs_workspace(2, 100000, 3)
    x = policy.B3Logits(64, 0, 2, 100000, 100000, None, 0)
    g = policy.B3Rollout(20000, 2, 64, (2, 1), 64, 0, (2, 1), 64, 1, 64, 0, (2, 1), 64, 64, (2, 1))
    size = lib.b3_advantages_workspace(20000, 2)
    assert need > 0 and size > 0
    for at in (None, 65, 68):
        assert lib.b3_log_probs_gpu(x, 64, 64, 64, None, 3, 64, 64, at, need, None) == 1
        assert lib.b3_advantages_gpu(C.byref(g), 0.9, 0.9, at, size, None) == 1
    assert lib.b3_log_probs_gpu(x, 64, 64, 64, None, 3, 64, 64, 64, need - 1, None) == 1
    assert lib.b3_advantages_gpu(C.byref(g), 0.9, 0.9, 64, 8, None) == 1      # the size is for either layout


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [None, 1.0])
def test_empty_tensors_count_their_steps(clip):
    """A gradient without elements is a gradient: steps() of the first tensor
    is what a run is taken up from."""
    from puffysics_amd import policy
    params = [torch.zeros(0, device="cuda"), torch.ones(5, device="cuda"), torch.zeros((3, 0), device="cuda")]
    opt = policy.AdamW(params, LR, max_grad_norm=clip)
    for t in range(3):
        opt.step([torch.ones_like(p) if t != 1 or i else None for i, p in enumerate(params)])
    assert [opt.steps(i) for i in range(3)] == [2, 3, 3]
