"""Log probabilities, entropies, best alternatives and their gradient
(puffysics_amd.policy.log_probs) against the definition in 64 bits.

Tolerances.  A row's sum of exp(z) is a sum of positive terms; each term is
off by a few units in the last place and by |z| 2^-24 of its argument, a
thread adds at most 512 terms one after the other, the rest pairwise: a
relative error of 600 * 2^-24 < 4e-5 at the very worst, and so the logarithm's
absolute error; the entropy's terms grow with |z|.  z itself is exact to half
a unit.  Gradients: the same relative error on p, one rounding of the
difference, and the logits' type at the end."""
import numpy as np
import pytest
import torch

from policytest import EPS32, log_probs_gradient_oracle, log_probs_oracle

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"f32": 1e-44, "f16": 2.0 ** -24, "bf16": 1e-40}
SUM = 4e-5


def close(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(all="ignore"):
        bad = ~same & ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off, first at %s: %r, not %r" % (
        what, bad.sum(), bad.size, np.argwhere(bad)[0], got[bad][0], want[bad][0])


def inputs(rows, actions, type, seed, scale=3.0, wide=0):
    g = torch.Generator().manual_seed(seed)
    full = (torch.randn(rows, wide or actions, generator=g) * scale).to(TYPES[type]).cuda()
    x = full[:, (wide - actions) // 2 if wide else 0:][:, :actions]
    taken = torch.randint(0, actions, (rows,), generator=g)
    return x, taken


def check(x, taken, type, mask=None, top=0, gradient=True):
    from puffysics_amd import policy
    rows, actions = x.shape
    x = x.detach().requires_grad_(gradient)
    got = policy.log_probs(x, taken.cuda(), None if mask is None else mask.cuda(), top=top)
    xs, ts = x.detach().double().cpu().numpy(), taken.numpy()
    ms = None if mask is None else mask.numpy()
    lp, h, top_lp, top_a, every = log_probs_oracle(xs, ts, ms, top)
    size = np.abs(np.where(np.isfinite(lp), lp, 0))
    close(got.log_prob.detach().cpu(), lp, SUM + EPS32 * (size + 40), "log_prob")
    close(got.entropy.detach().cpu(), h, SUM * (1 + np.log(actions)) + 40 * EPS32, "entropy")
    if top:
        assert (got.top_action.cpu().numpy() == top_a).all()
        close(got.top_log_prob.cpu(), top_lp, SUM + EPS32 * (np.abs(np.where(np.isfinite(top_lp), top_lp, 0)) + 40), "top")
    else:
        assert got.top_action is None and got.top_log_prob is None
    if gradient:
        rng = np.random.default_rng(rows * 7 + actions)
        dl, dh = rng.standard_normal(rows).astype(np.float32), rng.standard_normal(rows).astype(np.float32)
        d, = torch.autograd.grad((got.log_prob, got.entropy), x, (torch.from_numpy(dl).cuda(), torch.from_numpy(dh).cuda()))
        assert d.dtype == x.dtype and d.shape == x.shape
        want = log_probs_gradient_oracle(xs, ts, ms, dl.astype(float), dh.astype(float))
        with np.errstate(all="ignore"):
            p, l = np.exp(every), np.where(every == -np.inf, 0, every)
            parts = np.abs(dl)[:, None] + np.abs(dh)[:, None] * (np.abs(l) + np.log(actions) + 1)
        one = np.zeros_like(p)
        for r, a in enumerate(ts):
            if 0 <= a < actions:
                one[r, a] = abs(dl[r])
        tol = 3 * SUM * p * parts * (1 + np.log(actions)) + 4 * EPS32 * one + HALF_UNIT[type] * np.abs(want) * 1.01 + LEAST[type]
        close(d.float().cpu(), want, tol, "gradient")


SIZES = [1, 2, 3, 5, 8, 17, 31, 63, 64, 65, 127, 130, 255, 256, 257, 511, 513, 1000, 1024, 1025, 2047, 2049, 4099, 8192,
         12289, 16383, 16385, 33000, 65536, 100003]


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("actions", SIZES)
def test_sizes(actions, type):
    rows = 1 + 2000 // actions + actions % 3
    x, taken = inputs(rows, actions, type, actions)
    check(x, taken, type, top=min(actions, (actions * 7) % 33))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,actions", [(1, 262144), (3, 262143), (1, 150001), (700, 20011), (20011, 3), (1, 1), (70000, 2)])
def test_few_and_many_rows(rows, actions):
    x, taken = inputs(rows, actions, "bf16", rows)
    check(x, taken, "bf16", top=min(actions, 3))


@pytest.mark.gpu
@pytest.mark.parametrize("actions", [2 ** 20, 2 ** 20 + 1, 2 ** 21])
def test_the_longest_rows(actions):
    """As many pieces to a row as there may be, with as many alternatives."""
    x, taken = inputs(2, actions, "f32", actions)
    check(x, taken, "f32", top=32)


@pytest.mark.gpu
def test_rows_past_32_bits():
    """More than 2^31 logits: the last rows are what they are alone."""
    from puffysics_amd import policy
    rows, actions = 17000, 131072
    x = torch.zeros(rows, actions, dtype=torch.bfloat16, device="cuda")
    x[-3:].copy_(inputs(3, actions, "bf16", 1)[0])
    taken = torch.full((rows,), 7, device="cuda")
    x.requires_grad_(True)
    got = policy.log_probs(x, taken, top=2)
    dl = torch.ones(rows, device="cuda")
    d, = torch.autograd.grad((got.log_prob, got.entropy), x, (dl, dl))
    tail = x.detach()[-3:].clone().requires_grad_(True)
    alone = policy.log_probs(tail, taken[-3:], top=2)
    d_alone, = torch.autograd.grad((alone.log_prob, alone.entropy), tail, (dl[-3:], dl[-3:]))
    assert torch.allclose(got.log_prob[-3:], alone.log_prob, rtol=0, atol=SUM) and torch.equal(got.top_action[-3:], alone.top_action)
    assert abs(float(got.log_prob[rows // 2].detach()) + np.log(actions)) < SUM
    assert torch.allclose(d[-3:].float(), d_alone.float(), rtol=2.0 ** -7, atol=1e-9)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,actions", [(2 ** 24 + 3, 2), (2 ** 23 + 3, 4097)])
def test_more_rows_than_a_launch_takes(rows, actions):
    """What follows the rows of the first launch (2^24 - 1, or half as many of
    two pieces) is what it is alone, in every result."""
    from puffysics_amd import policy
    odd = torch.tensor([0, rows // 2, rows - 77, rows - 5, rows - 4, rows - 3, rows - 2, rows - 1])
    x = torch.zeros(rows, actions, dtype=torch.bfloat16, device="cuda")
    x[odd] = inputs(len(odd), actions, "bf16", 1)[0]
    taken = torch.zeros(rows, dtype=torch.int64, device="cuda")
    taken[odd] = torch.arange(len(odd), device="cuda") % 2
    mask = torch.ones(actions, dtype=torch.bool, device="cuda")
    if actions == 2:
        mask = mask.repeat(rows, 1)
        mask[odd[-2], 0] = False
    x.requires_grad_(True)
    dl, dh = torch.ones(rows, device="cuda"), torch.zeros(rows, device="cuda")
    dl[odd], dh[odd] = torch.randn(len(odd), device="cuda"), torch.randn(len(odd), device="cuda")
    got = policy.log_probs(x, taken, mask, top=2)
    d, = torch.autograd.grad((got.log_prob, got.entropy), x, (dl, dh))
    few = x.detach()[odd].requires_grad_(True)
    alone = policy.log_probs(few, taken[odd], mask[odd] if mask.dim() == 2 else mask, top=2)
    d_alone, = torch.autograd.grad((alone.log_prob, alone.entropy), few, (dl[odd], dh[odd]))
    for a, b in zip(got, alone):
        assert torch.allclose(a[odd].double(), b.double(), rtol=0, atol=SUM)
    assert torch.allclose(d[odd].float(), d_alone.float(), rtol=2.0 ** -7, atol=1e-9)
    other = torch.ones(rows, dtype=torch.bool, device="cuda")
    other[odd] = False
    assert float((got.log_prob.detach()[other] + np.log(actions)).abs().max()) < SUM
    assert float((got.entropy.detach()[other] - np.log(actions)).abs().max()) < SUM
    assert (got.top_action[other] == torch.arange(2, device="cuda")).all()
    assert float((d[:, 0][other].float() - (1 - 1 / actions)).abs().max()) < 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("actions,wide", [(3, 8), (21, 22), (1021, 1040), (4097, 5003), (40001, 40020)])
def test_slices_of_wider_rows(actions, wide, type):
    x, taken = inputs(9, actions, type, wide, wide=wide)
    assert x.storage_offset() % 2 == ((wide - actions) // 2) % 2
    check(x, taken, type, top=2)


@pytest.mark.gpu
@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("actions", [1, 3, 40, 64, 300, 1021, 5000, 20000, 70001])
def test_masks(actions, type):
    """Rows that allow some, one, and no action; masked places hold NaN,
    infinities and the type's lowest value; taken actions that are masked,
    padding, and past the last."""
    rows = 24
    x, taken = inputs(rows, actions, type, actions)
    g = torch.Generator().manual_seed(5)
    mask = torch.rand(rows, actions, generator=g) < 0.6
    mask[3] = False
    mask[7] = False
    mask[7, actions // 2] = True
    mask[8] = True
    x = x.clone()
    for k, odd in enumerate((np.nan, np.inf, -np.inf, torch.finfo(TYPES[type]).min, torch.finfo(TYPES[type]).max)):
        row = x[10 + k]
        row[~mask[10 + k].cuda()] = odd
    x[3] = np.nan                                # a row that allows nothing and holds nothing
    taken[20], taken[21] = -1, -100
    with_masked = taken.clone()
    for r in range(rows):                        # most rows take an allowed action, row 9 need not
        ok = mask[r].nonzero()[:, 0]
        if len(ok) and taken[r] >= 0 and r != 9:
            taken[r] = ok[with_masked[r] % len(ok)]
    check(x, taken, type, mask, top=min(actions, 6))
    check(x, taken, type, mask[8], top=min(actions, 6), gradient=False)      # one row for all


@pytest.mark.gpu
@pytest.mark.parametrize("actions", [1, 4, 100, 2000, 30001])
def test_logits_that_are_not_numbers(actions):
    from puffysics_amd import policy
    rows = 8
    x, taken = inputs(rows, actions, "f32", 11)
    at = actions // 2
    x[1, at], x[2, at], x[3, at] = np.nan, np.inf, -np.inf
    x[4] = -np.inf
    x[5] = torch.finfo(torch.float32).min
    x[6] *= 1e30
    x[7] = np.nan
    top = min(actions, 4)
    got = policy.log_probs(x, taken.cuda(), top=top)
    lp, h, top_lp, top_a, _ = log_probs_oracle(x.cpu().numpy(), taken.numpy(), None, top)
    close(got.log_prob.cpu(), lp, SUM + EPS32 * (np.abs(np.nan_to_num(lp, posinf=0, neginf=0)) + 40), "log_prob")
    close(got.entropy.cpu(), h, SUM * (1 + np.log(actions)) + 40 * EPS32, "entropy")
    assert (got.top_action.cpu().numpy() == top_a).all()
    if actions > 1:
        assert torch.isnan(got.log_prob[[1, 2, 7]]).all() and torch.isnan(got.entropy[[1, 2, 7]]).all()


@pytest.mark.gpu
def test_action_past_the_last():
    from puffysics_amd import policy
    for actions in (3, 500, 40000):
        x, taken = inputs(4, actions, "f32", 3)
        taken[1], taken[2] = actions, 2 ** 40
        x.requires_grad_(True)
        got = policy.log_probs(x, taken.cuda())
        assert torch.isnan(got.log_prob).tolist() == [False, True, True, False]
        assert not torch.isnan(got.entropy).any()
        d, = torch.autograd.grad(got.log_prob.sum(), x)
        assert torch.isnan(d).all(1).tolist() == [False, True, True, False]
        assert torch.isnan(d).any(1).tolist() == [False, True, True, False]


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("actions", [32, 64, 700, 2048, 16384, 16400, 90000])
@pytest.mark.parametrize("kind", ["equal", "few values", "rising", "falling", "one lane", "zeros of both signs"])
def test_order_of_alternatives(kind, actions, type):
    """Ties go to the lowest action, wherever the largest lie."""
    from puffysics_amd import policy
    j = torch.arange(actions)
    x = {"equal": torch.full((actions,), 0.5), "few values": (j * 2654435761 % 5).float(), "rising": j * 1e-3,
         "falling": -j * 1e-3, "one lane": ((j // 4) % 64 == 17).float() * (1 + j * 1e-4),
         "zeros of both signs": torch.where(j % 3 == 0, -0.0, 0.0)}[kind]
    x = x.to(TYPES[type]).repeat(3, 1)
    x[1] = x[1].flip(0)
    for top in (1, 7, 32):
        got = policy.log_probs(x.cuda(), torch.zeros(3, dtype=torch.int64, device="cuda"), top=top)
        want = log_probs_oracle(x.double().numpy(), np.zeros(3, int), None, top)
        assert (got.top_action.cpu().numpy() == want[3]).all(), top
        close(got.top_log_prob.cpu(), want[2], SUM + EPS32 * (np.abs(want[2]) + 40), "top")


@pytest.mark.gpu
def test_gradient_against_differences():
    """Along random directions, with the function in 64 bits: (f(x + s u) -
    f(x - s u)) / 2 s is off by s^2 and 1e-16 / s."""
    for actions in (3, 77, 3001):
        x, taken = inputs(5, actions, "f32", actions)
        from puffysics_amd import policy
        rng = np.random.default_rng(1)
        dl, dh = rng.standard_normal(5).astype(np.float32), rng.standard_normal(5).astype(np.float32)
        leaf = x.detach().requires_grad_(True)
        got = policy.log_probs(leaf, taken.cuda())
        d, = torch.autograd.grad((got.log_prob, got.entropy), leaf, (torch.from_numpy(dl).cuda(), torch.from_numpy(dh).cuda()))
        xs, d = x.double().cpu().numpy(), d.double().cpu().numpy()

        def f(y):
            lp, h, *_ = log_probs_oracle(y, taken.numpy())
            return (dl * lp + dh * h).sum()

        for k in range(4):
            u = rng.standard_normal(xs.shape) / np.sqrt(actions)
            s = 1e-5
            slope = (f(xs + s * u) - f(xs - s * u)) / (2 * s)
            assert abs(slope - (d * u).sum()) <= 1e-7 + 3 * SUM * np.abs(d * u).sum()


def test_gradient_oracle_against_differences():
    rng = np.random.default_rng(2)
    x, taken = rng.standard_normal((4, 9)) * 2, np.array([0, 5, -1, 8])
    mask = rng.random((4, 9)) < 0.7
    mask[np.arange(4), np.maximum(taken, 0)] = True
    dl, dh = rng.standard_normal(4), rng.standard_normal(4)
    d = log_probs_gradient_oracle(x, taken, mask, dl, dh)

    def f(y):
        lp, h, *_ = log_probs_oracle(y, taken, mask)
        return (dl * lp + dh * h).sum()

    for r in range(4):
        for j in range(9):
            u = np.zeros_like(x)
            u[r, j] = 1e-6
            assert abs((f(x + u) - f(x - u)) / 2e-6 - d[r, j]) < 1e-8


@pytest.mark.gpu
def test_one_of_the_outputs_alone():
    """A loss of only log probabilities, only entropies, or of a mean, whose
    gradient is one number for all rows."""
    from puffysics_amd import policy
    for actions in (5, 3000):
        x, taken = inputs(6, actions, "f32", 1)
        for pick in (0, 1):
            leaf = x.detach().requires_grad_(True)
            policy.log_probs(leaf, taken.cuda())[pick].mean().backward()
            one, zero = np.full(6, 1 / 6), np.zeros(6)
            want = log_probs_gradient_oracle(x.cpu().numpy(), taken.numpy(), None, *((one, zero) if pick == 0 else (zero, one)))
            close(leaf.grad.cpu(), want, 20 * SUM * np.abs(want) + 1e-6, "gradient")


@pytest.mark.gpu
def test_differentiated_once():
    from puffysics_amd import policy
    x, taken = inputs(4, 6, "f32", 2)
    x = x.detach().requires_grad_(True)
    lp = policy.log_probs(x, taken.cuda()).log_prob
    d, = torch.autograd.grad(lp.sum(), x, create_graph=True)
    plain, = torch.autograd.grad(policy.log_probs(x, taken.cuda()).log_prob.sum(), x)
    assert torch.equal(d, plain)
    with pytest.raises(RuntimeError):
        d.square().sum().backward()


@pytest.mark.gpu
def test_shapes_and_types_of_arguments():
    from puffysics_amd import policy
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 4, 6, generator=g).cuda()
    taken = torch.randint(0, 6, (3, 4), generator=g).cuda()
    a = policy.log_probs(x, taken, top=2)
    assert a.log_prob.shape == (3, 4) and a.top_action.shape == (3, 4, 2)
    b = policy.log_probs(x.reshape(12, 6), taken.reshape(12).int(), top=2)
    assert torch.equal(a.log_prob.reshape(12), b.log_prob) and torch.equal(a.top_action.reshape(12, 2), b.top_action)
    turned = x.transpose(0, 2).contiguous().transpose(0, 2)                 # the last axis is not the contiguous one
    assert torch.equal(policy.log_probs(turned, taken).log_prob, a.log_prob)
    assert torch.equal(policy.log_probs(x[1, 2], taken[1, 2]).log_prob, a.log_prob[1, 2])
    none = policy.log_probs(torch.zeros(0, 6, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), top=3)
    assert none.log_prob.shape == (0,) and none.top_action.shape == (0, 3)
    rows = x[0, 0].expand(5, 6)
    assert torch.equal(policy.log_probs(rows, torch.zeros(5, dtype=torch.int64, device="cuda")).log_prob,
                       policy.log_probs(rows.contiguous(), torch.zeros(5, dtype=torch.int64, device="cuda")).log_prob)


@pytest.mark.gpu
def test_same_results_every_time_and_on_another_stream():
    from puffysics_amd import policy
    for rows, actions in ((2, 100000), (300, 3000), (5000, 3)):
        x, taken = inputs(rows, actions, "bf16", 4)
        taken = taken.cuda()
        a = policy.log_probs(x, taken, top=2)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            y = x.clone()
            b = policy.log_probs(y, taken, top=2)
        torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        grads = []
        for stream in (torch.cuda.current_stream(), s):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                leaf = x.clone().requires_grad_(True)
                policy.log_probs(leaf, taken)[0].sum().backward()
            torch.cuda.current_stream().wait_stream(stream)
            grads.append(leaf.grad)
        assert torch.equal(*grads)


@pytest.mark.gpu
def test_captured():
    """Replayed on new inputs in the same place, with other work between."""
    from puffysics_amd import policy
    for rows, actions in ((64, 3), (40, 2000), (2, 70000)):
        x, taken = inputs(rows, actions, "f32", 8)
        x, taken = x.clone(), taken.cuda()
        dl = torch.randn(rows, device="cuda")

        def go():
            leaf = x.detach().requires_grad_(True)
            got = policy.log_probs(leaf, taken, top=2)
            return (*got, torch.autograd.grad((got.log_prob, got.entropy), leaf, (dl, dl))[0])

        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            go()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go()
        for k in range(4):
            x.copy_(torch.randn_like(x))
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(out, go()))


def test_refusals():
    """Nothing is launched: this runs without a GPU."""
    from puffysics_amd import policy
    x, t = torch.zeros(4, 6), torch.zeros(4, dtype=torch.int64)
    bad = [dict(logits=x.double()), dict(taken=t.float()), dict(taken=t[:3]), dict(taken=t.bool()), dict(top=-1),
           dict(top=7), dict(mask=x), dict(mask=torch.ones(3, 6, dtype=torch.bool)), dict(logits=x[:, :0]),
           dict(mask=torch.ones(4, dtype=torch.bool)), dict()]                  # dict(): not on the GPU
    for change in bad:
        with pytest.raises(ValueError):
            policy.log_probs(**{**dict(logits=x, taken=t), **change})
    with pytest.raises(ValueError):
        policy.log_probs(torch.zeros(4, 600), t, top=33)


def test_complex_actions_are_refused():
    from puffysics_amd import policy
    with pytest.raises(ValueError, match="whole numbers"):
        policy.log_probs(torch.zeros(4, 6), torch.zeros(4, dtype=torch.complex64))


def test_refusals_of_the_c_entry():
    from puffysics_amd import policy
    lib = policy.policy_lib()
    L = policy.B3Logits
    good = dict(data=64, type=0, rows=4, actions=6, row_stride=6, mask=None, mask_row_stride=0)
    call = lambda top=0, ws=0, **k: lib.b3_log_probs_gpu(L(**{**good, **k}), 64, 64, 64, None, top, 64, 64, None, ws, None)  # noqa: E731
    for k in (dict(type=3), dict(type=-1), dict(rows=-1), dict(actions=0), dict(actions=2 ** 30 + 1, row_stride=2 ** 31),
              dict(row_stride=5), dict(data=None), dict(mask=64, mask_row_stride=5), dict(top=7), dict(top=-1),
              dict(rows=2 ** 31)):
        assert call(**k) == 1, k
    assert call(actions=100, row_stride=100, top=33) == 1
    assert call(rows=0) == 0
    back = lambda **k: lib.b3_log_probs_backward_gpu(L(**{**good, **k}), 64, k.pop("stats", 64), 64, None, 0, None, 0, 64,  # noqa: E731
                                                     k.pop("d_stride", 6), None)
    assert back(row_stride=3) == 1 and back(rows=0) == 0
    assert lib.b3_log_probs_backward_gpu(L(**good), 64, 64, 64, None, 0, None, 0, 64, 5, None) == 1
    assert lib.b3_log_probs_backward_gpu(L(**good), 64, None, 64, None, 0, None, 0, 64, 6, None) == 1
    assert lib.b3_log_probs_backward_gpu(L(**good), 64, 64, 64, None, -1, None, 0, 64, 6, None) == 1
