"""puffysics_amd.policy.rms_norm, rms_norm_8bit and values_of_8bit against the
definition in 64 bits."""
import pytest
import torch

from memorytest import STEP, eight_bits_oracle, norm_gradient_oracle, norm_oracle

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
#        rows, width: both sides of every change of lanes, vectors and passes
SIZES = [(1, 1), (3, 7), (5, 8), (70, 32), (9, 33), (6, 128), (300, 129), (17, 256), (5, 257), (4, 512), (3, 513), (2, 1021),
         (3, 1024), (2, 1025), (3, 2048), (2, 2049), (3, 4096), (2, 5001), (2, 8193), (1, 16384), (2, 16385), (3, 40001)]


def made(rows, width, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x, r, dy, dh = (torch.randn(rows, width, generator=g).to(dtype).cuda() for _ in range(4))
    return x, 3 * r, (1 + 0.3 * torch.randn(width, generator=g)).cuda(), dy, dh


def close(got, want, factor, size, out_type):
    """Off by `factor` of `size`, and by half a step of the result's type."""
    least = 2.0 ** -25 if out_type == torch.float16 else 0.0
    bad = (got.double() - want).abs() > factor * size + STEP[out_type] * want.abs() + least + 1e-37
    assert not bad.any(), ((got.double() - want).abs()[bad].max(), int(bad.sum()))


def wide(width):
    """Roundings in 32 bits: the squares of a row are added in lanes and then
    over lanes, no more than width / 4 + 16 after another, half of what that
    gives goes into the root; and a few more of the root, products and sum."""
    return (width / 8 + 16) * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("weight", ["none", "f32", "same"])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_forward_and_gradient(size, type, weight):
    from puffysics_amd import policy
    dtype, eps = TYPES[type], 1e-5
    x, r, w, dy, dh = made(*size, dtype, sum(size))
    w = None if weight == "none" else w if weight == "f32" else w.to(dtype)
    for residual in (None, r):
        leaves = [y.detach().clone().requires_grad_() for y in (x, w, residual) if y is not None]
        lx, lw, lr = leaves[0], leaves[1] if w is not None else None, leaves[-1] if residual is not None else None
        got = policy.rms_norm(lx, lw, residual=lr, eps=eps)
        plain = policy.rms_norm(x, w, residual=residual, eps=eps)
        assert torch.equal(plain.out, got.out)
        y, h, s = norm_oracle(x, w, residual, eps)
        close(got.out, y, wide(size[1]), y.abs() + 2.0 ** -24, dtype)
        outs, ups = (got.out,), (dy,)
        if residual is None:
            assert got.sum is None
        else:
            assert torch.equal(got.sum, (x.float() + r.float()).to(dtype)) and torch.equal(plain.sum, got.sum)
            outs, ups = (got.out, got.sum), (dy, dh)
        grads = torch.autograd.grad(outs, leaves, ups)
        d, dw = norm_gradient_oracle(h, w, eps, dy, dh if residual is not None else None)
        one = 1.0 if w is None else w.double()
        inner = (one * dy.double() * h.double() * s).abs().mean(-1, keepdim=True)
        most = s * ((one * dy.double()).abs() + 3 * h.double().abs() * s * inner)
        close(grads[0], d, 2 * wide(size[1]), most + (dh.double().abs() if residual is not None else 0), dtype)
        if residual is not None:
            assert torch.equal(grads[0], grads[-1])
        if w is not None:
            most = (dy.double() * h.double() * s).abs().sum(0)
            close(grads[1], dw, wide(size[1]) + size[0] * 2.0 ** -24, most, w.dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("rows,width", [(20000, 40), (3000, 700), (1500, 3000)])
def test_many_rows(rows, width, type):
    """More rows than workgroups take at once."""
    from puffysics_amd import policy
    dtype = TYPES[type]
    x, r, w, dy, dh = made(rows, width, dtype, 5)
    leaves = [x.requires_grad_(), w.requires_grad_(), r.requires_grad_()]
    got = policy.rms_norm(x, w, residual=r)
    grads = torch.autograd.grad((got.out, got.sum), leaves, (dy, dh))
    with torch.no_grad():
        y, h, s = norm_oracle(x, w, r, 1e-6)
        close(got.out, y, wide(width), y.abs(), dtype)
        d, dw = norm_gradient_oracle(h, w, 1e-6, dy, dh)
        most = (dy.double() * h.double() * s).abs()
        inner = (most * w.double().abs()).mean(-1, keepdim=True)
        close(grads[0], d, 2 * wide(width),
              s * ((w.double() * dy.double()).abs() + 3 * h.double().abs() * s * inner) + dh.double().abs(), dtype)
        # rows are added by one after the other in a lane, lanes and workgroups in a few dozen sums
        close(grads[1], dw, (width / 8 + rows / 256 + 128) * 2.0 ** -24, most.sum(0), torch.float32)


@pytest.mark.gpu
def test_gradient_by_differences():
    from puffysics_amd import policy
    x, r, w, dy, dh = made(3, 37, torch.float32, 2)
    leaves = [y.requires_grad_() for y in (x, w, r)]
    got = policy.rms_norm(x, w, residual=r, eps=0.1)
    grads = torch.autograd.grad((got.out, got.sum), leaves, (dy, dh))

    def loss(x, w, r):
        y, h, _ = norm_oracle(x, w, r, 0.1)
        return (y * dy.double()).sum() + (h * dh.double()).sum()

    base = [y.detach().double() for y in leaves]
    for i, grad in enumerate(grads):
        for at in range(0, base[i].numel(), 5):
            up, down = ([y.clone() for y in base] for _ in range(2))
            up[i].view(-1)[at] += 1e-5
            down[i].view(-1)[at] -= 1e-5
            d = float(loss(*up) - loss(*down)) / 2e-5
            assert abs(d - float(grad.view(-1)[at])) < 1e-5 * (1 + abs(d))


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_eight_bits(size, type):
    """The numbers are those of values within the 32-bit roundings of the
    definition's: between the roundings of the two ends."""
    from puffysics_amd import policy
    dtype = TYPES[type]
    x, r, w, _, _ = made(*size, dtype, sum(size) + 3)
    x[0, ::3] *= 1e-3                                      # numbers below the least normal one of a group
    for residual in (None, r):
        got = policy.rms_norm_8bit(x, w, residual=residual)
        assert got.out.dtype == torch.float8_e4m3fn and got.out.shape == x.shape
        assert got.scale.dtype == torch.float8_e8m0fnu and got.scale.shape == (size[0], -(-size[1] // 32))
        assert (got.sum is None) if residual is None else torch.equal(got.sum, policy.rms_norm(x, w, residual=r).sum)
        y = norm_oracle(x, w, residual, 1e-6)[0]
        values = policy.values_of_8bit(got.out, got.scale, torch.float32).double()
        power = torch.log2(got.scale.view(torch.uint8).double().sub(127).exp2())
        near = (wide(size[1]) + 2.0 ** -22) * y.abs()
        for low, high in ((y - near, y + near),):
            ends = [eight_bits_oracle(z) for z in (low, high)]
            same = (ends[0][1] == ends[1][1])
            assert torch.equal(power[same], ends[0][1][same])
            assert ((power == ends[0][1]) | (power == ends[1][1])).all()
            each = same.repeat_interleave(32, 1)[:, :size[1]]
            a, b = (e[0] * torch.exp2(e[1]).repeat_interleave(32, 1)[:, :size[1]] for e in ends)
            assert (torch.minimum(a, b)[each] <= values[each]).all() and (values[each] <= torch.maximum(a, b)[each]).all()
        for t in TYPES.values():
            v = policy.values_of_8bit(got.out, got.scale, t)
            assert torch.equal(v, values.to(t)) and v.dtype == t


@pytest.mark.gpu
def test_eight_bits_of_zeros_and_borders():
    """448 of a power is held by it, what is over goes to the next; ties go to
    the even; zeros have the least power; what is not finite is NaN."""
    from puffysics_amd import policy
    x = torch.zeros(4, 64, device="cuda")
    x[0, :32] = 1.0
    x[1, 0], x[1, 40] = 2.0, 2.0
    x[2, 5] = float("nan")
    x[3, 5] = float("inf")
    got = policy.rms_norm_8bit(x, eps=0.0)
    v = policy.values_of_8bit(got.out, got.scale, torch.float32)
    assert got.scale.view(torch.uint8)[0, 1] == 1 and (v[0, 32:] == 0).all()
    assert v[2].isnan().all() and v[3, 5].isnan()
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(8, 32)
    for b in (0, 1, 119, 127, 140, 254, 255):
        scale = torch.full((8, 1), b, dtype=torch.uint8, device="cuda")
        got = policy.values_of_8bit(codes.view(torch.float8_e4m3fn), scale.view(torch.float8_e8m0fnu), torch.float32)
        want = codes.view(torch.float8_e4m3fn).float().double() * (2.0 ** (b - 127) if b < 255 else float("nan"))
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0), want.float().nan_to_num(7.0))


@pytest.mark.gpu
def test_rows_that_are_special():
    """A row of zeros is 0, with eps 0 NaN as 0 / 0 is; NaN and infinities stay
    in their row, also in the gradient."""
    from puffysics_amd import policy
    x = torch.randn(5, 40, device="cuda")
    want = policy.rms_norm(x).out
    x[1], x[3, 7] = 0.0, float("nan")
    leaf = x.clone().requires_grad_()
    out = policy.rms_norm(leaf).out
    assert (out[1] == 0).all() and out[3].isnan().all() and torch.equal(out[[0, 2, 4]], want[[0, 2, 4]])
    d, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert d[3].isnan().all() and torch.isfinite(d[[0, 1, 2, 4]]).all()
    assert policy.rms_norm(x, eps=0.0).out[1].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("type", TYPES)
def test_strides(type):
    from puffysics_amd import policy
    dtype = TYPES[type]
    g = torch.Generator().manual_seed(3)
    big = torch.randn(6, 9, 101, generator=g).to(dtype).cuda()
    w = torch.randn(100, generator=g).to(dtype).cuda()
    for x in (big[..., 1:], big.transpose(0, 1)[..., :100], big[:, :, 1:51].repeat_interleave(2, 2)[..., ::1],
              big[2:3, 4:5, 1:].expand(4, 5, 100), big[1, 2, :100]):
        xs = [x.detach().requires_grad_() for _ in range(2)]
        ys = [x.detach().contiguous().requires_grad_() for _ in range(2)]
        a, b = policy.rms_norm(xs[0], w, residual=xs[1]), policy.rms_norm(ys[0], w, residual=ys[1])
        assert torch.equal(a.out, b.out) and torch.equal(a.sum, b.sum) and a.out.shape == x.shape
        up = torch.randn(x.shape, generator=g).to(dtype).cuda()
        wide_up = torch.stack([up, up], -1)[..., 0]
        da = torch.autograd.grad((a.out, a.sum), xs, (wide_up, wide_up))
        db = torch.autograd.grad((b.out, b.sum), ys, (up, up))
        assert all(torch.equal(i, j) for i, j in zip(da, db))
        p, q = policy.rms_norm_8bit(x, w, residual=x), policy.rms_norm_8bit(x.contiguous(), w, residual=x.contiguous())
        assert torch.equal(p.out.view(torch.uint8), q.out.view(torch.uint8))
        assert torch.equal(p.scale.view(torch.uint8), q.scale.view(torch.uint8)) and torch.equal(p.sum, q.sum)


@pytest.mark.gpu
def test_nothing_to_do():
    from puffysics_amd import policy
    x, w = torch.zeros(0, 8, device="cuda", requires_grad=True), torch.ones(8, device="cuda", requires_grad=True)
    got = policy.rms_norm(x, w, residual=x)
    dx, dw = torch.autograd.grad((got.out, got.sum), (x, w), (torch.ones_like(x), torch.ones_like(x)))
    assert dx.shape == (0, 8) and torch.equal(dw, torch.zeros(8, device="cuda"))
    x = x.detach()
    e = policy.rms_norm_8bit(x)
    assert e.out.shape == (0, 8) and e.scale.shape == (0, 1) and policy.values_of_8bit(e.out, e.scale).shape == (0, 8)


@pytest.mark.gpu
def test_partial_gradients():
    """Of one output alone, of one input alone; into the same leaf twice."""
    from puffysics_amd import policy
    x, r, w, dy, dh = made(7, 300, torch.float32, 8)
    x, r, w = (y.requires_grad_() for y in (x, r, w))
    got = policy.rms_norm(x, w, residual=r)
    of_out = torch.autograd.grad(got.out, (x, w), dy, retain_graph=True)
    of_sum = torch.autograd.grad(got.sum, (x,), dh, retain_graph=True)
    both = torch.autograd.grad((got.out, got.sum), (x, w), (dy, dh))
    assert torch.equal(of_sum[0], dh) and torch.allclose(of_out[0] + dh, both[0], atol=1e-6) and torch.equal(of_out[1], both[1])
    alone = policy.rms_norm(x.detach(), w, residual=r.detach())
    assert torch.equal(torch.autograd.grad(alone.out, w, dy)[0], both[1])
    twice = policy.rms_norm(x, w, residual=x)
    d, = torch.autograd.grad(twice.sum, x, dh)
    assert torch.equal(d, 2 * dh)
    (policy.rms_norm(x, w, residual=r).out * dy).sum().backward()
    assert x.grad.data_ptr() != r.grad.data_ptr() and torch.equal(x.grad, r.grad)


@pytest.mark.gpu
def test_streams_and_replays():
    from puffysics_amd import policy
    x, r, w, dy, dh = made(50, 600, torch.bfloat16, 9)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    want = policy.rms_norm(x, w, residual=r)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = policy.rms_norm(x, w, residual=r)
    side.synchronize()
    assert torch.equal(got.out, want.out)
    with torch.cuda.graph(graph):
        a, b = policy.rms_norm(x, w, residual=r), policy.rms_norm_8bit(x, w, residual=r)
        values = policy.values_of_8bit(b.out, b.scale)
    for _ in range(3):
        x.add_(0.5)
        graph.replay()
        c, d = policy.rms_norm(x, w, residual=r), policy.rms_norm_8bit(x, w, residual=r)
        torch.cuda.synchronize()
        assert torch.equal(a.out, c.out) and torch.equal(a.sum, c.sum)
        assert torch.equal(values, policy.values_of_8bit(d.out, d.scale))


@pytest.mark.gpu
def test_negated_arrays():
    """Tensors that are only marked as negated are read as what they are."""
    from puffysics_amd import policy
    from test_policy_arguments import negated
    x, r, w, dy, dh = made(6, 50, torch.float32, 4)
    want, got = policy.rms_norm(x, w, residual=r), policy.rms_norm(negated(x), negated(w), residual=negated(r))
    assert torch.equal(got.out, want.out) and torch.equal(got.sum, want.sum)
    a, b = policy.rms_norm_8bit(x, w, residual=r), policy.rms_norm_8bit(negated(x), negated(w), residual=negated(r))
    assert torch.equal(a.out.view(torch.uint8), b.out.view(torch.uint8)) and torch.equal(a.sum, b.sum)
    leaf = x.clone().requires_grad_()
    c, = torch.autograd.grad(policy.rms_norm(leaf, w).out, leaf, dy)
    d, = torch.autograd.grad(policy.rms_norm(leaf, w).out, leaf, negated(dy))
    assert torch.equal(c, d)


@pytest.mark.gpu
def test_the_longest_rows():
    """Of 2^21 elements, whose weights' gradient is summed by few workgroups."""
    from puffysics_amd import policy
    x = torch.randn(20, 2 ** 21, device="cuda").requires_grad_()
    w = torch.ones(2 ** 21, device="cuda").requires_grad_()
    out = policy.rms_norm(x, w).out
    y, _, s = norm_oracle(x.detach(), None, None, 1e-6)
    # a lane of 256 adds 1,024 vectors of 8 one after the other
    assert (out - y).abs().max() < 1040 * 2.0 ** -24 * float(y.abs().max())
    dx, dw = torch.autograd.grad(out, (x, w), out.detach())
    assert (dw - y.square().sum(0)).abs().max() < 1100 * 2.0 ** -23 * float(y.square().sum(0).max())
    assert torch.isfinite(dx).all()


@pytest.mark.gpu
def test_places_past_32_bits():
    """The last rows of an array of more than 2^32 bytes, and of 2^31 elements."""
    from puffysics_amd import policy
    rows, width = 2 ** 20 + 3, 2048 + 8
    x = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    x[-3:] = torch.randn(3, width, device="cuda").bfloat16()
    x[:3] = 1.0
    out = policy.rms_norm(x).out
    assert torch.equal(out[-3:], policy.rms_norm(x[-3:].clone()).out) and torch.equal(out[:3], policy.rms_norm(x[:3].clone()).out)


def test_refusals():
    """Nothing is launched: this runs without a GPU."""
    from puffysics_amd import policy
    x, w = torch.zeros(4, 6), torch.zeros(6)
    for call in (policy.rms_norm, policy.rms_norm_8bit):
        for what, args in (("float32, float16", dict(x=x.double())), ("2.21", dict(x=torch.zeros(4, 0))),
                           ("2.21", dict(x=torch.zeros(()))), ("2.21", dict(x=w[:1].expand(2, 2 ** 21 + 1))),
                           ("2.31", dict(x=w[:1].expand(2 ** 31, 1))), ("shape and type", dict(x=x, residual=x[:2])),
                           ("shape and type", dict(x=x, residual=x.half())), ("weight", dict(x=x, weight=w[:5])),
                           ("weight", dict(x=x, weight=w.half())), ("weight", dict(x=x.half(), weight=w.bfloat16())),
                           ("eps", dict(x=x, eps=-1e-6)), ("eps", dict(x=x, eps=float("nan"))),
                           ("CUDA device", dict(x=x, weight=w, residual=x))):
            with pytest.raises(ValueError, match=what):
                call(**args)
    with pytest.raises(ValueError, match="no gradient"):
        policy.rms_norm_8bit(x, w.clone().requires_grad_())
    e, s = torch.zeros(4, 40, dtype=torch.float8_e4m3fn), torch.zeros(4, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    for args in ((x, s), (e, x), (e, s[:, :1]), (e, s, torch.float64), (e, s)):
        with pytest.raises(ValueError):
            policy.values_of_8bit(*args)
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), pytest.raises(ValueError, match="forward-mode"):
        policy.rms_norm(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(30, 32), (6, 5, 32), (2, 3, 5, 32), (32,)], ids=str)
def test_results_written_in_place(shape):
    """A program may go on in place from either result, whatever its axes."""
    from puffysics_amd import policy
    x, r = (torch.randn(shape, device="cuda").bfloat16().requires_grad_() for _ in range(2))
    w = torch.randn(32, device="cuda", requires_grad=True)
    up = torch.randn(shape, device="cuda").bfloat16()
    got = policy.rms_norm(x, w, residual=r)
    want = torch.autograd.grad((got.out * 2, got.sum + up), (x, r, w), (up, up))
    got = policy.rms_norm(x, w, residual=r)
    got.out.mul_(2)
    got.sum.add_(up)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad((got.out, got.sum), (x, r, w), (up, up)), want))
    out = policy.rms_norm(x, w).out
    out.relu_()
    want = torch.autograd.grad(torch.relu(policy.rms_norm(x, w).out), x, up)[0]
    assert torch.equal(torch.autograd.grad(out, x, up)[0], want)
    with torch.no_grad():
        policy.rms_norm(x, w, residual=r).sum.add_(up)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(30, 32), (6, 5, 32)], ids=str)
def test_gradients_of_two_leaves_are_two(shape):
    """x and the residual get gradients of their own, which a program may
    write to one by one."""
    from puffysics_amd import policy
    x, r = (torch.randn(shape, device="cuda").requires_grad_() for _ in range(2))
    got = policy.rms_norm(x, residual=r)
    (got.out.sum() + got.sum.square().sum()).backward()
    assert torch.equal(x.grad, r.grad) and x.grad.shape == shape
    before = r.grad.clone()
    x.grad.zero_()
    assert torch.equal(r.grad, before)
