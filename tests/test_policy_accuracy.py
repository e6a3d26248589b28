"""How exact puffysics_amd.policy is, against the definitions in 64 bits,
with bounds of the summations that the kernels make.

u = 2^-24 is half a unit in the last place.  Log probabilities: a term exp(z)
is off by |z| (u of the rounded argument, half a u of the rounded log2 e) and
by 2 u of the exponential.  A lane adds at most 32 terms one after the other
and a wave's lanes 6 times; waves (at most 4) and pieces (4 to a lane, then 6
times) are joined by a product with another exponential, 5 u each.  So S is
off by (N + 2 E|z|) u of itself with N = 45 in rows of up to 2,048 actions, 60
up to 8,192 and 120 beyond, E over the row's probabilities.  The logarithm is
good to 2 u of its value, the differences to u of theirs.  The entropy's terms
are z exp(z): the same errors times |z|.

AdamW's norm: a thread adds 16 rounded squares in 32 bits, 17 u of the sum,
the rest is in 64; half of that after the root and u of the result: 10 u.  The
clip's factor then has two more roundings, a clipped gradient one more (14 u),
and a moment is two products of rounded rates and a sum."""
import numpy as np
import pytest
import torch

from policytest import adamw_oracle, log_probs_gradient_oracle, log_probs_oracle

U = 2.0 ** -24


def bounds(x, taken):
    """(log probability's, entropy's, every log probability's) bounds."""
    actions = x.shape[1]
    n = 45 if actions <= 2048 else 60 if actions <= 8192 else 120
    *_, lp = log_probs_oracle(x, taken)
    p, z = np.exp(lp), x - x.max(1, keepdims=True)
    log_s = (z - lp)[:, :1]
    e1, e2 = (p * np.abs(z)).sum(1, keepdims=True), (p * z * z).sum(1, keepdims=True)
    of_s = (n + 2 * e1) * U + 2 * U * log_s
    every = of_s + U * (np.abs(z) + np.abs(lp) + log_s)
    h = of_s + ((n + 8) * e1 + 2 * e2) * U + 2 * U * (log_s + e1)
    return np.take_along_axis(every, taken[:, None], 1)[:, 0], h[:, 0], every


@pytest.mark.gpu
@pytest.mark.parametrize("scale,shift", [(3.0, 0.0), (0.2, 0.0), (3.0, 1000.0), (3.0, -1e6)])
@pytest.mark.parametrize("actions", [1, 2, 3, 17, 64, 257, 1000, 1025, 2048, 2049, 4097, 8192, 8193, 65536, 100003, 262144])
def test_log_probs(actions, scale, shift):
    from puffysics_amd import policy
    rows = max(2, min(300, 200000 // actions))
    g = torch.Generator().manual_seed(actions)
    x = (torch.randn(rows, actions, generator=g) * scale + shift).cuda().requires_grad_()
    taken = torch.randint(0, actions, (rows,), generator=g)
    dl, dh = torch.randn(rows, generator=g), torch.randn(rows, generator=g)
    got = policy.log_probs(x, taken.cuda())
    d, = torch.autograd.grad(got[:2], x, (dl.cuda(), dh.cuda()))
    f64 = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    xs, ts, dl, dh = f64(x), taken.numpy(), f64(dl), f64(dh)
    lp, h, _, _, every = log_probs_oracle(xs, ts)
    of_lp, of_h, of_every = bounds(xs, ts)
    assert (np.abs(f64(got.log_prob) - lp) <= of_lp).all()
    assert (np.abs(f64(got.entropy) - h) <= of_h).all()
    # p is off by the log probability's error and the exponential's own; the
    # bracket by its terms' errors and roundings, the difference by one more
    want, p = log_probs_gradient_oracle(xs, ts, None, dl, dh), np.exp(every)
    inner = np.abs(dl[:, None] + dh[:, None] * (every + h[:, None]))
    of_p = of_every + 4 * U + 2 * U * np.abs(every)
    of_inner = np.abs(dh)[:, None] * (of_every + of_h[:, None] + 2 * U * np.abs(every + h[:, None])) + 2 * U * inner
    one = np.zeros_like(p)
    one[np.arange(rows), ts] = np.abs(dl)
    tol = p * (inner * of_p + of_inner) + U * (one + p * inner + np.abs(want)) + 1e-44
    assert (np.abs(f64(d) - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", [[1], [5, 300], [4096] * 3, [70001, 4097, 3], [3_000_000], [999] * 200])
def test_norm_and_clipped_moments(sizes):
    from puffysics_amd import policy
    lr, betas, eps, most = 0.01, (0.9, 0.999), 1e-8, 0.7
    g = torch.Generator().manual_seed(len(sizes))
    params = [torch.randn(n, generator=g).cuda() for n in sizes]
    opt = policy.AdamW(params, lr, betas, eps, 0.0, max_grad_norm=most)
    old = [(np.zeros(n), np.zeros(n)) for n in sizes]
    for t in range(1, 4):
        grads = [torch.randn(n, generator=g).cuda() for n in sizes]
        flat = np.concatenate([x.double().cpu().numpy() for x in grads])
        want = np.sqrt((flat ** 2).sum())
        norm = float(opt.step(grads))
        assert abs(norm - want) <= 10 * U * want
        clip = min(1.0, most / (want + 1e-6))
        m, v = (x.double().cpu().numpy() for x in opt.moments())
        for i, n in enumerate(sizes):
            at, (m0, v0) = opt.offsets[i], old[i]
            gc = grads[i].double().cpu().numpy()
            _, wm, wv = adamw_oracle(np.zeros(n), gc, m0, v0, t, lr, *betas, eps, 0.0, clip)
            gc = np.abs(gc) * clip
            gm, gv = m[at:at + n], v[at:at + n]
            assert (np.abs(gm - wm) <= U * (4 * betas[0] * np.abs(m0) + 18 * (1 - betas[0]) * gc)).all()
            assert (np.abs(gv - wv) <= U * (4 * betas[1] * v0 + 34 * (1 - betas[1]) * gc * gc) + 1e-45).all()
            old[i] = (gm, gv)
