"""Performance cases of the policy operators.

What a trainer runs around the environments' steps, through the entry points
it calls (puffysics_amd.policy): the advantages of a rollout, the log
probabilities and entropies of the taken actions with their gradient, and the
optimiser's step over the policy's tensors.  Where `own` is false the same
operators are computed in their plain form, elementary torch operations in
32 bits on the same inputs.

Kinds of case:
  log_probs   `rows` distributions over `actions` choices.  "train" runs the
              backward pass too and returns the logits' gradient; "masked"
              passes the allowed actions (and has rows that allow none and
              rows that are padding); "wide" logits are a slice of wider rows.
  advantages  `steps` of `envs` environments, "major" the axis that varies
              slowest.
  adamw       `params` weights in `tensors` tensors, moments in `bits` bits,
              with the clip of the gradients' global norm where `clip` > 0.
"""
import math
import random

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GAMMA, LAMBDA = 0.99, 0.95
LR, BETA1, BETA2, EPS, DECAY = 1e-3, 0.9, 0.999, 1e-8, 0.01
STEP = 100          # steps the optimiser has behind it
SEGMENT = 256       # a tensor's first weight lies at a multiple of this in the trainer's flat buffers
GROUP = 32          # 8-bit moments: values to a scale
SEED = 7            # 8-bit moments: of their rounding


def _lp(name, rows, actions, type, train, masked=False, wide=0, top=0):
    c = {"kind": "log_probs", "rows": rows, "actions": actions, "type": type, "train": train, "masked": masked,
         "wide": wide, "top": top}
    return dict(c, name=name) if name else c


def _adv(name, steps, envs, major, type):
    c = {"kind": "advantages", "steps": steps, "envs": envs, "major": major, "type": type}
    return dict(c, name=name) if name else c


def _adam(name, params, tensors, type, bits, clip):
    c = {"kind": "adamw", "params": params, "tensors": tensors, "type": type, "bits": bits, "clip": clip}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one environment step's answer: the hover batch and its three thrust
        # levels; launches and latency are all of it
        _lp("act_4096x3", 4096, 3, "f32", False),
        # an update's minibatch of the same: 16 steps of the batch
        _lp("update_65536x3", 65536, 3, "f32", True),
        # a wider set of choices of which some are not allowed, odd sizes,
        # the head's logits a slice of a fused output
        _lp("masked_8191x1021", 8191, 1021, "bf16", True, masked=True, wide=1040),
        # a few answers over a large vocabulary with their best alternatives
        _lp("answer_16x131072", 16, 131072, "bf16", False, top=20),
        # the update of a token policy
        _lp("tokens_4096x131072", 4096, 131072, "bf16", True),
        # rollouts of the hover batch, step after step, and of many more
        # environments with values from a 16-bit head
        _adv("rollout_128x4096", 128, 4096, "steps", "f32"),
        _adv("rollout_500x65537", 500, 65537, "steps", "bf16"),
        # three long episodes, each contiguous
        _adv("long_200003x3", 200003, 3, "envs", "f32"),
        # a policy of a few small layers: launches and latency
        _adam("policy_5k", 5_000, 8, "f32", 32, 0.5),
        # 16-bit weights with their 32-bit copies, many odd tensors
        _adam("mixed_30m", 30_000_003, 120, "bf16", 32, 1.0),
        # moments in 8 bits
        _adam("moments8_200m", 200_000_000, 150, "f32", 8, 0.0),
        # the largest in 32 bits, with the clip
        _adam("full_400m", 400_000_000, 200, "f32", 32, 1.0),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["log_probs", "log_probs", "advantages", "adamw"])
    if kind == "log_probs":
        actions = _spread(rng, 2, 262144)
        rows = _spread(rng, 1, max(1, min(262144, 2 ** 28 // actions)))
        return _lp(None, rows, actions, rng.choice(["f32", "f16", "bf16", "bf16"]), rng.random() < 0.5,
                   rng.random() < 0.4, rng.choice([0, 0, actions + rng.randrange(1, 40)]),
                   rng.choice([0, 0, min(actions, rng.randrange(1, 33))]))
    if kind == "advantages":
        envs = _spread(rng, 1, 65536)
        steps = _spread(rng, 1, max(1, min(400000, 2 ** 25 // envs)))
        return _adv(None, steps, envs, rng.choice(["steps", "envs"]), rng.choice(["f32", "bf16", "f16"]))
    params = _spread(rng, 1000, 300_000_000)
    type = rng.choice(["f32", "f32", "bf16", "f16"])
    return _adam(None, params, _spread(rng, 1, 200), type, rng.choice([8, 32]), rng.choice([0.0, 0.5, 1.0]))


class State:
    pass


def _sizes(case):
    """The tensors' sizes: a few large ones, many small, as layers have them."""
    rng = random.Random(case["params"] * 1000 + case["tensors"])
    n = case["tensors"]
    w = [math.exp(2.0 * rng.gauss(0, 1)) for _ in range(n)]
    total = sum(w)
    sizes = [max(1, int(case["params"] * x / total)) for x in w]
    sizes[sizes.index(max(sizes))] += case["params"] - sum(sizes)
    return sizes


def _offsets(sizes):
    at, got = 0, []
    for n in sizes:
        got.append(at)
        at += -(-n // SEGMENT) * SEGMENT
    return got, at


def prepare(case, seed):
    s = State()
    s.case = case
    gen = torch.Generator("cuda")
    gen.manual_seed(seed)
    randn = lambda *shape, dtype=torch.float32: torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)  # noqa: E731
    rand = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    if case["kind"] == "log_probs":
        return _prepare_log_probs(s, case, gen, randn, rand)
    if case["kind"] == "advantages":
        t, n = case["steps"], case["envs"]
        shape = (t, n) if case["major"] == "steps" else (n, t)
        turn = (lambda x: x) if case["major"] == "steps" else (lambda x: x.t())
        # the hover task's rewards lie in [-1, 1]; an episode ends after 64 steps at the mean
        s.rewards = turn(2.0 * rand(*shape) - 1.0)
        s.values = turn((3.0 * randn(*shape)).to(DTYPE[case["type"]]))
        s.terminals = turn((rand(*shape) < 1.0 / 64.0).to(torch.float32))
        s.last = (3.0 * randn(n)).to(DTYPE[case["type"]])
        return s
    return _prepare_adamw(s, case, randn)


def _prepare_log_probs(s, case, gen, randn, rand):
    r, v, dtype = case["rows"], case["actions"], DTYPE[case["type"]]
    width = case["wide"] or v
    # rows from nearly even to sharp
    logits = randn(r, width, dtype=dtype)
    logits.mul_((0.5 + 3.5 * rand(r, 1)).to(dtype))
    s.logits = logits[:, :v]
    # taken: half the likeliest action, half any
    s.taken = torch.where(rand(r) < 0.5, s.logits.argmax(-1), torch.randint(0, v, (r,), generator=gen, device="cuda"))
    s.mask = None
    if case["masked"]:
        s.mask = rand(r, v) < 0.7
        s.mask.scatter_(1, s.taken[:, None], True)
        s.mask[rand(r) < 0.01] = False            # finished: no action left
        s.taken[rand(r) < 0.05] = -1              # padding
    s.d_log_prob = s.d_entropy = None
    if case["train"]:
        s.d_log_prob = randn(r) / r               # advantages over the batch
        s.d_entropy = torch.full((r,), -0.01 / r, device="cuda")
        s.logits.requires_grad_(True)
    return s


def _prepare_adamw(s, case, randn):
    dtype, bits = DTYPE[case["type"]], case["bits"]
    s.sizes = _sizes(case)
    s.offsets, total = _offsets(s.sizes)

    def flat(scale, dtype=torch.float32):
        x = randn(total, dtype=dtype).mul_(scale)
        for at, n in zip(s.offsets, s.sizes):
            x[at + n:at + -(-n // SEGMENT) * SEGMENT] = 0
        return x

    s.master = flat(0.02)
    s.param = s.master if dtype == torch.float32 else s.master.to(dtype)
    s.grad = flat(1e-3, dtype)
    s.exp_avg = flat(3e-4)
    s.exp_avg_sq = flat(1.0).square_().add_(0.1).mul_(1e-6)
    for at, n in zip(s.offsets, s.sizes):
        s.exp_avg_sq[at + n:at + -(-n // SEGMENT) * SEGMENT] = 0
    if bits == 8:
        s.exp_avg, s.exp_avg_sq = _to_8_bits(s.exp_avg, 0, 0), _to_8_bits(s.exp_avg_sq.sqrt(), 0, 1).square()
    s.step = STEP
    s.params = [s.param[at:at + n] for at, n in zip(s.offsets, s.sizes)]
    s.grads = [s.grad[at:at + n] for at, n in zip(s.offsets, s.sizes)]
    if own:      # the handle that a trainer makes once, with the moments it resumes from
        from puffysics_amd import policy
        s.optimizer = policy.AdamW(s.params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=bits,
                                   max_grad_norm=case["clip"] or None, seed=SEED)
        cut = lambda x: [x[at:at + n] for at, n in zip(s.offsets, s.sizes)]  # noqa: E731
        s.optimizer.load_moments(cut(s.exp_avg), cut(s.exp_avg_sq), step=STEP,
                                 master=None if dtype == torch.float32 else cut(s.master))
    return s


def run(s):
    kind = s.case["kind"]
    if kind == "log_probs":
        return (_own_log_probs if own else _plain_log_probs)(s)
    if kind == "advantages":
        if own:
            from puffysics_amd import policy
            adv, ret = policy.advantages(s.rewards, s.values, s.terminals, s.last, GAMMA, LAMBDA)
        else:
            adv, ret = _plain_advantages(s)
        return {"advantages": adv, "returns": ret}
    return (_own_adamw if own else _plain_adamw)(s)


def _own_log_probs(s):
    from puffysics_amd import policy
    top = s.case["top"]
    got = policy.log_probs(s.logits, s.taken, mask=s.mask, top=top)
    out = {"log_prob": got.log_prob.detach(), "entropy": got.entropy.detach()}
    if top:
        out.update(top_log_prob=got.top_log_prob, top_action=got.top_action)
    if s.case["train"]:
        out["d_logits"], = torch.autograd.grad((got.log_prob, got.entropy), s.logits, (s.d_log_prob, s.d_entropy))
    return out


@torch.no_grad()
def _plain_log_probs(s):
    x = s.logits.float()
    if s.mask is not None:
        x = torch.where(s.mask, x, -math.inf)
    most = x.amax(-1, keepdim=True)
    none = most == -math.inf
    z = x - torch.where(none, 0.0, most)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    z = z - torch.log(total)                                     # log probabilities
    z = torch.where(none, -math.inf, z)
    entropy = -torch.where(e > 0, e * z, 0.0).sum(-1) / torch.where(none, 1.0, total)[:, 0]
    pad = s.taken < 0
    log_prob = torch.where(pad, 0.0, z.gather(1, s.taken.clamp(min=0)[:, None])[:, 0])
    out = {"log_prob": log_prob, "entropy": entropy}
    if s.case["top"]:
        # ties go to the lowest index: one whole number that orders by value, then by index
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
        index = torch.arange(x.shape[1], device=x.device)
        top = torch.topk(order * (1 << 20) + ((1 << 20) - 1 - index), s.case["top"], dim=-1).values
        out["top_action"] = (1 << 20) - 1 - (top & ((1 << 20) - 1))
        out["top_log_prob"] = z.gather(1, out["top_action"])
    if s.case["train"]:
        p = torch.where(none, 0.0, e / total)
        d = torch.where(pad, 0.0, s.d_log_prob)[:, None]
        inner = torch.where(e > 0, z + entropy[:, None], 0.0).mul_(s.d_entropy[:, None]).add_(d)
        g = p.mul_(inner).neg_()
        at = s.taken.clamp(min=0)[:, None]
        allowed = x.gather(1, at) > -math.inf
        g.scatter_add_(1, at, torch.where(allowed, d, 0.0))
        out["d_logits"] = g.to(s.logits.dtype)
    return out


def _plain_advantages(s):
    values = s.values.float()
    after = torch.cat([values[1:], s.last.float()[None]])
    go = s.terminals == 0
    b = s.rewards + torch.where(go, GAMMA * after, 0.0) - values
    a = torch.where(go, GAMMA * LAMBDA, 0.0)
    # x -> a x + b, composed over 1, 2, 4 .. later steps
    span = 1
    while span < b.shape[0]:
        b = torch.cat([b[:-span] + a[:-span] * b[span:], b[-span:]])
        a = torch.cat([a[:-span] * a[span:], a[-span:]])
        span *= 2
    return b, b + values


def _own_adamw(s):
    norm = s.optimizer.step(s.grads)
    exp_avg, exp_avg_sq = s.optimizer.moments()
    out = {"param": s.param, "exp_avg": exp_avg, "exp_avg_sq": exp_avg_sq}
    if s.master is not s.param:
        out["master"] = s.optimizer.master()
    if norm is not None:
        out["norm"] = norm
    return out


def _plain_adamw(s):
    out = {}
    s.step += 1
    g = s.grad.float()
    if s.case["clip"]:
        out["norm"] = g.square().sum().sqrt()
        g = g * torch.clamp(s.case["clip"] / (out["norm"] + 1e-6), max=1.0)
    m = s.exp_avg * BETA1 + g * (1 - BETA1)
    v = s.exp_avg_sq * BETA2 + g * g * (1 - BETA2)
    root = v.sqrt()
    update = m * (LR / (1 - BETA1 ** s.step)) / (root * (1 / math.sqrt(1 - BETA2 ** s.step)) + EPS)
    s.master.mul_(1 - LR * DECAY).sub_(update)
    if s.master is not s.param:
        s.param.copy_(s.master)
        out["master"] = s.master
    if s.case["bits"] == 8:
        s.exp_avg, s.exp_avg_sq = _to_8_bits(m, s.step, 0), _to_8_bits(root, s.step, 1).square()
        # four significant bits, squared: both are exact in bf16
        out["exp_avg"], out["exp_avg_sq"] = s.exp_avg.bfloat16(), s.exp_avg_sq.bfloat16()
    else:
        s.exp_avg, s.exp_avg_sq = m, v
        out["exp_avg"], out["exp_avg_sq"] = m, v
    out["param"] = s.param
    return out


def _mix(x):
    """32 well mixed bits of a 32-bit number."""
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _to_8_bits(x, step, half):
    """The values that e4m3 numbers with one power of two for every 32 of
    them stand for: the least power with which none passes 448.  x is rounded
    to one of its two neighbours by 16 random bits, the low (half 0: first
    moments) or the high (half 1: roots of second moments) half of a number
    that the step and the place in the flat buffer give.  To the nearest, a
    second moment that changes by a thousandth a step would never change at
    all.  A root over 0 stays over 0, since the update divides by it."""
    key = _mix((step * 0x9e3779b9 + SEED) & 0xffffffff)
    random_bits = (_mix(torch.arange(x.numel(), device=x.device) ^ key) >> (16 * half)) & 0xffff
    x = x.view(-1, GROUP)
    fraction, power = torch.frexp(x.abs().amax(-1, keepdim=True))      # fraction in [0.5, 1)
    power = (power - 9 + (fraction > 0.875)).clamp(-126, 127)
    y = torch.ldexp(x.abs(), -power)
    low = torch.where(y < 2.0 ** -6, 2.0 ** -6, 0.0)                   # below it the steps stay 2^-9
    z = (y + low).view(torch.int32) + (random_bits.view_as(y) << 4).int()
    z = (z & ~0xfffff).view(torch.float32) - low
    if half:
        z = torch.where(y > 0, z.clamp(min=2.0 ** -9), z)
    return torch.copysign(torch.ldexp(z, power), x).view(-1)


def work(case):
    size = 4 if case.get("type") == "f32" else 2
    if case["kind"] == "log_probs":
        r, v = case["rows"], case["actions"]
        n = r * v
        bytes = n * (size + (1 if case["masked"] else 0)) + r * (8 + 4 + 4 + 12 * case["top"])
        flops = n * 5
        if case["train"]:
            bytes += n * size + r * 8
            flops += n * 6
        return {"bytes": bytes, "flops": flops}
    if case["kind"] == "advantages":
        n = case["steps"] * case["envs"]
        return {"bytes": n * (4 + size + 4 + 8) + case["envs"] * size, "flops": n * 8}
    n = case["params"]
    weight = 2 * size + (8 if size == 2 else 0) + size               # weights in and out, their 32-bit copies, gradients
    moments = 16 if case["bits"] == 32 else 4 + 4 / GROUP + 4         # read and written; 8 bits: read out as bf16 as well
    return {"bytes": n * (weight + moments), "flops": n * 16}


def exact(case, seed):
    """The definitions in 64 bits."""
    s = prepare(case, seed)
    return {"log_probs": _exact_log_probs, "advantages": _exact_advantages, "adamw": _exact_adamw}[case["kind"]](s, case)


@torch.no_grad()
def _exact_log_probs(s, case):
    r, v = case["rows"], case["actions"]
    out = {"log_prob": torch.zeros(r, dtype=torch.float64, device="cuda"), "entropy": torch.zeros(r, dtype=torch.float64, device="cuda")}
    if case["top"]:
        out["top_action"], out["top_log_prob"] = None, torch.zeros(r, case["top"], dtype=torch.float64, device="cuda")
    if case["train"]:
        out["d_logits"] = torch.zeros(r, v, dtype=torch.float64, device="cuda")
    part = max(1, 2 ** 26 // v)
    for lo in range(0, r, part):
        at = slice(lo, min(r, lo + part))
        x = s.logits[at].double()
        if s.mask is not None:
            x = x.masked_fill(~s.mask[at], -math.inf)
        lp = x - torch.logsumexp(x, -1, keepdim=True)
        lp = lp.nan_to_num(nan=-math.inf, posinf=-math.inf, neginf=-math.inf)      # rows that allow nothing
        p = lp.exp()
        h = -(p * lp.clamp(min=-1e300)).sum(-1)
        taken = s.taken[at]
        out["log_prob"][at] = torch.where(taken < 0, 0.0, lp.gather(1, taken.clamp(min=0)[:, None])[:, 0])
        out["entropy"][at] = h
        if case["top"]:
            out["top_log_prob"][at] = lp.sort(-1, descending=True).values[:, :case["top"]]
        if case["train"]:
            dl, dh = s.d_log_prob[at].double()[:, None], s.d_entropy[at].double()[:, None]
            dl = torch.where((taken < 0)[:, None], 0.0, dl)
            one = torch.zeros_like(p).scatter_(1, taken.clamp(min=0)[:, None], 1.0)
            one = torch.where(lp > -math.inf, one, 0.0)
            out["d_logits"][at] = dl * (one - p) - dh * p * (lp.clamp(min=-1e300) + h[:, None])
    return out


def _exact_advantages(s, case):
    values, go = s.values.double(), (s.terminals == 0).double()
    after = torch.cat([values[1:], s.last.double()[None]])
    delta = s.rewards.double() + GAMMA * go * after - values
    if case["steps"] > 20000:            # as one long sum: step after step on the host
        delta, go = delta.cpu().numpy(), go.cpu().numpy()
        if delta.shape[1] > 64:
            return None
        adv, run_ = delta.copy(), delta[-1].copy()
        for t in range(delta.shape[0] - 2, -1, -1):
            run_ = delta[t] + GAMMA * LAMBDA * go[t] * run_
            adv[t] = run_
        adv = torch.from_numpy(adv).cuda()
    else:
        adv = delta.clone()
        for t in range(delta.shape[0] - 2, -1, -1):
            adv[t].addcmul_(go[t], adv[t + 1], value=GAMMA * LAMBDA)
    return {"advantages": adv, "returns": adv + values}


def _exact_adamw(s, case):
    out = {}
    t = STEP + 1
    g = s.grad.double()
    if case["clip"]:
        out["norm"] = torch.linalg.vector_norm(g)
        g = g * min(1.0, case["clip"] / (float(out["norm"]) + 1e-6))
    m = torch.lerp(g, s.exp_avg.double(), BETA1)
    v = torch.lerp(g * g, s.exp_avg_sq.double(), BETA2)
    p = s.master.double() * (1 - LR * DECAY) - LR * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    out["param"] = p
    if s.master is not s.param:
        out["master"] = p
    out["exp_avg"], out["exp_avg_sq"] = m, v
    if case["bits"] == 8:
        for half, (name, x) in enumerate((("exp_avg", m), ("exp_avg_sq", v.sqrt()))):
            at = torch.arange(x.numel(), dtype=torch.int64, device="cuda")
            h = ((t * 2654435769 + SEED) % 2 ** 32)
            for by, k in ((16, 0x7feb352d), (15, 0x846ca68b), (16, 1)):
                h = (h ^ (h >> by)) * k % 2 ** 32
            h = at.bitwise_xor_(h)
            for by, k in ((16, 0x7feb352d), (15, 0x846ca68b), (16, 1)):
                h = (h ^ (h >> by)).mul_(k).bitwise_and_(2 ** 32 - 1)
            u = ((h >> 16 if half else h) % 2 ** 16).double().div_(2 ** 16).view(-1, GROUP)
            x = x.view(-1, GROUP)
            power = torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True).clamp(min=1e-38) / 448.0))
            y = x.abs() / torch.exp2(power)
            # e4m3: steps of 1/8 of the power of two below, 2^-9 at the least
            grain = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
            y = torch.floor(y / grain + u) * grain
            if half:
                y = torch.where(x > 0, y.clamp(min=2.0 ** -9), y)
            y = y * torch.exp2(power)
            out[name] = (y * y if half else torch.copysign(y, x)).view(-1)
    return out
