"""Oracles of the operators of a policy with memory (include/b3_policy.h): the
definitions in 64 bits, with torch, on the device of their arguments."""
import torch

STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}      # half a step of rounding


def attention_oracle(q, k, v, decay, state=None, starts=None, scale=1.0):
    """(out, state after every step [steps, ...]); what an episode's start
    drops is not multiplied by 0."""
    q, k, v, decay = q.double(), k.double(), v.double(), decay.double()[:, None, None]
    steps = q.shape[0]
    s = torch.zeros(*q.shape[1:], v.shape[-1], dtype=torch.float64, device=q.device) if state is None else state.double()
    out, states = torch.zeros(v.shape, dtype=torch.float64, device=q.device), []
    for t in range(steps):
        s = decay * s
        if starts is not None:
            s = torch.where((starts[t] != 0)[:, None, None, None], 0.0, s)
        s = s + k[t][..., :, None] * v[t][..., None, :]
        states.append(s)
        out[t] = scale * (q[t][..., :, None] * s).sum(-2)
    return out, states


def attention_gradient_oracle(q, k, v, decay, state, starts, scale, d_out, d_last=None):
    """(dq, dk, dv, dstate)"""
    _, states = attention_oracle(q, k, v, decay, state, starts, scale)
    q, k, v, d_out, by = q.double(), k.double(), v.double(), d_out.double(), decay.double()[:, None, None]
    g = torch.zeros(*q.shape[1:], v.shape[-1], dtype=torch.float64, device=q.device) if d_last is None else d_last.double()
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for t in range(q.shape[0] - 1, -1, -1):
        g = g + scale * q[t][..., :, None] * d_out[t][..., None, :]
        dq[t] = scale * (states[t] * d_out[t][..., None, :]).sum(-1)
        dk[t] = (g * v[t][..., None, :]).sum(-1)
        dv[t] = (g * k[t][..., :, None]).sum(-2)
        g = by * g
        if starts is not None:
            g = torch.where((starts[t] != 0)[:, None, None, None], 0.0, g)
    return dq, dk, dv, g


def norm_oracle(x, weight, residual, eps):
    """(out, sum, 1 / root mean square)"""
    h = x.double() if residual is None else x.double() + residual.double()
    s = 1.0 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return h * s * (1.0 if weight is None else weight.double()), h, s


def norm_gradient_oracle(h, weight, eps, d_out, d_sum=None):
    """(dh, dweight) of the sum h."""
    h, d = h.double(), d_out.double()
    s = 1.0 / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    w = 1.0 if weight is None else weight.double()
    dh = s * (w * d - h * s * s * (w * d * h).mean(-1, keepdim=True))
    if d_sum is not None:
        dh = dh + d_sum.double()
    return dh, (d * h * s).reshape(-1, h.shape[-1]).sum(0)


def eight_bits_oracle(y):
    """(e4m3 values, powers of two) of rows: the least power with which none of
    32 passes 448, each rounded to the nearest, to the even of two."""
    y = y.double()
    rows, width = y.shape
    z = torch.nn.functional.pad(y, (0, -width % 32)).view(rows, -1, 32)
    power = torch.ceil(torch.log2(z.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -126) / 448.0)).clamp(min=-126)
    z = z / torch.exp2(power)
    grain = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)
    return ((z / grain).round() * grain).view(rows, -1)[:, :width], power.view(rows, -1)


def orthogonalised_oracle(u, steps=5, eps=1e-7):
    """What Muon's steps make of u."""
    x = u.double()
    turned = x.shape[0] > x.shape[1]
    x = x.t() if turned else x
    x = x / (x.square().sum().sqrt() + eps)
    for _ in range(steps):
        y = x @ x.t()
        x = 3.4445 * x + (-4.7750 * y + 2.0315 * (y @ y)) @ x
    return x.t() if turned else x
