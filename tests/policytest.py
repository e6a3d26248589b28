"""Oracles of the policy operators (include/b3_policy.h): the definitions in
64 bits, with numpy on the host."""
import numpy as np

EPS32 = 2.0 ** -23


def log_probs_oracle(x, taken, mask=None, top=0):
    """(log_prob, entropy, top_log_prob, top_action, all log probabilities)."""
    x = np.array(x, np.float64)
    if mask is not None:
        x = np.where(np.broadcast_to(mask, x.shape), x, -np.inf)
    rows, actions = x.shape
    with np.errstate(all="ignore"):
        most = x.max(1, keepdims=True)                       # NaN where one is NaN
        none = most[:, 0] == -np.inf
        z = x - np.where(none[:, None], 0.0, most)
        e = np.exp(z)
        lp = z - np.log(e.sum(1, keepdims=True))
        lp[none] = -np.inf
        p = np.exp(lp)
        h = -np.where(p == 0, 0.0, p * lp).sum(1)
        h[none] = 0.0
    got = np.zeros(rows)
    for r in range(rows):
        a = int(taken[r])
        got[r] = 0.0 if a < 0 else np.nan if a >= actions else lp[r, a]
    order = np.zeros((rows, top), np.int64)
    for r in range(rows):
        nan = np.isnan(x[r])
        order[r] = np.lexsort((np.arange(actions), -np.where(nan, np.inf, x[r]), ~nan))[:top]
    return got, h, np.take_along_axis(lp, order, 1), order, lp


def log_probs_gradient_oracle(x, taken, mask, d_log_prob, d_entropy):
    x = np.array(x, np.float64)
    allowed = x > -np.inf if mask is None else (x > -np.inf) & np.broadcast_to(mask, x.shape)
    _, h, _, _, lp = log_probs_oracle(x, taken, mask)
    p = np.exp(lp)
    with np.errstate(all="ignore"):
        inner = np.where(p == 0, 0.0, lp + h[:, None])
    d = -p * (np.where(taken < 0, 0.0, d_log_prob)[:, None] + d_entropy[:, None] * inner)
    for r, a in enumerate(taken):
        if a >= 0:
            d[r, a] += d_log_prob[r]
    return np.where(allowed, d, 0.0)


def advantages_oracle(rewards, values, terminals, last, gamma, lam):
    """[steps, envs] arrays."""
    adv = np.zeros(rewards.shape)
    after, run = np.array(last, np.float64), np.zeros(rewards.shape[1])
    for t in range(rewards.shape[0] - 1, -1, -1):
        v = np.array(values[t], np.float64)
        end = terminals[t] != 0
        run = rewards[t] - v + np.where(end, 0.0, gamma * after + gamma * lam * run)
        adv[t], after = run, v
    return adv, adv + np.array(values, np.float64)


def mix(x):
    """The 32-bit hash of the 8-bit moments' rounding."""
    x = np.array(x, np.uint64)
    for shift, by in ((16, 0x7feb352d), (15, 0x846ca68b), (16, 1)):
        x = ((x ^ (x >> np.uint64(shift))) * np.uint64(by)) & np.uint64(0xffffffff)
    return x


def round_bits(size, t, seed, first=0):
    """The 16 random bits for first moments and for roots, of the places
    first .. first + size - 1 of the flat arrays, as fractions in [0, 1)."""
    key = mix([(t * 0x9e3779b9 + seed) & 0xffffffff])[0]
    h = mix(np.arange(first, first + size, dtype=np.uint64) ^ key)
    return (h & np.uint64(0xffff)).astype(float) / 65536, (h >> np.uint64(16)).astype(float) / 65536


def grid_of(x):
    """(steps of the grid that an 8-bit moment is rounded on, at |x|) for x in
    groups of 32: the e4m3 numbers times the least power of two with which
    none passes 448."""
    x = np.abs(np.array(x, np.float64)).reshape(-1, 32)
    most = x.max(1, keepdims=True)
    power = np.ceil(np.log2(np.maximum(most, 2.0 ** -126) / 448.0))
    power = np.maximum(power, -126.0)
    y = x / 2.0 ** power
    return (2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3 + power)).reshape(-1), \
        np.broadcast_to(2.0 ** (power - 9), x.shape).reshape(-1)


def adamw_oracle(w, g, m, v, t, lr, beta1, beta2, eps, decay, clip=1.0):
    """One step in 64 bits: (w, m, v)."""
    g = np.array(g, np.float64) * clip
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    w = w * (1 - lr * decay) - lr * (m / (1 - beta1 ** t)) / (np.sqrt(v / (1 - beta2 ** t)) + eps)
    return w, m, v
