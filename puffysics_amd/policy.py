"""What a policy's update needs next to the environments' step
(include/b3_policy.h): `advantages` of a rollout, `log_probs` of the taken
actions with entropies, best alternatives and the gradient, and `AdamW`.

The arrays are torch CUDA tensors; the work is enqueued on the current torch
stream and runs in libb3policy.so.  Arguments that do not fit raise
ValueError before anything is launched; an error of a call raises B3Error.
The reference leaves these to the trainer (docs/RL_LIBRARY.md).
"""
import array
import collections
import ctypes as C
import operator
import os

import torch
from torch.autograd import forward_ad

from . import _native
from .engine import B3Error

POLICY_PATH = os.path.join(_native.HERE, "libb3policy.so")
MAX_TOP = 32
MAX_ACTIONS = 1 << 21
MAX_ROWS = (1 << 31) - 1     # and steps and environments of a rollout
SEGMENT = 256
_SMALL = 2048                # rows of up to so many actions need no workspace
_EMPTY = 8                   # stands for the address of a gradient without elements; NULL is no gradient
# what a step asks of every tensor, called by map: a policy may have many small ones
_address, _is_contiguous, _is_neg, _get_device = (
    getattr(torch._C.TensorBase, name) for name in ("data_ptr", "is_contiguous", "is_neg", "get_device"))

_F32, _F16, _BF16, _U8 = 0, 1, 2, 3
_TYPE = {torch.float32: _F32, torch.float16: _F16, torch.bfloat16: _BF16}
_vp, _i, _ll, _d, _sz = C.c_void_p, C.c_int, C.c_int64, C.c_double, C.c_size_t


class B3Logits(C.Structure):
    _fields_ = [("data", _vp), ("type", _i), ("rows", _ll), ("actions", _ll), ("row_stride", _ll), ("mask", _vp),
                ("mask_row_stride", _ll)]


class B3Rollout(C.Structure):
    _fields_ = [("steps", _ll), ("envs", _ll), ("rewards", _vp), ("rewards_stride", _ll * 2), ("values", _vp),
                ("values_type", _i), ("values_stride", _ll * 2), ("last_values", _vp), ("last_values_stride", _ll),
                ("terminals", _vp), ("terminals_type", _i), ("terminals_stride", _ll * 2), ("advantages", _vp),
                ("returns", _vp), ("out_stride", _ll * 2)]


class B3AdamWTensor(C.Structure):
    _fields_ = [("param", _vp), ("type", _i), ("numel", _ll), ("weight_decay", _d)]


class B3AdamWState(C.Structure):
    _fields_ = [("bits", _i), ("exp_avg", _vp), ("exp_avg_sq", _vp), ("exp_avg_scale", _vp),
                ("exp_avg_sq_scale", _vp), ("master", _vp)]


class B3AdamWConfig(C.Structure):
    _fields_ = [("beta1", _d), ("beta2", _d), ("eps", _d), ("seed", C.c_uint32)]


POLICY_SYMBOLS = [
    ("b3_log_probs_workspace", _sz, [_ll, _ll, _i]),
    ("b3_log_probs_gpu", _i, [B3Logits, _vp, _vp, _vp, _vp, _i, _vp, _vp, _vp, _sz, _vp]),
    ("b3_log_probs_backward_gpu", _i, [B3Logits, _vp, _vp, _vp, _vp, _ll, _vp, _ll, _vp, _ll, _vp]),
    ("b3_advantages_workspace", _sz, [_ll, _ll]),
    ("b3_advantages_gpu", _i, [C.POINTER(B3Rollout), _d, _d, _vp, _sz, _vp]),
    ("b3_adamw_size", _ll, [C.POINTER(B3AdamWTensor), _i]),
    ("b3_adamw_create", _i, [C.POINTER(_vp), C.POINTER(B3AdamWTensor), _i, B3AdamWState, B3AdamWConfig]),
    ("b3_adamw_step_gpu", _i, [_vp, _vp, _vp, _d, _d, _vp, _vp]),
    ("b3_adamw_steps", _ll, [_vp, _i]),
    ("b3_adamw_set_steps", _i, [_vp, _i, _ll]),
    ("b3_adamw_moments_gpu", _i, [_vp, _vp, _vp, _vp]),
    ("b3_adamw_load_moments_gpu", _i, [_vp, _vp, _vp, _vp]),
    ("b3_adamw_destroy", _i, [_vp]),
]

_lib = None


def policy_lib():
    """libb3policy.so, loaded once; raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(POLICY_PATH):
            raise RuntimeError("%s is missing: run __graft_entry__.build()" % POLICY_PATH)
        _native._torch_runtime_first()
        lib = C.CDLL(POLICY_PATH)
        for name, res, args in POLICY_SYMBOLS:
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _lib = lib
    return _lib


def _check(name, code):
    if code != 0:
        raise B3Error(name, code)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _stream():
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _on(*tensors):
    """Raise unless all are on the current device, where the work runs."""
    device = -1
    for t in tensors:
        if t is None:
            continue
        at = t.get_device()                  # -1: on the host
        if at >= 0 and device < 0:
            device = torch.cuda.current_device()
        if at != device or at < 0:
            raise ValueError("tensors have to be on the current CUDA device")


def _as_read(x):
    """x, or where its elements are only marked as negated, as those of a
    conjugate's imaginary part are, a copy that holds them so."""
    return x if x is None or not x.is_neg() else x.resolve_neg()


# ---- log probabilities ----

LogProbs = collections.namedtuple("LogProbs", "log_prob entropy top_log_prob top_action")


def _logits(x, mask):
    """B3Logits of x [rows, actions] and a mask [rows or 1, actions]."""
    rows, actions = x.shape
    # the stride of a lone row says nothing
    stride = x.stride(0) if rows > 1 else actions
    if mask is None:
        return B3Logits(x.data_ptr(), _TYPE[x.dtype], rows, actions, stride, None, 0)
    mask_stride = 0 if mask.shape[0] == 1 else mask.stride(0)
    return B3Logits(x.data_ptr(), _TYPE[x.dtype], rows, actions, stride, mask.data_ptr(), mask_stride)


def _rows(x):
    """x, or a copy of it, with contiguous rows that do not overlap."""
    if x.stride(1) == 1 and (x.shape[0] == 1 or x.stride(0) >= x.shape[1]):
        return x
    return x.contiguous()


def _forward(x, taken, mask, top, kept):
    """(log_prob, entropy, top_log_prob, top_action, stats), the last only
    where `kept`."""
    rows, actions = x.shape
    lib = policy_lib()
    log_prob = torch.empty(rows, dtype=torch.float32, device=x.device)
    entropy = torch.empty_like(log_prob)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=x.device) if kept else None
    top_lp = top_action = work = None
    if top:
        top_lp = torch.empty((rows, top), dtype=torch.float32, device=x.device)
        top_action = torch.empty((rows, top), dtype=torch.int64, device=x.device)
    size = 0 if actions <= _SMALL else lib.b3_log_probs_workspace(rows, actions, top)
    if size:
        work = torch.empty(size, dtype=torch.uint8, device=x.device)
    _check("b3_log_probs_gpu", lib.b3_log_probs_gpu(
        _logits(x, mask), taken.data_ptr(), log_prob.data_ptr(), entropy.data_ptr(), stats.data_ptr() if kept else None,
        top, top_lp.data_ptr() if top else None, top_action.data_ptr() if top else None,
        work.data_ptr() if size else None, size, _stream()))
    return log_prob, entropy, top_lp, top_action, stats


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, taken, mask, top):
        x = _rows(x)
        log_prob, entropy, top_lp, top_action, stats = _forward(x, taken, mask, top, True)
        ctx.save_for_backward(x, taken, mask, stats, entropy)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(top_lp, top_action)
        return log_prob, entropy, top_lp, top_action

    @staticmethod
    def backward(ctx, d_log_prob, d_entropy, *_):
        # a gradient that is differentiated again says that it cannot be
        return (_backward_once if torch.is_grad_enabled() else _backward)(ctx, d_log_prob, d_entropy)


def _backward(ctx, d_log_prob, d_entropy):
    x, taken, mask, stats, entropy = ctx.saved_tensors
    d_log_prob, d_entropy = _as_read(d_log_prob), _as_read(d_entropy)
    d = torch.empty_like(x, memory_format=torch.contiguous_format)
    _check("b3_log_probs_backward_gpu", policy_lib().b3_log_probs_backward_gpu(
        _logits(x, mask), taken.data_ptr(), stats.data_ptr(), entropy.data_ptr(), *_upstream(d_log_prob),
        *_upstream(d_entropy), d.data_ptr(), x.shape[1], _stream()))
    return d, None, None, None


_backward_once = torch.autograd.function.once_differentiable(_backward)


def _upstream(d):
    """Pointer and stride of a gradient [rows] (None: zero)."""
    return (None, 0) if d is None else (d.data_ptr(), d.stride(0))


def log_probs(logits, taken, mask=None, top=0):
    """Log probabilities of the actions `taken` under `logits`, as
    LogProbs(log_prob, entropy, top_log_prob, top_action).

    logits  [..., actions], float32, float16 or bfloat16
    taken   [...] whole numbers; below 0 for padding, whose log_prob is 0
    mask    None or bool, [..., actions] or [actions]: the allowed actions
    top     how many of each row's best actions to return (at most 32), by
            descending log probability, the lowest action first among equals

    log_prob and entropy are float32 [...] and differentiable in the logits
    (backward and once; a tangent is refused);
    top_log_prob and top_action are [..., top], or None without `top`.  A row
    that allows nothing has log_prob -inf, entropy 0 and no gradient; an
    action past the last has log_prob NaN."""
    _need(logits.dtype in _TYPE, "logits have to be float32, float16 or bfloat16")
    _need(logits.dim() >= 1 and logits.shape[-1] >= 1, "logits need at least one action")
    _need(not (taken.is_floating_point() or taken.is_complex() or taken.dtype == torch.bool), "taken has to be whole numbers")
    _need(taken.shape == logits.shape[:-1], "taken has to have the shape of logits without the last axis")
    # where a level is entered the tensor may have a tangent
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(logits).tangent is not None:
        raise ValueError("log_probs has no forward-mode derivative")
    actions = logits.shape[-1]
    if actions > MAX_ACTIONS or taken.numel() > MAX_ROWS:
        raise ValueError("at most 2^21 actions and 2^31 - 1 rows")
    _need(0 <= top <= MAX_TOP and top <= actions, "top has to be between 0 and 32, and at most the actions")
    _on(logits, taken, mask)
    if mask is not None:
        _need(mask.dtype == torch.bool, "mask has to be bool")
        _need(mask.shape == logits.shape or mask.shape == (actions,),
              "mask has to have the shape of logits, or of one row")
        mask = _rows(mask.reshape(-1, actions))
    if logits.is_neg():
        logits = _as_read(logits)
    shape = taken.shape
    if len(shape) != 1:
        logits, taken = logits.reshape(-1, actions), taken.reshape(-1)
    if taken.dtype != torch.int64 or not taken.is_contiguous():
        taken = taken.to(torch.int64).contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        log_prob, entropy, top_lp, top_action = _LogProbs.apply(logits, taken, mask, top)
    else:
        log_prob, entropy, top_lp, top_action, _ = _forward(_rows(logits), taken, mask, top, False)
    if len(shape) != 1:
        log_prob, entropy = log_prob.reshape(shape), entropy.reshape(shape)
        if top:
            top_lp, top_action = top_lp.reshape(*shape, top), top_action.reshape(*shape, top)
    return LogProbs(log_prob, entropy, top_lp, top_action)


# ---- advantages ----

def advantages(rewards, values, terminals, last_values, gamma=0.99, lam=0.95):
    """(advantages, returns) of a rollout, both float32 and laid out like the
    rewards: A_t = r_t + gamma V_{t+1} - V_t + gamma lam A_{t+1}, where a
    terminal at t drops what lies after it, and R_t = A_t + V_t.

    rewards      [steps, envs] float32
    values       [steps, envs] float32, float16 or bfloat16: before each step
    terminals    [steps, envs] float32, bool or uint8: nonzero where the step
                 ended an episode (HoverEnvs.terminals)
    last_values  [envs], of values' type: after the last step

    Any strides; the result has no gradient and no tangent."""
    _need(rewards.dim() == 2 and rewards.dtype == torch.float32, "rewards have to be float32 [steps, envs]")
    _need(values.shape == rewards.shape and terminals.shape == rewards.shape,
          "values and terminals have to have the shape of rewards")
    _need(values.dtype in _TYPE, "values have to be float32, float16 or bfloat16")
    _need(last_values.shape == rewards.shape[1:] and last_values.dtype == values.dtype,
          "last_values have to be [envs], of the type of values")
    _need(terminals.dtype in (torch.float32, torch.bool, torch.uint8), "terminals have to be float32, bool or uint8")
    steps, envs = rewards.shape
    if (steps > MAX_ROWS or envs > MAX_ROWS) and rewards.numel():
        raise ValueError("at most 2^31 - 1 steps and environments")
    _need(0 <= gamma <= 1 and 0 <= lam <= 1, "gamma and lam have to be between 0 and 1")
    _on(rewards, values, terminals, last_values)
    if rewards.is_neg() or values.is_neg() or last_values.is_neg():
        rewards, values, last_values = _as_read(rewards), _as_read(values), _as_read(last_values)
    lib = policy_lib()
    # the longer stride is the outer axis: (steps, envs) unless the rewards are a transposed array
    turned = rewards.stride(0) < rewards.stride(1)
    out = torch.empty((2, envs, steps) if turned else (2, steps, envs), dtype=torch.float32, device=rewards.device)
    adv, ret = (out[0].t(), out[1].t()) if turned else (out[0], out[1])
    g = B3Rollout(steps, envs, rewards.data_ptr(), rewards.stride(), values.data_ptr(), _TYPE[values.dtype],
                  values.stride(), last_values.data_ptr(), last_values.stride(0), terminals.data_ptr(),
                  _F32 if terminals.dtype == torch.float32 else _U8, terminals.stride(), adv.data_ptr(), ret.data_ptr(),
                  adv.stride())
    size = lib.b3_advantages_workspace(steps, envs)
    work = torch.empty(size, dtype=torch.uint8, device=rewards.device) if size else None
    _check("b3_advantages_gpu", lib.b3_advantages_gpu(C.byref(g), gamma, lam, work.data_ptr() if size else None, size,
                                                      _stream()))
    return adv, ret


# ---- AdamW ----

class AdamW:
    """AdamW over all of `params` in one step: contiguous float32, float16 or
    bfloat16 tensors on the current device, no two of which overlap.

    state_bits     32, or 8: moments as e4m3 numbers (the first, and the root
                   of the second) with a power of two for every 32 of them,
                   rounded by random bits that `seed`, step and place give
    max_grad_norm  the global norm that gradients are scaled down to, or None
    weight_decay   a number, or one for each tensor
    master         keep 32-bit copies of 16-bit weights and round those; without
                   them small updates of such weights are lost.  A weight that
                   was written between two steps counts, not its copy

    The moments lie in flat arrays, tensor i's from offsets[i] on.  Steps of
    one optimizer follow one another: on several streams, order them.  A step
    that is captured in a graph repeats the bias corrections of its own count
    in every replay; 8-bit moments are rounded by other bits each time."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32,
                 max_grad_norm=None, master=True, seed=0):
        self._h = _vp()
        self.params = list(params)
        n = len(self.params)
        decay = list(weight_decay) if isinstance(weight_decay, (list, tuple)) else [weight_decay] * n
        for p in self.params:
            _need(p.dtype in _TYPE, "parameters have to be float32, float16 or bfloat16")
            _need(p.is_contiguous() and not p.is_neg(), "parameters have to be contiguous, and not marked as negated")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        _need(all(a[1] <= b[0] for a, b in zip(spans, spans[1:])), "a parameter is given twice, or two overlap")
        _on(*self.params)
        _need(len(decay) == n and all(d >= 0 for d in decay), "weight_decay has to be at least 0, one for each tensor")
        _need(0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0, "betas have to be in [0, 1), eps at least 0")
        _need(state_bits in (8, 32), "state_bits has to be 8 or 32")
        _need(max_grad_norm is None or max_grad_norm > 0, "max_grad_norm has to be over 0, or None")
        self.lr, self.max_grad_norm, self.state_bits = lr, max_grad_norm, state_bits
        self.device = torch.device("cuda", torch.cuda.current_device())
        self._lib = policy_lib()
        table = (B3AdamWTensor * max(n, 1))(*[B3AdamWTensor(p.data_ptr(), _TYPE[p.dtype], p.numel(), d)
                                              for p, d in zip(self.params, decay)])
        self.size = self._lib.b3_adamw_size(table, n)
        self.offsets, at = [], 0
        for p in self.params:
            self.offsets.append(at)
            at += -(-p.numel() // SEGMENT) * SEGMENT
        assert at == self.size
        kind = torch.float32 if state_bits == 32 else torch.uint8
        new = lambda count, dtype: torch.zeros(count, dtype=dtype, device=self.device)  # noqa: E731
        self._exp_avg, self._exp_avg_sq = new(self.size, kind), new(self.size, kind)
        scales = self.size // 32 if state_bits == 8 else 0
        self._scale = new((2, scales), torch.uint8).fill_(1)
        self._master = None
        if master and any(p.dtype != torch.float32 for p in self.params):
            self._master = new(self.size, torch.float32)
            self._copy_weights()
        state = B3AdamWState(state_bits, self._exp_avg.data_ptr(), self._exp_avg_sq.data_ptr(),
                             self._scale[0].data_ptr(), self._scale[1].data_ptr(),
                             self._master.data_ptr() if self._master is not None else None)
        self._at, self._shapes, self._dtypes = ([f(p) for p in self.params] for f in (
            torch.Tensor.data_ptr, lambda p: p.shape, lambda p: p.dtype))
        self._empty = any(p.numel() == 0 for p in self.params)
        torch.cuda.current_stream().synchronize()     # the state is ready for a step on any stream
        _check("b3_adamw_create", self._lib.b3_adamw_create(C.byref(self._h), table, n, state,
                                                            B3AdamWConfig(betas[0], betas[1], eps, seed)))

    def _views(self, flat):
        return [flat[at:at + p.numel()].view(p.shape) for at, p in zip(self.offsets, self.params)]

    def _rounded(self):
        """The 16-bit parameters and the views of their copies."""
        return [(p, m) for p, m in zip(self.params, self._views(self._master)) if p.dtype != torch.float32]

    @torch.inference_mode()
    def _copy_weights(self):
        for p, m in self._rounded():
            m.copy_(p)
        self._master_version = self._version()

    @torch.inference_mode()
    def _round_copies(self):
        for p, m in self._rounded():
            p.copy_(m)
        self._master_version = self._version()

    def _version(self):
        """Changes where a program writes to the copies."""
        return None if self._master.is_inference() else self._master._version

    def step(self, grads=None, lr=None):
        """One step by `grads` (one for each parameter, of its type or
        float32, None to leave it out), or by the parameters' own `.grad`.
        Returns the gradients' norm before the clip as a tensor, or None
        without max_grad_norm."""
        if grads is None:
            grads = [p.grad for p in self.params]
        _need(len(grads) == len(self.params), "need one gradient for each parameter")
        lr = self.lr if lr is None else lr
        _need(lr >= 0, "lr has to be at least 0")
        _need(self.max_grad_norm is None or self.max_grad_norm > 0, "max_grad_norm has to be over 0, or None")
        if list(map(_address, self.params)) != self._at:
            raise ValueError("a parameter's memory is not where it was")
        stepped, shapes, dtypes, given = self.params, self._shapes, self._dtypes, grads
        with_grad = [i for i, g in enumerate(grads) if g is not None]
        if len(with_grad) < len(grads):
            stepped, shapes, dtypes, given = ([x[i] for i in with_grad] for x in (stepped, shapes, dtypes, grads))
        if any(map(_is_neg, given)):
            grads = [_as_read(g) for g in grads]
            given = [g for g in grads if g is not None]
        if not set(map(_get_device, given)) <= {torch.cuda.current_device()}:
            raise ValueError("gradients have to be on the current CUDA device")
        if [g.shape for g in given] != shapes or not all(map(_is_contiguous, given)):
            raise ValueError("gradients have to be contiguous, of the parameters' shapes")
        types = [g.dtype for g in given]
        if types != dtypes and any([t is not d and t is not torch.float32 for t, d in zip(types, dtypes)]):
            raise ValueError("gradients have to be of the parameters' type or float32")
        if len(given) == len(grads) and not self._empty:
            pointers = array.array("Q", list(map(_address, grads)))
        else:
            pointers = array.array("Q", [0 if g is None else g.data_ptr() or _EMPTY for g in grads])
        kinds = None if types == dtypes else \
            array.array("i", [_TYPE[d if g is None else g.dtype] for g, d in zip(grads, self._dtypes)])
        if self._master is not None and self._version() != self._master_version:
            self._round_copies()
        norm = torch.empty((), dtype=torch.float32, device=self.device) if self.max_grad_norm is not None else None
        _check("b3_adamw_step_gpu", self._lib.b3_adamw_step_gpu(
            self._h, pointers.buffer_info()[0], kinds.buffer_info()[0] if kinds else None,
            lr, self.max_grad_norm or 0.0,
            norm.data_ptr() if norm is not None else None, _stream()))
        torch.autograd.graph.increment_version(stepped)      # as an operation in place does
        return norm

    def moments(self):
        """The flat arrays (exp_avg, exp_avg_sq): the state's own in 32 bits,
        in 8 bits the values it stands for as new bfloat16 arrays, which hold
        them exactly but for what lies below their range."""
        if self.state_bits == 32:
            return self._exp_avg, self._exp_avg_sq
        out = torch.empty((2, self.size), dtype=torch.bfloat16, device=self.device)
        _check("b3_adamw_moments_gpu", self._lib.b3_adamw_moments_gpu(self._h, out[0].data_ptr(), out[1].data_ptr(),
                                                                      _stream()))
        return out[0], out[1]

    def master(self):
        """The flat array of 32-bit copies of 16-bit weights (the places of
        32-bit weights hold nothing), or None.  What is written there is what
        the next step goes on from."""
        return self._master

    def steps(self, i=0):
        """Steps that parameter i has taken."""
        return self._lib.b3_adamw_steps(self._h, i)

    def load_moments(self, exp_avg, exp_avg_sq, step, master=None):
        """Go on from moments (lists of a tensor for each parameter) after
        `step` steps, a number or a list of one for each parameter.  Where
        32-bit copies of the weights are given, 16-bit weights become what
        these round to; else the copies are the weights."""
        n = len(self.params)
        _need(len(exp_avg) == n and len(exp_avg_sq) == n and (master is None or len(master) == n),
              "need one tensor for each parameter")
        counts = list(step) if isinstance(step, (list, tuple)) else [step] * n
        _need(len(counts) == n and all(hasattr(k, "__index__") and 0 <= k < 2 ** 63 for k in counts),
              "step has to be a whole number from 0 on, or a list of one for each parameter")
        _need(master is None or self._master is not None, "this optimizer keeps no 32-bit copies")
        for given in (exp_avg, exp_avg_sq, master or []):
            _need(all(x.shape == p.shape for x, p in zip(given, self.params)), "need tensors of the parameters' shapes")
        flat = (self._exp_avg, self._exp_avg_sq) if self.state_bits == 32 else \
            torch.zeros((2, self.size), dtype=torch.float32, device=self.device)
        lists = [(flat[0], exp_avg), (flat[1], exp_avg_sq)] + ([(self._master, master)] if master is not None else [])
        for to, given in lists:
            for view, x in zip(self._views(to), given):
                view.copy_(x)
        if self.state_bits == 8:
            _check("b3_adamw_load_moments_gpu", self._lib.b3_adamw_load_moments_gpu(
                self._h, flat[0].data_ptr(), flat[1].data_ptr(), _stream()))
        if master is not None:
            self._round_copies()
        elif self._master is not None:
            self._copy_weights()
        for i, k in enumerate(counts):
            _check("b3_adamw_set_steps", self._lib.b3_adamw_set_steps(self._h, i, operator.index(k)))

    def close(self):
        if self._h:
            code = self._lib.b3_adamw_destroy(self._h)
            self._h = _vp()
            _check("b3_adamw_destroy", code)

    def __del__(self):
        try:
            if getattr(self, "_h", None):
                self._lib.b3_adamw_destroy(self._h)
                self._h = _vp()
        except Exception:
            pass
