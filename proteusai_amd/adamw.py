"""AdamW on HIP kernels: a step over all tensors in few launches, moments in 32 bits or in 8, and the optimizer around it.

The reference trains with torch.optim.AdamW (utils/train_utils/training_run.py:75-210); AdamW stands in its place with its first five arguments.
"""
import ctypes

import torch

from . import _lib
from .grad_clip import _TYPES, _bound, _dense, grad_norm

ROW, CODES, GROUP = 1056, 512, 32                           # bytes and elements of a row of 8-bit moments (PROTEUS_ADAMW_ROW), elements of a scale


def adamw_(params, grads, exp_avgs, exp_avg_sqs, step, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, masters=None, norm=None, max_norm=None):
    """One AdamW step on lists of tensors, in place:

        m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2;   p = p (1 - lr weight_decay) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    Parameters are fp32, bf16 or fp16, mixed or not, all on one GPU, dense in any order; gradients of the same shapes, fp32 or (with fp32 parameters: any of the three) the parameter's type; the moments
    fp32, of the parameters' shapes and strides.  16-bit parameters are updated in fp32 and rounded once, to the nearest; masters (a list of fp32 tensors, None where a parameter has none) holds
    the weights that they are rounded from, without which updates below half a step of theirs are lost.

    step: t, the number of this step, from 1 on, or an int64 tensor of one element on the GPU with the number of steps done, to which the call adds one; lr: a number or an fp32 tensor of one
    element on the GPU.  What a captured call reads of these tensors is what they hold when it is replayed; a number is the same in every replay.  norm (an fp32 tensor of one element on the GPU, as grad_norm returns it) and
    max_norm: the gradients count as multiplied by min(1, max_norm / (norm + 1e-6)), as clip_grad_norm_ would leave them; they are not written.  Nothing synchronises with the device
    and nothing is recorded for a backward.  Tensors that are written must not share memory with one another or with a gradient: that is refused."""
    _step(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), step, lr, betas, eps, weight_decay, masters, norm, max_norm, 0)


def adamw8_(params, grads, states, step, *, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, masters=None, norm=None, max_norm=None, seed=0):
    """adamw_ with both moments in 8 bits: states[i] is what adamw8_state(params[i]) returns, of which adamw8_moments gives the values.

    A moment is an e4m3 number times a power of two for each 32 elements; of the second its root is kept.  They are rounded stochastically (a decay of 0.1 % would be lost to
    rounding to nearest), by a hash of `seed` (its lower 32 bits), the step, the tensor's place in the list and the element's in the tensor: the same call gives the same bits.  The parameters are
    updated from the moments as they were before they are rounded."""
    _step(list(params), list(grads), list(states), None, step, lr, betas, eps, weight_decay, masters, norm, max_norm, seed)


def adamw8_state(param):
    """Moments of zero for a parameter: uint8 rows of 1056 bytes, one for each 512 of its elements in the order of its memory: 512 codes of the first moment, 512 of the root of the
    second, 16 scales (a power of two, biased by 127) of the first, 16 of the second."""
    return torch.zeros(-(-param.numel() // CODES), ROW, dtype=torch.uint8, device=param.device)


def adamw8_moments(param, state):
    """(exp_avg, exp_avg_sq): what `state` stands for, fp32 tensors like `param`."""
    if state.dtype != torch.uint8 or tuple(state.shape) != (-(-param.numel() // CODES), ROW):
        raise AssertionError(f"the state of {param.numel()} elements is uint8 of shape ({-(-param.numel() // CODES)}, {ROW}), not {state.dtype} of {tuple(state.shape)}")
    like = _dense(param.detach())

    def values(codes, scales):
        codes = codes.contiguous().view(torch.float8_e4m3fn).float().view(-1, CODES // GROUP, GROUP)
        flat = torch.ldexp(codes, scales.int()[:, :, None] - 127).view(-1)[:param.numel()]
        return torch.as_strided(flat, like.shape, like.stride())
    return (values(state[:, :CODES], state[:, 2 * CODES:2 * CODES + 16]), values(state[:, CODES:2 * CODES], state[:, 2 * CODES + 16:]).square())


def _betas(betas):
    b1, b2 = betas
    b1, b2 = float(b1), float(b2)
    if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
        raise ValueError(f"betas must be at least 0 and below 1, not {b1} and {b2}")
    return b1, b2


def _not_negative(name, x):
    x = float(x)
    if not x >= 0.0:
        raise ValueError(f"{name} must not be negative, but is {x}")
    return x


def _step(params, grads, firsts, seconds, step, lr, betas, eps, weight_decay, masters, norm, max_norm, seed):
    b1, b2 = _betas(betas)
    eps, weight_decay, seed = _not_negative("eps", eps), _not_negative("weight_decay", weight_decay), int(seed) & 0xffffffff
    if not isinstance(lr, torch.Tensor):
        lr = _not_negative("lr", lr)
    if not isinstance(step, torch.Tensor):
        step = int(step)
        if not 1 <= step < 1 << 63:
            raise ValueError(f"step is the number of this step, from 1 on, not {step}")
    if (norm is None) != (max_norm is None):
        raise ValueError("norm and max_norm go together")
    max_norm = 0.0 if max_norm is None else _bound(max_norm)
    masters = None if masters is None else list(masters)
    n = len(params)
    if len(grads) != n or len(firsts) != n or (seconds is not None and len(seconds) != n) or (masters is not None and len(masters) != n):
        raise AssertionError(f"there must be a tensor for each of the {n} parameters in every list")
    args = params, grads, firsts, seconds, masters, step, lr, b1, b2, eps, weight_decay, norm, max_norm, seed
    rc = _lib.ops().adamw(*args)
    if rc is None:
        _general(*args)
    else:
        _lib.check(rc, "proteus_adamw")


def _scalar(t, name, dtype, dev):
    if t.dtype != dtype or t.numel() != 1 or t.device != dev or t.layout != torch.strided:
        raise ValueError(f"{name} must be a tensor of one {dtype} on {dev}, not {tuple(t.shape)} of {t.dtype} on {t.device}")
    return t


@torch.no_grad()
def _general(params, grads, firsts, seconds, masters, step, lr, b1, b2, eps, weight_decay, norm, max_norm, seed):
    """What is not plain: what is wrong is refused, gradients that lie otherwise than their parameters are copied."""
    written = [t for t in [*params, *firsts, *(seconds or ()), *(masters or ()), *([step] if isinstance(step, torch.Tensor) else [])] if t is not None]
    for t in [*written, *grads]:
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided:
            raise NotImplementedError(f"AdamW takes dense tensors, not {t.layout if isinstance(t, torch.Tensor) else type(t)}")
    if not params and not isinstance(step, torch.Tensor):
        return
    dev = params[0].device if params else step.device
    for t in [*written, *grads]:
        if not t.is_cuda or t.device != dev:
            raise _lib.ProteusError("an AdamW step needs tensors on the GPU, all on one (there is no CPU path)")
        if not torch._C._has_storage(t):
            raise NotImplementedError("tensors without memory of their own (under a functional transform) have no AdamW step here")
    for t in written:
        if t.is_inference() and not torch.is_inference_mode_enabled():
            raise RuntimeError("a tensor made in inference mode is not written outside of it")
    src = []
    for i, (p, g) in enumerate(zip(params, grads)):
        if p.dtype not in _TYPES or g.dtype not in _TYPES or (p.dtype != torch.float32 and g.dtype not in (p.dtype, torch.float32)):
            raise NotImplementedError(f"parameters are float32, bfloat16 or float16 with gradients in float32 or (float32 parameters: any of these) their own type, not {p.dtype} with {g.dtype}")
        if g.shape != p.shape:
            raise AssertionError(f"a gradient of shape {tuple(g.shape)} does not go with a parameter of shape {tuple(p.shape)}")
        if _dense(p) is not p:
            raise ValueError("a parameter must fill a stretch of memory")
        like = [(seconds is not None and firsts[i], "exp_avg"), (seconds is not None and seconds[i], "exp_avg_sq"), (masters and masters[i] is not None and masters[i], "a master weight")]
        for t, name in like:
            if isinstance(t, torch.Tensor) and (t.dtype != torch.float32 or t.shape != p.shape or (t.stride() != p.stride() and p.numel() > 0)):
                raise ValueError(f"{name} must be float32 of its parameter's shape and strides, {tuple(p.shape)} and {p.stride()}, not {t.dtype} of {tuple(t.shape)} and {t.stride()}")
        if masters and masters[i] is not None and p.dtype == torch.float32:
            raise ValueError("a float32 parameter has no master weight")
        if seconds is None and (firsts[i].dtype != torch.uint8 or tuple(firsts[i].shape) != (-(-p.numel() // CODES), ROW) or not firsts[i].is_contiguous()):
            raise ValueError(f"the state of {p.numel()} elements is dense uint8 of shape ({-(-p.numel() // CODES)}, {ROW}), not {firsts[i].dtype} of {tuple(firsts[i].shape)}")
        src.append(g if g.stride() == p.stride() and _dense(g) is g else torch.empty_like(p, dtype=g.dtype).copy_(g))
    spans = [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), w) for ts, w in ((written, 1), ([*src, *(t for t in (lr, norm) if isinstance(t, torch.Tensor))], 0)) for t in ts if t.numel()]
    ends = {0: 0, 1: 0}
    for begin, end, w in sorted(spans):
        if begin < ends[1] or (w and begin < ends[0]):
            raise ValueError("tensors that an AdamW step writes must not share memory with one another or with a gradient")
        ends[w] = max(ends[w], end)
    n = len(params)
    a = _lib.AdamwArgs(count=n, beta1=b1, beta2=b2, eps=eps, weight_decay=weight_decay, max_norm=max_norm, seed=seed)

    def pointers(tensors):
        return (ctypes.c_void_p * n)(*[None if t is None else t.data_ptr() for t in tensors])
    a.params, a.grads = pointers(params), pointers(src)
    a.masters = None if masters is None else pointers(masters)
    if seconds is None:
        a.states = pointers(firsts)
    else:
        a.exp_avgs, a.exp_avg_sqs = pointers(firsts), pointers(seconds)
    a.numel = (ctypes.c_int64 * n)(*[t.numel() for t in params])
    a.param_types, a.grad_types = (ctypes.c_int * n)(*[_TYPES[t.dtype] for t in params]), (ctypes.c_int * n)(*[_TYPES[t.dtype] for t in src])
    if isinstance(lr, torch.Tensor):
        a.lr_gpu = _scalar(lr, "lr", torch.float32, dev).data_ptr()
    else:
        a.lr = lr
    if isinstance(step, torch.Tensor):
        a.step_gpu = _scalar(step, "step", torch.int64, dev).data_ptr()
    else:
        a.step = step
    if norm is not None:
        a.norm = _scalar(norm, "norm", torch.float32, dev).data_ptr()
    with _lib.on_device(dev):
        rc = _lib.load().proteus_adamw(ctypes.byref(a), _lib.raw_stream(dev))
    if rc >= 0:                                             # (one that failed after its first launch has written, too)
        for t in written:
            if not t.is_inference():
                torch.autograd.graph.increment_version(t)
    _lib.check(rc, "proteus_adamw")


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW on the kernels, a few launches a step.  fp32, bf16 and fp16 parameters on one GPU.

    bits: 32, or 8 for moments in 8 bits (adamw8_).  master_weights: 16-bit parameters are rounded from fp32 weights kept beside them.  max_norm: gradients count as clipped to this norm, as
    clip_grad_norm_ would over all parameters of the optimizer, in one pass over them more (self.norm holds the norm, a tensor on the GPU).  capturable: the number of steps lies on the GPU, one for
    a parameter group, whose parameters have gradients together from the first step on; such a step can be captured into a graph once one has run outside of it (without it that is refused).  lr may be an
    fp32 tensor of one element on the GPU, which a schedule fills; a rate that is a number stays what it was when the step was captured.  What torch's has beyond that (amsgrad, maximize, foreach, fused, differentiable) is not taken.

    The state of a parameter: "exp_avg" and "exp_avg_sq" in fp32 like it, or "moments", which adamw8_moments reads; "master" in fp32; "step", the number of its steps (a capturable group has its own
    "steps").  state_dict and load_state_dict keep all of these in their types."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, bits=32, master_weights=False, max_norm=None, capturable=False, seed=0):
        if bits not in (8, 32):
            raise ValueError(f"bits must be 32 or 8, not {bits}")
        _betas(betas)
        for name, x in (("eps", eps), ("weight_decay", weight_decay), ("lr", 0.0 if isinstance(lr, torch.Tensor) else lr)):
            _not_negative(name, x)
        self.bits, self.master_weights, self.capturable, self.seed = bits, bool(master_weights), bool(capturable), int(seed)
        self.max_norm = None if max_norm is None else _bound(max_norm)
        self.norm = None
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):
        return {**super().__getstate__(), **{k: getattr(self, k) for k in ("bits", "master_weights", "capturable", "seed", "max_norm", "norm")}}

    def _begin(self, p, group):
        if not p.is_cuda:
            raise _lib.ProteusError("AdamW needs parameters on the GPU (there is no CPU path)")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first step of a parameter makes its state: it cannot be captured into a graph")
        s = self.state[p]
        if self.bits == 8:
            s["moments"] = adamw8_state(p)
        else:
            s["exp_avg"], s["exp_avg_sq"] = (torch.zeros_like(p, dtype=torch.float32) for _ in range(2))
        if self.master_weights and p.dtype != torch.float32:
            s["master"] = p.detach().float()
        if not self.capturable:
            s["step"] = 0
        elif "steps" not in group:
            group["steps"] = torch.zeros((), dtype=torch.int64, device=p.device)

    @torch.no_grad()
    def step(self, closure=None):
        # (a captured step is launched with the numbers that it has now: every replay would be the same step once more)
        if not self.capturable and torch.cuda.is_initialized() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a step of AdamW is captured into a graph only with capturable=True, where the number of steps lies on the GPU and replays count it")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        new = []
        for group in self.param_groups:
            params = [p for p in group["params"] if p.grad is not None]
            begun = [id(p) for p in group["params"] if p in self.state]
            if self.capturable and "steps" in group and params and begun != [id(p) for p in params]:
                raise RuntimeError("the parameters of a capturable group have gradients together from the first step on: put those that begin later or are left out at times into a group of their own")
            new += [(p, group) for p in params if p not in self.state]
        for p, group in new:
            self._begin(p, group)
        jobs = []
        for i, group in enumerate(self.param_groups):
            params = [p for p in group["params"] if p.grad is not None]
            if not params:
                continue
            if self.capturable:
                jobs.append((i, group, params, group["steps"]))
                continue
            by_step = {}
            for p in params:
                by_step.setdefault(self.state[p]["step"] + 1, []).append(p)
            jobs += [(i, group, some, step) for step, some in by_step.items()]
        self.norm = grad_norm([p.grad for _, _, params, _ in jobs for p in params]) if self.max_norm is not None and jobs else None
        for i, group, params, step in jobs:
            states = [self.state[p] for p in params]
            # (a group has rounding of its own)
            how = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"], norm=self.norm, max_norm=self.max_norm,
                       masters=[s.get("master") for s in states] if self.master_weights else None)
            grads = [p.grad for p in params]
            if self.bits == 8:
                adamw8_(params, grads, [s["moments"] for s in states], step, seed=self.seed + 0x632be5ab * i, **how)
            else:
                adamw_(params, grads, [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], step, **how)
            if not self.capturable:
                for s in states:
                    s["step"] = step
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch's, but the state keeps its types: moments of 16-bit parameters stay what they were.  What torch.optim.AdamW saved is taken where this optimizer keeps the same (bits=32, no master weights, not
        capturable), its moments in fp32.  Tensors that the optimizer has already, its rate's among them, are filled: a step captured before, and a schedule that fills the rate, go on with what was loaded.  (One rate
        tensor of several groups whose saved rates differ, and tensors that the saved state has no counterpart of, are given up: such a step has to be captured again.)"""
        saved = state_dict["state"]
        params = [p for g in self.param_groups for p in g["params"]]
        places = [i for g in state_dict["param_groups"] for i in g["params"]]
        names = {"moments"} if self.bits == 8 else {"exp_avg", "exp_avg_sq"}
        for i, p in zip(places, params):
            if i in saved and (not names <= set(saved[i]) or (self.capturable == ("step" in saved[i])) or ("master" in saved[i]) != (self.master_weights and p.dtype != torch.float32)):
                raise ValueError(f"this optimizer keeps {', '.join(sorted(names))} of a parameter (bits={self.bits}, master_weights={self.master_weights}, capturable={self.capturable}): the saved state holds {', '.join(sorted(saved[i]))}")
        if any(g.get("amsgrad") or g.get("maximize") for g in state_dict["param_groups"]):
            raise ValueError("a state of amsgrad or maximize has no continuation here")
        states, groups = {p: dict(self.state[p]) for p in params if p in self.state}, [dict(g) for g in self.param_groups]
        super().load_state_dict(state_dict)
        for i, p in zip(places, params):
            for k, v in saved.get(i, {}).items():
                if k == "step":
                    self.state[p][k] = int(v)
                elif isinstance(v, torch.Tensor):
                    v = v.float() if k in ("exp_avg", "exp_avg_sq") else v
                    like = torch.empty_like(p, dtype=v.dtype, device="meta") if v.shape == p.shape else torch.empty(v.shape, dtype=v.dtype, device="meta")
                    self.state[p][k] = _filled(states.get(p, {}).get(k), v, like, p.device)
        for name, dtype in (("steps", torch.int64), ("lr", torch.float32)):
            wanted = {}                                     # of each tensor there is, what the groups would have in it
            for g, old in zip(self.param_groups, groups):
                wanted.setdefault(id(old.get(name)), set()).add(float(g.get(name, 0)))
            for g, old in zip(self.param_groups, groups):
                v, had = g.get(name), old.get(name)
                if v is None or not g["params"] or not (isinstance(v, torch.Tensor) or isinstance(had, torch.Tensor)):
                    continue
                v, dev = (int if dtype == torch.int64 else float)(v), g["params"][0].device
                same = isinstance(had, torch.Tensor) and had.dtype == dtype and had.device == dev and len(wanted[id(had)]) == 1
                g[name] = had.fill_(v) if same else torch.full((), v, dtype=dtype, device=dev)


def _filled(had, values, like, device):
    """The values in the tensor that there is, where that is one like `like` on the device, else in a new one."""
    if not (isinstance(had, torch.Tensor) and had.device == device and had.dtype == like.dtype and had.shape == like.shape and had.stride() == like.stride()):
        had = torch.empty_strided(like.shape, like.stride(), dtype=like.dtype, device=device)
    return had.copy_(values)
