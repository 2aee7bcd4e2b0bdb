"""The norm over all gradients of a training step and their clipping, two launches of HIP kernels whatever the number of tensors.

The reference clips between backward and optimizer with torch.nn.utils.clip_grad_norm_ (utils/train_utils/training_run_utils.py:97-169); clip_grad_norm_
stands in its place with its first four arguments: the same formula, from squares and sums in 64 bits.  What it does not take: `foreach`, norms other than 1, 2 and infinity, gradients on
several devices, gradients that share memory (clip_grad_norm_ of torch's scales them twice).
"""
import ctypes
import math

import torch

from . import _lib

_TYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_NORMS = {1.0: _lib.NORM_1, 2.0: _lib.NORM_2, math.inf: _lib.NORM_INF}


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False):
    """torch.nn.utils.clip_grad_norm_: the norm over the gradients of `parameters` (a tensor or an iterable of tensors; those without a gradient are left
    out), which are multiplied in place by min(1, max_norm / (norm + 1e-6)).  Returns the norm, an fp32 tensor of one element on their device.

    Gradients: fp32, bf16 or fp16, mixed or not, all on one GPU.  norm_type: 1, 2 or infinity.  Where the norm is within the bound nothing is written.  Nothing
    synchronises with the device unless error_if_nonfinite (which then takes the norm in a pass of its own, and raises before anything is scaled).  Gradients that share
    memory are refused, and tensors made in inference mode outside of it; nothing is recorded for a backward.
    """
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    parameters = list(parameters)
    kind, max_norm = _norm_type(norm_type), _bound(max_norm)
    if not error_if_nonfinite:
        norm = _lib.ops().clip(parameters, True, parameters, kind, max_norm)
        if norm is not None:
            return norm
    grads = [p.grad for p in parameters if p.grad is not None]
    return _clip(grads, grads, kind, max_norm, error_if_nonfinite)


def clip_grad_norm(grads, max_norm: float, norm_type: float = 2.0, out=None, error_if_nonfinite: bool = False):
    """(norm, clipped): the norm over the tensors `grads` and all of them multiplied by min(1, max_norm / (norm + 1e-6)), in `out`, tensors of the same shapes in fp32,
    bf16 or fp16 (made like `grads` where None; `grads` themselves: in place), none of which shares memory with another or with another's gradient.  For gradients that an
    optimizer wants elsewhere or in another type than they were summed in.  Otherwise as clip_grad_norm_."""
    grads = list(grads)
    out = [torch.empty_like(g) for g in grads] if out is None else list(out)
    kind, max_norm = _norm_type(norm_type), _bound(max_norm)
    if len(out) != len(grads):
        raise AssertionError(f"out must have a tensor for each of the {len(grads)} gradients, not {len(out)}")
    if not error_if_nonfinite:
        norm = _lib.ops().clip(grads, False, out, kind, max_norm)
        if norm is not None:
            return norm, out
    return _clip(grads, out, kind, max_norm, error_if_nonfinite), out


def grad_norm(grads, norm_type: float = 2.0, error_if_nonfinite: bool = False):
    """The norm over all elements of the tensors `grads`, as clip_grad_norm_ takes it."""
    grads, kind = list(grads), _norm_type(norm_type)
    norm = _lib.ops().clip(grads, False, None, kind, 0.0)
    if norm is None:
        return _clip(grads, None, kind, 0.0, error_if_nonfinite)
    return _finite(norm) if error_if_nonfinite else norm


def _norm_type(norm_type):
    kind = _NORMS.get(float(norm_type))
    if kind is None:
        raise NotImplementedError(f"norm_type must be 1, 2 or infinity, not {norm_type}")
    return kind


def _bound(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, but is {max_norm}")
    return max_norm


def _finite(norm):
    if not math.isfinite(norm.item()):
        raise RuntimeError(f"the norm of the gradients is {norm.item()}, so they cannot be clipped; to scale them all the same leave error_if_nonfinite at False")
    return norm


def _dense(t):
    """The tensor itself where its elements fill a stretch of memory in some order, else a copy."""
    return t if torch._C._has_storage(t) and torch.ops.aten.is_non_overlapping_and_dense.default(t) else t.contiguous()


@torch.no_grad()
def _clip(grads, out, kind, max_norm, error_if_nonfinite):
    """What is not plain: what is wrong is refused, what is not dense (or `out` in another order than its gradient) goes through copies."""
    if not grads:
        return torch.tensor(0.0)
    for t in [*grads, *(out or ())]:
        if not isinstance(t, torch.Tensor) or t.layout != torch.strided or t.dtype not in _TYPES:
            raise NotImplementedError(f"gradients must be dense float32, bfloat16 or float16 tensors, not {t.dtype if isinstance(t, torch.Tensor) else type(t)}")
        if not t.is_cuda or t.device != grads[0].device:
            raise _lib.ProteusError("the norm of gradients needs tensors on the GPU, all on one (there is no CPU path)")
        if not torch._C._has_storage(t):
            raise NotImplementedError("gradients without memory of their own (under a functional transform) have no norm here")
    for o in out or ():
        if o.is_inference() and not torch.is_inference_mode_enabled():
            raise RuntimeError("a tensor made in inference mode is not written outside of it: clip a clone")
    for g, o in zip(grads, out or ()):
        if o.shape != g.shape:
            raise AssertionError(f"a gradient of shape {tuple(g.shape)} does not go into a tensor of shape {tuple(o.shape)}")
    dev = grads[0].device
    src = [_dense(g) for g in grads]
    dst = back = None
    if out is not None:
        dst, back = [], []
        for g, s, o in zip(grads, src, out):
            if o is g:
                dst.append(s)
            elif o.stride() == s.stride() and _dense(o) is o:
                dst.append(o)
            else:
                dst.append(torch.empty_like(s, dtype=o.dtype))
            if dst[-1] is not o:
                back.append((o, dst[-1]))
    with _lib.on_device(dev):
        if error_if_nonfinite:
            _finite(_launch(src, None, kind, 0.0))
        norm = _launch(src, dst, kind, max_norm)
        for o, d in back or ():
            o.copy_(d)
    return norm


def _launch(src, dst, kind, max_norm):
    if dst is not None:
        def span(t, written):
            return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), written
        # (a gradient scaled in place is written where it is read, by the same threads; another pair's reading of it is not)
        spans = [span(d, 1) for d in dst if d.numel()] + [span(s, 0) for s, d in zip(src, dst) if s.numel() and span(s, 0) != span(d, 0)]
        ends = {0: 0, 1: 0}
        for begin, end, w in sorted(spans):
            if begin < ends[1] or (w and begin < ends[0]):
                raise ValueError("gradients that are scaled must not share memory with one another")
            ends[w] = max(ends[w], end)
    n, dev = len(src), src[0].device
    norm = torch.empty((), dtype=torch.float32, device=dev)
    lib = _lib.load()
    nbytes = lib.proteus_clip_grads_workspace_bytes(n)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)

    def ints(values, of=ctypes.c_int):
        return (of * n)(*values)
    rc = lib.proteus_clip_grads(ints([t.data_ptr() for t in src], ctypes.c_void_p), None if dst is None else ints([t.data_ptr() for t in dst], ctypes.c_void_p),
                                ints([t.numel() for t in src], ctypes.c_int64), ints([_TYPES[t.dtype] for t in src]), None if dst is None else ints([_TYPES[t.dtype] for t in dst]),
                                n, kind, max_norm, norm.data_ptr(), ws.data_ptr(), nbytes, _lib.raw_stream(dev))
    _lib.check(rc, "proteus_clip_grads")
    for t in dst or ():
        if not t.is_inference():
            torch.autograd.graph.increment_version(t)
    return norm
