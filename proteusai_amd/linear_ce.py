"""Softmax cross entropy over a vocabulary straight from features, on HIP kernels: loss and gradients without the logits in memory.

The reference puts torch's cross entropy behind a linear head (utils/train_utils/losses.py); linear_cross_entropy is both in one, for heads of a few words and of many.
"""
import ctypes

import torch
import torch.nn.functional as F

from . import _lib, train_ops

_TYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_REDUCTIONS = {"none": _lib.CE_NONE, "mean": _lib.CE_MEAN, "sum": _lib.CE_SUM}


def cleaned(values, target, words, ignore_index):
    """(values, target) for torch's cross entropy of values [..., n] (features, or logits), as the kernels take tokens: zeros for those that are left out, whose target becomes -100 (torch multiplies what
    lies there by 0), NaN for those whose target is no word, which becomes 0 (on the GPU torch reads at whatever place a target names)."""
    left_out = target == ignore_index
    no_word = ~left_out & ((target < 0) | (target >= words))
    nothing = torch.zeros_like(target, dtype=values.dtype).masked_fill(no_word, float("nan"))          # (a where of two numbers would copy them to the GPU, which no captured graph can hold)
    values = values.masked_fill(left_out[..., None], 0.0) + nothing[..., None]
    return values, target.masked_fill(left_out, -100).masked_fill(no_word, 0)


def _expression(x, weight, bias, target, ignore_index, label_smoothing, reduction):
    x, words = cleaned(x, target, weight.shape[0], ignore_index)
    logits = F.linear(x, weight, bias).float()
    loss = F.cross_entropy(logits.reshape(-1, logits.shape[-1]), words.reshape(-1), label_smoothing=label_smoothing, reduction=reduction)
    return loss.view(target.shape) if reduction == "none" else loss


def _args(x, weight, bias, target, ignore_index, label_smoothing, reduction):
    d = weight.shape[1]
    return _lib.CeArgs(x=x.data_ptr(), weight=weight.data_ptr(), bias=None if bias is None else bias.data_ptr(), target=target.data_ptr(), ignore_index=ignore_index, rows=x.numel() // d, d=d,
                       vocab=weight.shape[0], dtype=_TYPES[x.dtype], reduction=reduction, label_smoothing=label_smoothing)


def _forward(x, weight, bias, target, how, keep):
    """(loss, what the backward reads) of dense tensors."""
    lib, dev = _lib.load(), x.device
    a = _args(x, weight, bias, target, *how)
    n = lib.proteus_linear_ce_fwd_bytes(ctypes.byref(a))
    _lib.check(lib.proteus_linear_ce_check(ctypes.byref(a)), "proteus_linear_ce_check")
    loss = torch.empty(target.shape if how[2] == _lib.CE_NONE else (), dtype=torch.float32, device=dev)
    kept_bytes = lib.proteus_linear_ce_kept_bytes(ctypes.byref(a)) if keep else 0
    kept = train_ops._workspace(kept_bytes, dev)
    train_ops._call("proteus_linear_ce_fwd", dev, ctypes.byref(a), loss, kept, kept_bytes, train_ops._workspace(n, dev), n)
    return loss, kept


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, how):
        dense = [None if t is None else train_ops._dense(t) for t in (x, weight, bias, target)]
        loss, kept = _forward(*dense, how, True)
        ctx.save_for_backward(x, weight, bias, target, kept)
        ctx.how = how
        return loss

    @staticmethod
    def backward(ctx, d):
        return (*_backward(ctx.saved_tensors, d, ctx.how, ctx.needs_input_grad[:3]), None, None)


def _general_backward(saved, d, ignore_index, label_smoothing, reduction, need):
    """What the C++ path's backward does not take."""
    return _backward(saved, d, (ignore_index, label_smoothing, reduction), need)


@train_ops._without_autocast
def _backward(saved, d, how, need):
    """Gradients of x, weight, bias, whatever form the tensors come in."""
    x, weight, bias, target, kept = saved
    if d is None:
        return (None,) * 3
    if train_ops._by_expression(d):
        inputs = [(p, n) for p, n in zip((x, weight, bias), need) if p is not None]
        with torch.enable_grad():
            # (each a tensor of its own: one that stands in two places has a gradient for each)
            given = [p.view_as(p) for p, _ in inputs]

        def expr(x_, weight_, bias_=None):
            return _expression(x_, weight_, bias_, target, how[0], how[1], {v: k for k, v in _REDUCTIONS.items()}[how[2]])
        got = iter(train_ops._recorded(expr, given, [n for _, n in inputs], d))
        return tuple(None if p is None else next(got) for p in (x, weight, bias))
    dev, dtype, lib = weight.device, weight.dtype, _lib.load()
    V, D = weight.shape
    rows = x.numel() // D
    xs, ws = train_ops._saved(x, rows * D, dev, dtype), train_ops._saved(weight, V * D, dev, dtype)
    bs = None if bias is None else train_ops._saved(bias, V, dev, dtype)
    ts = train_ops._saved(target, rows, dev, torch.int64)
    a = _args(xs, ws, bs, ts, *how)
    kept_bytes = lib.proteus_linear_ce_kept_bytes(ctypes.byref(a))
    ks = train_ops._saved(kept, kept_bytes, dev, torch.uint8)
    if d.dtype != torch.float32 or d.device != dev or d.numel() != (rows if how[2] == _lib.CE_NONE else 1):
        raise RuntimeError(f"the gradient of the loss is {tuple(d.shape)} of {d.dtype} on {d.device}")
    grads = [torch.empty(t.shape, dtype=dtype, device=dev) if t is not None and n else None for t, n in zip((x, weight, bias), need)]
    n = lib.proteus_linear_ce_bwd_bytes(ctypes.byref(a))
    train_ops._call("proteus_linear_ce_bwd", dev, ctypes.byref(a), d.contiguous(), ks, kept_bytes, *grads, train_ops._workspace(n, dev), n)
    return tuple(grads)


def linear_cross_entropy(x, weight, target, bias=None, *, ignore_index: int = -100, label_smoothing: float = 0.0, reduction: str = "mean"):
    """torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, weight, bias), target, ...) for features x [..., d], weight [vocab, d], bias [vocab] or None and targets [...] (int64, words'
    numbers), without the logits in memory: the forward keeps 16 bytes a token (up to 64 words: 4 for each of them), the backward makes the logits again, a piece of the vocabulary at a time, and holds their
    gradient for it: 2 bytes a logit (fp32: 6), up to 1 GB or, if that is more, for 2048 words of all tokens, so that with few words and very many tokens it takes as much as logits would.  The loss is fp32, whatever the
    features' type: [...] (reduction "none"; zero where the target is ignore_index), their sum ("sum"), or the mean over the tokens that are not left out ("mean"; NaN if there is none).

    fp32, bf16 or fp16, all tensors alike on one GPU, d a multiple of 8 (fp32: 4) up to 65536, at most 2^24 tokens and words.  Sums are fp32; the logits' gradient is rounded to the tensors' type (up to 64 tokens, left out or not, to twice its bits), as which the gradients'
    products read it.  Features of tokens that are left out are not read.  Above 64 words the products leave them out: with one token in seven they cost a seventh, beside what goes over the weights whatever the tokens.  A target that is neither a word nor ignore_index gives a NaN loss, as does a token all of whose logits are -infinity.
    Under autocast, functional transforms, forward-mode differentiation or tracing the torch expression is taken, as it is by a backward that is itself recorded: the same numbers and tokens left out, with the logits in memory.
    """
    ignore_index, label_smoothing = int(ignore_index), float(label_smoothing)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(_REDUCTIONS)}, not {reduction}")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"label_smoothing must be between 0 and 1, not {label_smoothing}")
    how = ignore_index, label_smoothing, _REDUCTIONS[reduction]
    loss = _lib.ops().linear_ce(x, weight, bias, target, *how)
    if loss is not None:
        return loss
    if x.dim() < 1 or weight.dim() != 2 or x.shape[-1] != weight.shape[1]:
        raise AssertionError(f"weight must be of shape (vocab, {x.shape[-1] if x.dim() else '?'}), not {tuple(weight.shape)}")
    if target.shape != x.shape[:-1]:
        raise AssertionError(f"target must be of shape {tuple(x.shape[:-1])}, not {tuple(target.shape)}")
    if bias is not None and bias.shape != weight.shape[:1]:
        raise AssertionError(f"bias must be of shape ({weight.shape[0]},), not {tuple(bias.shape)}")
    if target.dtype != torch.int64:
        raise NotImplementedError(f"targets are words' numbers in int64, not {target.dtype}")
    given = [t for t in (x, weight, bias) if t is not None]
    if not x.is_cuda or any(t.device != x.device for t in (*given, target)):
        raise _lib.ProteusError("linear_cross_entropy needs tensors on the GPU, all on one (there is no CPU path)")
    if weight.shape[0] == 0 and target.numel() > 0:
        raise ValueError("a vocabulary of no words has no cross entropy")
    if (torch.is_autocast_enabled("cuda") or not train_ops.unobserved() or x.numel() == 0 or weight.shape[0] == 0 or any(type(t) not in train_ops._PLAIN_TYPES for t in (*given, target))):
        return _expression(x, weight, bias, target, ignore_index, label_smoothing, reduction)
    if x.dtype not in _TYPES or any(t.dtype != x.dtype for t in given):
        raise NotImplementedError("linear_cross_entropy takes float32, bfloat16 or float16 tensors, all alike")
    if any(t.layout != torch.strided for t in (*given, target)):
        raise NotImplementedError("linear_cross_entropy takes dense tensors")
    rows, (V, D) = x.numel() // weight.shape[1], weight.shape
    if D % (4 if x.dtype == torch.float32 else 8) or max(rows, V) > 1 << 24 or D > 1 << 16:
        raise ValueError(f"linear_cross_entropy does not take {rows} rows of {D} features and {V} words in {x.dtype}: features must be a multiple of {4 if x.dtype == torch.float32 else 8} and at most 65536, "
                         f"rows and words at most {1 << 24}")
    if torch.is_grad_enabled() and any(t.requires_grad for t in given):
        return _LinearCrossEntropy.apply(x, weight, bias, target, how)
    return _forward(*[None if t is None else train_ops._dense(t) for t in (x, weight, bias, target)], how, False)[0]
