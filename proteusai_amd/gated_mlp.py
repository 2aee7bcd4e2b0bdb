"""Gated feed-forward block on HIP kernels: (act(x Wg' + bg) * (x Wu' + bu)) Wo' + bo, forward and backward.

The gated counterpart of the encoder's MLP (utils/model_utils/base_modules/base_modules.py:6-52; encoder.MLP), which the reference does not have.
"""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import _lib, train_ops

_ACTS = {"silu": 0, "gelu": 1, "relu": 2, "sigmoid": 3}        # PROTEUS_ACT_*
_FUNCTIONS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu, "sigmoid": torch.sigmoid}
_TYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


def _expression(x, w_in, b_in, w_out, b_out, act):
    gate, value = F.linear(x, w_in, b_in).chunk(2, -1)
    return F.linear(_FUNCTIONS[act](gate) * value, w_out, b_out)


class _GatedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_in, b_in, w_out, b_out, act):
        xc = train_ops._dense(x)
        params = [None if p is None else train_ops._dense(p) for p in (w_in, b_in, w_out, b_out)]
        y, kept = _forward(xc, params, act, True)
        ctx.save_for_backward(x, w_in, b_in, w_out, b_out, kept)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, d):
        return (*_backward(ctx.saved_tensors, d, ctx.act, ctx.needs_input_grad[:5]), None)


def _general_backward(saved, d, act, need):
    """What the C++ path's backward does not take (its activation's number)."""
    return _backward(saved, d, list(_ACTS)[act], need)


@train_ops._without_autocast
def _backward(saved, d, act, need):
    """Gradients of x, w_in, b_in, w_out, b_out, whatever form the tensors come in."""
    x, w_in, b_in, w_out, b_out, kept = saved
    params = (w_in, b_in, w_out, b_out)
    if d is None:
        return (None,) * 5
    if train_ops._by_expression(d):
        inputs = [(p, n) for p, n in zip((x, *params), need) if p is not None]
        with torch.enable_grad():
            # (each a tensor of its own: one that stands in two places has a gradient for each)
            given = [p.view_as(p) for p, _ in inputs]

        def expr(x_, *rest):
            rest = iter(rest)
            return _expression(x_, *(None if p is None else next(rest) for p in params), act)
        got = iter(train_ops._recorded(expr, given, [n for _, n in inputs], d))
        return tuple(None if p is None else next(got) for p in (x, *params))
    dev, (hidden2, d_in), d_out, dtype = d.device, w_in.shape, w_out.shape[0], d.dtype
    sizes = d.numel() // d_out, d_in, hidden2 // 2, d_out, _TYPES[dtype]
    xs = train_ops._saved(x, sizes[0] * d_in, dev, dtype)
    p = [None if t is None else train_ops._saved(t, t.numel(), dev, dtype) for t in params]
    kept = train_ops._saved(kept, train_ops._bytes("proteus_gated_mlp_kept_bytes", *sizes), dev, torch.uint8)
    if kept.data_ptr() % 256:
        kept = kept.clone()
    dx = torch.empty(x.shape, dtype=dtype, device=dev) if need[0] else None
    grads = [torch.empty_like(t, memory_format=torch.contiguous_format) if t is not None and n else None for t, n in zip(params, need[1:5])]
    n = train_ops._bytes("proteus_gated_mlp_bwd_bytes", *sizes)
    train_ops._call("proteus_gated_mlp_bwd", dev, xs, train_ops._pointers(p), train_ops._dense(d), dx, train_ops._pointers(grads), kept, kept.numel(),
                    train_ops._workspace(n, dev), n, *sizes[:4], _ACTS[act], sizes[4])
    return (dx, *grads)


def _forward(x, params, act, keep):
    """(y, what the backward reads) of dense tensors."""
    w_in, _, w_out, _ = params
    d_in, hidden, d_out, dev = x.shape[-1], w_in.shape[0] // 2, w_out.shape[0], x.device
    sizes = x.numel() // d_in, d_in, hidden, d_out, _TYPES[x.dtype]
    y = torch.empty(*x.shape[:-1], d_out, dtype=x.dtype, device=dev)
    kept_bytes = train_ops._bytes("proteus_gated_mlp_kept_bytes", *sizes) if keep else 0
    ws_bytes = train_ops._bytes("proteus_gated_mlp_train_fwd_bytes" if keep else "proteus_gated_mlp_fwd_bytes", *sizes)
    kept = train_ops._workspace(kept_bytes, dev)
    train_ops._call("proteus_gated_mlp_fwd", dev, x, train_ops._pointers(params), y, kept, kept_bytes, train_ops._workspace(ws_bytes, dev), ws_bytes, *sizes[:4], _ACTS[act], sizes[4])
    return y, kept


def _taken(x, params):
    """Are these tensors of the kernels' types and sizes, on one GPU, and does nothing look on that expects torch operators?"""
    w_in, _, w_out, _ = params
    if torch.is_autocast_enabled("cuda") or not train_ops.unobserved():
        return False
    dev = x.get_device()
    if not x.is_cuda or x.dtype not in _TYPES or x.numel() == 0:
        return False
    for t in (x, *params):
        if t is not None and (type(t) not in train_ops._PLAIN_TYPES or t.dtype != x.dtype or t.get_device() != dev or t.layout != torch.strided):
            return False
    d_in = x.shape[-1]
    return train_ops._bytes("proteus_gated_mlp_kept_bytes", x.numel() // d_in, d_in, w_in.shape[0] // 2, w_out.shape[0], _TYPES[x.dtype]) > 0


def gated_mlp(x, w_in, b_in, w_out, b_out, act: str = "silu"):
    """(act(x @ w_in[:hidden].T + b_in[:hidden]) * (x @ w_in[hidden:].T + b_in[hidden:])) @ w_out.T + b_out for x [..., d_in], w_in [2 hidden, d_in] (the gates'
    rows, then the values'), w_out [d_out, hidden], biases [2 hidden] and [d_out] or None; act: "silu", "gelu" (exact), "relu" or "sigmoid".

    fp32 or bf16, all tensors alike on one GPU, widths multiples of 4 (fp32) or 8 (bf16).  Sums are fp32; in bf16 the hidden features are rounded to bf16, as which
    the second product and the backward read them, their gradients likewise, and the gates and values are kept for the backward to 20 bits.  Under autocast, functional transforms, forward-mode differentiation or
    tracing the torch expression is taken, as it is by a backward that is itself recorded.
    """
    params = (w_in, b_in, w_out, b_out)
    if act not in _ACTS:
        raise NotImplementedError(f"act must be one of {', '.join(_ACTS)}, not {act}")
    y = _lib.ops().gated_mlp(x, *params, _ACTS[act])
    if y is not None:
        return y
    if x.dim() < 1 or w_in.dim() != 2 or w_out.dim() != 2 or w_in.shape[0] != 2 * w_out.shape[1] or x.shape[-1] != w_in.shape[1]:
        raise AssertionError(f"w_in must be of shape (2 hidden, {x.shape[-1] if x.dim() else '?'}) and w_out of (d_out, hidden), not {tuple(w_in.shape)} and {tuple(w_out.shape)}")
    if (b_in is not None and b_in.shape != w_in.shape[:1]) or (b_out is not None and b_out.shape != w_out.shape[:1]):
        raise AssertionError(f"biases must be of shape ({w_in.shape[0]},) and ({w_out.shape[0]},)")
    if _taken(x, params):
        return _run(x, params, act)
    if not x.is_cuda or any(t is not None and t.device != x.device for t in params):
        raise _lib.ProteusError("gated_mlp needs tensors on the GPU, all on one (there is no CPU path)")
    if torch.is_autocast_enabled("cuda") or not train_ops.unobserved() or x.numel() == 0 or any(t is not None and type(t) not in train_ops._PLAIN_TYPES for t in (x, *params)):
        return _expression(x, *params, act)
    if x.dtype not in _TYPES or any(t is not None and t.dtype != x.dtype for t in params):
        raise NotImplementedError("gated_mlp takes float32 or bfloat16 tensors, all alike")
    raise ValueError(f"gated_mlp does not take {x.numel() // x.shape[-1]} rows of {x.shape[-1]} through {w_out.shape[1]} to {w_out.shape[0]} features in {x.dtype}: widths must be multiples of "
                     f"{4 if x.dtype == torch.float32 else 8}" + (", matrices below 2 GiB" if x.dtype == torch.float32 else ""))


def _run(x, params, act):
    if torch.is_grad_enabled() and (x.requires_grad or any(t is not None and t.requires_grad for t in params)):
        return _GatedMLP.apply(x, *params, act)
    return _forward(train_ops._dense(x), [None if t is None else train_ops._dense(t) for t in params], act, False)[0]


class GatedMLP(nn.Module):
    """in_proj -> act(first half) * second half -> dropout -> out_proj: MLP (encoder.py) with a gate.  in_proj has 2 d_hidden rows, the gates' first.  fp32 and bf16 on the
    GPU, without active dropout or hooks, run on the kernels (gated_mlp); anything else takes the torch expression."""

    def __init__(self, d_in=512, d_out=512, d_hidden=1024, dropout=0.1, act="silu", bias=True):
        super().__init__()
        if act not in _ACTS:
            raise NotImplementedError(f"act must be one of {', '.join(_ACTS)}, not {act}")
        self.in_proj = nn.Linear(d_in, 2 * d_hidden, bias=bias)
        self.out_proj = nn.Linear(d_hidden, d_out, bias=bias)
        self.dropout = nn.Dropout(dropout)
        self.act = act
        with torch.no_grad():
            for half in self.in_proj.weight.chunk(2):
                nn.init.xavier_uniform_(half)
        nn.init.xavier_uniform_(self.out_proj.weight)
        if bias:
            nn.init.zeros_(self.in_proj.bias)
            nn.init.zeros_(self.out_proj.bias)

    def forward(self, x):
        a, b = self.in_proj, self.out_proj
        if train_ops.plain_module(a, nn.Linear) and train_ops.plain_module(b, nn.Linear) and train_ops.inactive_dropout(self.dropout):
            params = (a.weight, a.bias, b.weight, b.bias)
            y = _lib.ops().gated_mlp(x, *params, _ACTS[self.act]) if x.is_cuda else None
            if y is not None:
                return y
            if (x.dim() and a.weight.shape[0] == 2 * b.weight.shape[1] and x.shape[-1] == a.weight.shape[1] and all(p is None or p.shape == w.shape[:1] for p, w in ((a.bias, a.weight), (b.bias, b.weight)))
                    and _taken(x, params)):
                return _run(x, params, self.act)
        gate, value = a(x).chunk(2, -1)
        return b(self.dropout(_FUNCTIONS[self.act](gate) * value))
