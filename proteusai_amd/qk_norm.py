"""Root-mean-square norm of every head's queries and keys and their rotation by position, in one pass of a HIP kernel, with gradients.

The reference's attention has neither (old/old_scripts/encoder.py:94-121); GeoAttention(rotary_base=...) puts the operator between its
projections and the attention.
"""
import torch

from . import _lib

_TYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def qk_norm_rotate(q, k, q_weight=None, k_weight=None, positions=None, base: float = 10000.0, eps: float = 1e-6, interleaved: bool = False, mask=None, out_dtype=None):
    """(q', k') of q [Z,Hq,N,d] and k [Z,Hk,N,d], d = 32, 64 or 128: x / sqrt(mean(x^2) + eps) * weight over the d elements of every head, then every pair of
    features turned by the angle position * base^(-2i/d), i = 0 .. d/2 - 1.

    q_weight, k_weight: [d], or [Hq,d] and [Hk,d] (one per head), or None (ones).  positions: whole numbers [N] or [Z,N] of any sign (angles are taken in 64
    bits), None: 0 .. N - 1.  interleaved: features 2i and 2i + 1 are a pair, otherwise i and i + d/2.  mask [Z,N] bool, True = padded: zeros come out, and
    nothing goes into the gradients of the weights.
    q and k: fp32, bf16 or fp16; out_dtype: theirs (default), or bf16 or fp16 for fp32 tensors (what the attention reads next).  Norm and rotation are computed in
    fp32 and rounded once.  q and k may be views with any batch / head / token strides (slices of a fused projection); results and gradients come in the
    memory order of q and k, dense.
    """
    for name, t in (("q", q), ("k", k)):
        if not isinstance(t, torch.Tensor) or t.dim() != 4:
            raise AssertionError(f"{name} must be a tensor of shape (batch, heads, N, d_k), not {tuple(t.shape) if isinstance(t, torch.Tensor) else type(t)}")
    return _call(q, k, q_weight, k_weight, positions, mask, base, eps, interleaved, out_dtype)


def qk_norm_rotate_qkv(qkv, q_weight=None, k_weight=None, positions=None, base: float = 10000.0, eps: float = 1e-6, interleaved: bool = False, mask=None, out_dtype=None):
    """qk_norm_rotate for self-attention on a fused projection qkv [Z,N,3,H,d] (q, k, v = qkv[:, :, 0 / 1 / 2]): returns [Z,N,3,H,d], dense, with the values passed on
    in out_dtype (zeros where padded), as geometric_attn_qkv takes it; the gradient of qkv comes back as one tensor.  Same arguments otherwise."""
    if not isinstance(qkv, torch.Tensor) or qkv.dim() != 5 or qkv.size(2) != 3:
        raise AssertionError(f"qkv must be a tensor of shape (batch, N, 3, heads, d_k), not {tuple(qkv.shape) if isinstance(qkv, torch.Tensor) else type(qkv)}")
    return _call(qkv, None, q_weight, k_weight, positions, mask, base, eps, interleaved, out_dtype)


def _call(q, k, qw, kw, positions, mask, base, eps, interleaved, out_dtype):
    base, eps, interleaved = float(base), float(eps), bool(interleaved)
    if not 0.0 < base < float("inf"):
        raise AssertionError(f"base must be a positive number, not {base}")
    if not 0.0 <= eps < float("inf"):
        raise AssertionError(f"eps must not be negative, but is {eps}")
    out_type = -1 if out_dtype is None else _TYPES.get(out_dtype, -2)
    if out_type >= -1:
        out = _lib.ops().qk_norm_rotate(q, k, qw, kw, positions, mask, base, eps, interleaved, out_type)
        if out is not None:
            return out
    return _general(q, k, qw, kw, positions, mask, base, eps, interleaved, out_dtype)


def _general(q, k, qw, kw, positions, mask, base, eps, interleaved, out_dtype):
    """Calls that are not plain: what is wrong is refused, what lies otherwise than the kernel reads it is laid out, and what the kernel cannot do (functional
    transforms, forward-mode differentiation, a dispatch mode, tracing) takes the expression."""
    fused = k is None
    Z, N = (q.size(0), q.size(1)) if fused else (q.size(0), q.size(2))
    H, Hk, d = (q.size(3), q.size(3), q.size(4)) if fused else (q.size(1), k.size(1), q.size(3))
    if not fused and (k.size(0), k.size(2), k.size(3)) != (Z, N, d):
        raise AssertionError(f"q and k must agree in all but their heads, but got {tuple(q.shape)} and {tuple(k.shape)}")
    if d not in (32, 64, 128):
        raise AssertionError(f"the size of a head must be 32, 64 or 128, not {d}")
    if q.dtype not in _TYPES or (not fused and k.dtype != q.dtype):
        raise NotImplementedError(f"q and k must be float32, bfloat16 or float16, both alike, not {q.dtype}" + ("" if fused else f" and {k.dtype}"))
    out_dtype = out_dtype or q.dtype
    if out_dtype not in _TYPES or (out_dtype != q.dtype and q.dtype != torch.float32):
        raise NotImplementedError(f"out_dtype must be {q.dtype}" + (", bfloat16 or float16" if q.dtype == torch.float32 else "") + f", not {out_dtype}")
    dev = q.device
    if not q.is_cuda or not (fused or k.device == dev):
        raise _lib.ProteusError("qk_norm_rotate needs tensors on the GPU, all on one (there is no CPU path)")
    weights = [w for w in (qw, kw) if w is not None]
    for w, heads, name in ((qw, H, "q_weight"), (kw, Hk, "k_weight")):
        if w is not None and tuple(w.shape) not in ((d,), (heads, d)):
            raise AssertionError(f"{name} must be of shape ({d},) or ({heads}, {d}), not {tuple(w.shape)}")
        if w is not None and (w.dtype not in _TYPES or w.device != dev):
            raise NotImplementedError(f"{name} must be float32, bfloat16 or float16 on {dev}, not {w.dtype} on {w.device}")
    if len(weights) == 2 and (qw.dim() != kw.dim() or qw.dtype != kw.dtype):
        raise NotImplementedError("q_weight and k_weight must be alike in type, and both or neither one per head")
    if positions is not None:
        if not isinstance(positions, torch.Tensor) or positions.dtype.is_floating_point or positions.dtype.is_complex or positions.dtype == torch.bool:
            raise AssertionError("positions must be a tensor of whole numbers")
        if tuple(positions.shape) not in ((N,), (Z, N)):
            raise AssertionError(f"positions must be of shape ({N},) or ({Z}, {N}), not {tuple(positions.shape)}")
        positions = positions.to(device=dev, dtype=torch.int64)
        positions = positions if positions.size(-1) < 2 or positions.stride(-1) == 1 else positions.contiguous()
    if mask is not None:
        if tuple(mask.shape) != (Z, N):
            raise AssertionError(f"mask must be of shape ({Z}, {N}), not {tuple(mask.shape)}")
        mask = mask.to(device=dev, dtype=torch.bool).contiguous()
    from . import train_ops
    if q.numel() == 0 or (not fused and k.numel() == 0) or not train_ops.unobserved() or any(type(t) not in train_ops._PLAIN_TYPES for t in (q, k, *weights) if t is not None):
        return _expression(q, k, qw, kw, positions, mask, base, eps, interleaved, out_dtype)

    def dense(t):
        return t.clone(memory_format=torch.contiguous_format) if t.data_ptr() % 16 or not t.is_contiguous() else t
    # (a copy that autograd sees, where the rows are not the kernel's to read)
    if not all(_rows_ok(t) for t in ([q[:, :, i].permute(0, 2, 1, 3) for i in range(3)] if fused else [q, k])):
        q, k = dense(q), None if fused else dense(k)
    qw, kw = (None if w is None else w.contiguous() for w in (qw, kw))
    with _lib.on_device(dev):
        out = _lib.ops().qk_norm_rotate(q, k, qw, kw, positions, mask, base, eps, interleaved, _TYPES[out_dtype])
    if out is None:
        raise _lib.ProteusError(f"qk_norm_rotate could not be launched on {tuple(q.shape)}")
    return out


def _rows_ok(t):
    """Can the kernel read this [Z,H,N,d] in place?"""
    return t.data_ptr() % 16 == 0 and t.stride(3) == 1 and all(t.size(i) == 1 or t.stride(i) * t.element_size() % 16 == 0 for i in range(3))


def _turned(x, w, positions, mask, base, eps, interleaved, out_dtype):
    """The operator on one [Z,H,N,d] as torch operators, in fp32 from angles in 64 bits."""
    Z, _, N, d = x.shape
    pos = torch.arange(N, device=x.device) if positions is None else positions
    angle = pos.double()[..., None] * base ** (torch.arange(d // 2, device=x.device, dtype=torch.float64) * (-2.0 / d))
    angle = angle if angle.dim() == 2 else angle[:, None]
    c, s = torch.cos(angle).float(), torch.sin(angle).float()
    v, padded = x.float(), None if mask is None else mask[:, None, :, None]
    if padded is not None:
        # (ones: with eps = 0 the norm of zeros has neither a value nor a derivative)
        v = torch.where(padded, 1.0, v)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps)
    if w is not None:
        v = v * (w.float()[:, None] if w.dim() == 2 else w.float())
    a, b = (v[..., 0::2], v[..., 1::2]) if interleaved else (v[..., :d // 2], v[..., d // 2:])
    turned = a * c - b * s, b * c + a * s
    v = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return (v if padded is None else torch.where(padded, 0.0, v)).to(out_dtype)


def _expression(q, k, qw, kw, positions, mask, base, eps, interleaved, out_dtype):
    how = positions, mask, base, eps, interleaved, out_dtype
    if k is not None:
        return _turned(q, qw, *how), _turned(k, kw, *how)
    x, y, v = (q[:, :, i].permute(0, 2, 1, 3) for i in range(3))
    v = v.to(out_dtype) if mask is None else torch.where(mask[:, None, :, None], 0.0, v).to(out_dtype)
    return torch.stack([t.permute(0, 2, 1, 3) for t in (_turned(x, qw, *how), _turned(y, kw, *how), v)], 2)


def _general_backward(q, k, qw, kw, positions, mask, grads, base, eps, interleaved, out_type, fused):
    """Gradients of (q, k) or qkv and of the two weights where the backward is itself recorded, or a gradient has another form than the kernel reads."""
    from . import train_ops
    out_dtype = {v: t for t, v in _TYPES.items()}[out_type]
    inputs = [t for t in ((q,) if fused else (q, k)) + (qw, kw) if t is not None]
    needs = [t.requires_grad for t in inputs]
    with torch.enable_grad():
        # (each a tensor of its own: one that stands in two places has a gradient for each)
        inputs = [t.view_as(t) for t in inputs]

    def expr(*given):
        given = iter(given)
        x = [next(given) for _ in range(1 if fused else 2)]
        w = [None if t is None else next(given) for t in (qw, kw)]
        outs = _expression(x[0], None if fused else x[1], *w, positions, mask, base, eps, interleaved, out_dtype)
        outs = (outs,) if fused else outs
        return torch.cat([o.reshape(-1) for o, g in zip(outs, grads) if g is not None])
    present = [g.reshape(-1) for g in grads if g is not None]
    if not present or not any(needs):
        return (None,) * (3 if fused else 4)
    got = iter(train_ops._recorded(expr, inputs, needs, torch.cat(present)))
    return tuple(None if t is None else next(got) for t in ((q,) if fused else (q, k)) + (qw, kw))
