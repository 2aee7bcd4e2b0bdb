"""Refusals of the norm and rotation of queries and keys and of the clipping of gradients, which need no GPU: the library's checks before any HIP call, and the
errors of the Python functions."""
import contextlib
import ctypes
import math
import types

import pytest
import torch

import proteusai_amd as pa
from proteusai_amd import _lib

P = 0x10000                     # an aligned address that nothing reads


def qk_args(**kw):
    a = _lib.QkArgs()
    for i in range(3):
        a.x[i] = a.dy[i] = a.y[i] = P
        for k in range(3):
            a.x_strides[i][k] = a.dy_strides[i][k] = a.y_strides[i][k] = 512
    a.base, a.eps = 10000.0, 1e-6
    a.Z, a.N, a.heads_q, a.heads_k, a.heads_v, a.d_head = 2, 10, 8, 4, 4, 64
    a.x_type = a.y_type = a.weight_type = _lib.DTYPE_BF16
    for k, v in kw.items():
        if isinstance(v, tuple):
            at = getattr(a, k)
            for i in v[0][:-1]:
                at = at[i]
            at[v[0][-1]] = v[1]
        else:
            setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(x=((0,), None)), -1), (dict(x=((2,), None)), -1), (dict(y=((1,), None)), -1), (dict(heads_v=0, x=((2,), None)), 0),
    (dict(d_head=48), -3), (dict(Z=0), -2), (dict(N=-1), -2), (dict(heads_q=0), -2), (dict(heads_v=-1), -2), (dict(Z=1 << 16, N=1 << 15), -2),
    (dict(eps=-1.0), -2), (dict(eps=math.nan), -2), (dict(base=0.0), -2), (dict(base=math.inf), -2), (dict(base=math.nan), -2),
    (dict(x_type=7), -9), (dict(y_type=_lib.DTYPE_F32), -9), (dict(y_type=_lib.DTYPE_F16), -9), (dict(weight_type=3), -9),
    (dict(x_type=_lib.DTYPE_F32), 0), (dict(x=((1,), P + 8)), -5), (dict(y=((0,), P + 2)), -5), (dict(x_strides=((0, 2), 65)), -5), (dict(y_strides=((1, 0), 4)), -5),
    (dict(weight=((0,), P + 1)), -5), (dict(positions=P + 4), -5),
])
def test_qk_argument_checks(kw, code):
    lib = _lib.load()
    assert lib.proteus_qk_norm_rotate_check(qk_args(**kw), 0) == code
    if code < 0:
        assert lib.proteus_qk_norm_rotate_fwd(qk_args(**kw), None) == code


def test_qk_backward_argument_checks():
    lib = _lib.load()
    assert lib.proteus_qk_norm_rotate_check(qk_args(), 1) == 0
    assert lib.proteus_qk_norm_rotate_check(qk_args(x=((2,), None)), 1) == 0                   # (the values' input is not read again)
    assert lib.proteus_qk_norm_rotate_check(qk_args(dy=((0,), None)), 1) == -1
    assert lib.proteus_qk_norm_rotate_check(qk_args(dy=((1,), P + 8)), 1) == -5
    assert lib.proteus_qk_norm_rotate_check(qk_args(dy_strides=((2, 1), 12)), 1) == -5
    n = lib.proteus_qk_norm_rotate_bwd_workspace_bytes(2, 10, 8, 4, 4, 64, 0)
    assert n > 0 and lib.proteus_qk_norm_rotate_bwd_workspace_bytes(2, 10, 8, 4, 4, 48, 0) == 0
    assert lib.proteus_qk_norm_rotate_bwd(qk_args(), P, None, None, 0, None) == -1             # a gradient without a workspace
    assert lib.proteus_qk_norm_rotate_bwd(qk_args(), P, None, P, n - 1, None) == -8
    assert lib.proteus_qk_norm_rotate_bwd(qk_args(), P + 1, None, P, n, None) == -5
    assert lib.proteus_qk_norm_rotate_check(None, 0) == -1


def test_qk_refusals():
    q = torch.zeros(2, 4, 10, 64)
    with pytest.raises(_lib.ProteusError, match="on the GPU"):
        pa.qk_norm_rotate(q, q)
    with pytest.raises(_lib.ProteusError, match="on the GPU"):
        pa.qk_norm_rotate_qkv(torch.zeros(2, 10, 3, 4, 64))
    for bad in (dict(base=0.0), dict(base=-1.0), dict(base=math.inf), dict(eps=-1e-6), dict(eps=math.nan)):
        with pytest.raises(AssertionError):
            pa.qk_norm_rotate(q, q, **bad)
    for a, b in ((q[0], q), (q, q[:, :, :5]), (q, q[:1]), (q, q[..., :32]), (q[..., :48], q[..., :48])):
        with pytest.raises(AssertionError):
            pa.qk_norm_rotate(a, b)
    with pytest.raises(AssertionError):
        pa.qk_norm_rotate_qkv(torch.zeros(2, 10, 2, 4, 64))
    for a, b, out in ((q.double(), q.double(), None), (q, q.bfloat16(), None), (q.bfloat16(), q.bfloat16(), torch.float32), (q, q, torch.float64), (q.half(), q.half(), torch.bfloat16)):
        with pytest.raises(NotImplementedError):
            pa.qk_norm_rotate(a, b, out_dtype=out)


@pytest.mark.parametrize("kw,error", [
    (dict(qw=(65,)), AssertionError), (dict(qw=(3, 64)), AssertionError), (dict(qw=(64,), kw=(2, 64)), NotImplementedError), (dict(positions=(11,)), AssertionError),
    (dict(positions=(1, 10)), AssertionError), (dict(mask=(2, 11)), AssertionError), (dict(qw=(64,), wtype=torch.float64), NotImplementedError),
    (dict(positions=(10,), ptype=torch.float32), AssertionError), (dict(positions=(10,), ptype=torch.bool), AssertionError),
])
def test_qk_refusals_behind_the_device_check(kw, error):
    """The checks of what comes with q and k, on stand-ins that claim to be on the GPU."""
    from proteusai_amd import qk_norm

    class OnGpu(torch.Tensor):
        is_cuda = True
    q, k = (torch.zeros(2, h, 10, 64).as_subclass(OnGpu) for h in (4, 2))

    def like(name, dtype=torch.float32):
        return torch.zeros(kw[name], dtype=dtype).as_subclass(OnGpu) if name in kw else None
    with pytest.raises(error):
        qk_norm._general(q, k, like("qw", kw.get("wtype", torch.float32)), like("kw"), like("positions", kw.get("ptype", torch.int64)), like("mask", torch.bool), 1e4, 1e-6, False, None)


@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("fused", [False, True])
def test_the_expression_leaves_padded_tokens_out(eps, fused):
    """What recorded backwards, transforms and tracing take: zeros come out of padded tokens, and nothing of them goes into a gradient of the first or second order,
    whatever they or the gradients at their places hold.  The other tokens' operations are the same without them but for the order of sums: fewer than 100 roundings of
    2^-24 behind one another, of terms up to eight times the largest element: 2^-14 of it."""
    from proteusai_amd import qk_norm
    g = torch.Generator().manual_seed(3)
    Z, H, N, d, n = 2, 3, 6, 32, 4                               # tokens n, n + 1, ... are padded
    x = torch.randn(Z, N, 3, H, d, generator=g, dtype=torch.float32)
    dy = torch.randn(Z, N, 3, H, d, generator=g)
    x[:, n], dy[:, n] = math.nan, math.inf
    x[:, n + 1], dy[:, n + 1] = 0.0, math.nan
    w = [1.0 + 0.1 * torch.randn(H, d, generator=g) for _ in range(2)]
    mask = (torch.arange(N) >= n).expand(Z, N)

    def run(x, dy, mask):
        x, qw, kw = x.clone().requires_grad_(), *(t.clone().requires_grad_() for t in w)
        how = None, mask, 1e4, eps, False, torch.float32
        if fused:
            outs, dys = (qk_norm._expression(x, None, qw, kw, *how),), (dy,)
        else:
            outs = qk_norm._expression(x[:, :, 0].permute(0, 2, 1, 3), x[:, :, 1].permute(0, 2, 1, 3), qw, kw, *how)
            dys = tuple(dy[:, :, i].permute(0, 2, 1, 3) for i in range(2))
        first = torch.autograd.grad(outs, (x, qw, kw), dys, create_graph=True)
        second = torch.autograd.grad(sum(t.square().sum() for t in first), (x, qw, kw))
        return [o.detach() if fused else o.detach().permute(0, 2, 1, 3) for o in outs], [t.detach() for t in first], second
    outs, first, second = run(x, dy, mask)
    wants = run(x[:, :n], dy[:, :n], None)
    for t, want in zip((*outs, first[0], second[0]), (*wants[0], wants[1][0], wants[2][0])):
        assert not t[:, n:].any() and float((t[:, :n] - want).abs().max()) <= 2.0 ** -14 * float(want.abs().max())
    for t, want in zip((*first[1:], *second[1:]), (*wants[1][1:], *wants[2][1:])):
        assert float((t - want).abs().max()) <= 2.0 ** -14 * float(want.abs().max())


def arrays(n=2, **kw):
    v = dict(grads=[P] * n, out=[P] * n, numel=[10] * n, types=[0] * n, out_types=[0] * n, count=n, norm_type=2, max_norm=1.0, norm=P, ws=P, ws_bytes=1 << 20)
    v.update(kw)

    def of(ctype, values):
        return None if values is None else (ctype * len(values))(*values)
    return (of(ctypes.c_void_p, v["grads"]), of(ctypes.c_void_p, v["out"]), of(ctypes.c_int64, v["numel"]), of(ctypes.c_int, v["types"]), of(ctypes.c_int, v["out_types"]),
            v["count"], v["norm_type"], v["max_norm"], v["norm"], v["ws"], v["ws_bytes"])


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(out=None, out_types=None, max_norm=math.nan), 0), (dict(count=-1), -2), (dict(grads=None), -1), (dict(norm=None), -1), (dict(ws=None), -1), (dict(ws_bytes=64), -8),
    (dict(ws=P + 4), -5), (dict(out_types=None), -1), (dict(norm_type=4), -7), (dict(max_norm=-1.0), -2), (dict(max_norm=math.nan), -2), (dict(numel=[10, -1]), -2),
    (dict(types=[0, 3]), -9), (dict(out_types=[-1, 0]), -9), (dict(grads=[P, None]), -1), (dict(grads=[P, None], numel=[10, 0]), 0), (dict(grads=[P, P + 2]), -5),
    (dict(grads=[P, P + 2], types=[0, 1]), 0), (dict(out=[P + 1, P], out_types=[1, 0]), -5), (dict(grads=[P, (1 << 48) - 8]), -5),
])
def test_clip_argument_checks(kw, code):
    lib = _lib.load()
    assert lib.proteus_clip_grads_check(*arrays(**kw)) == code
    if code < 0:
        assert lib.proteus_clip_grads(*arrays(**kw), None) == code
    assert lib.proteus_clip_grads_workspace_bytes(-1) == 0


def test_clip_refusals():
    g = [torch.zeros(3)]
    with pytest.raises(_lib.ProteusError, match="on the GPU"):
        pa.grad_norm(g)
    with pytest.raises(_lib.ProteusError, match="on the GPU"):
        pa.clip_grad_norm(g, 1.0)
    p = torch.nn.Parameter(torch.zeros(3))
    p.grad = torch.zeros(3)
    with pytest.raises(_lib.ProteusError, match="on the GPU"):
        pa.clip_grad_norm_([p], 1.0)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError):
            pa.clip_grad_norm(g, bad)
    for bad in (3.0, 0.0, -math.inf, math.nan):
        with pytest.raises(NotImplementedError):
            pa.grad_norm(g, bad)
    with pytest.raises(AssertionError):
        pa.clip_grad_norm(g, 1.0, out=[])
    for bad in ([torch.zeros(3, dtype=torch.float64)], [torch.zeros(3, dtype=torch.int32)], [torch.eye(3).to_sparse()], [1.0]):
        with pytest.raises(NotImplementedError):
            pa.grad_norm(bad)
    assert float(pa.grad_norm([])) == 0.0 and float(pa.clip_grad_norm_(iter([]), 1.0)) == 0.0


def test_shared_memory_is_found_whatever_the_order():
    """The look at overlapping tensors, on stand-ins with addresses alone."""
    from proteusai_amd import grad_clip

    def at(begin, n=10):
        return types.SimpleNamespace(data_ptr=lambda: begin, numel=lambda: n, element_size=lambda: 4, dtype=torch.float32, device=torch.device("cpu"))
    a, b = at(1000), at(1040)
    for src, dst in (([a, a], [a, a]), ([a, b], [b, a]), ([a], [at(1004)]), ([at(1036), a], [at(1036), a]), ([at(0), a], [at(1004), at(5000)])):
        with pytest.raises(ValueError, match="share memory"):
            grad_clip._launch(src, dst, 2, 1.0)


def test_a_gradient_scaled_in_place_and_read_for_another_is_refused(monkeypatch):
    """The second pair would read what the first one's workgroups write.  (Nothing is launched: the library is out of reach.)"""
    from proteusai_amd import grad_clip

    class Reached(Exception):
        pass

    def reached():
        raise Reached
    monkeypatch.setattr(_lib, "load", reached)
    a, b, c, none = torch.ones(10), torch.ones(10), torch.ones(10), torch.ones(0)
    for src, dst in (([a, a], [a, b]), ([a, a], [b, a]), ([a, b, a], [a, b, c]), ([a[:5], a[4:]], [a[:5], b[:6]]), ([b, a], [a, c]), ([a, a.half()], [a, a.view(torch.float16)[:10]])):
        with pytest.raises(ValueError, match="share memory"):
            grad_clip._launch(src, dst, 2, 1.0)
    # what is read alone may be read twice, and empty tensors are nowhere
    for src, dst in (([a, b], [a, b]), ([a, a], [b, c]), ([a, b], [a, c]), ([a[:5], a[5:]], [a[:5], b[:5]]), ([none, a], [none, a]), ([a.half()], [b])):
        with pytest.raises(Reached):
            grad_clip._launch(src, dst, 2, 1.0)


def test_tensors_made_in_inference_mode_are_not_written_outside_of_it(monkeypatch):
    """On stand-ins that claim to be on the GPU (nothing is launched: the library is out of reach)."""
    from proteusai_amd import grad_clip

    class OnGpu(torch.Tensor):
        is_cuda = True

    class Reached(Exception):
        pass

    def reached(*a):
        raise Reached
    monkeypatch.setattr(_lib, "load", reached)
    monkeypatch.setattr(_lib, "on_device", lambda dev: contextlib.nullcontext())
    with torch.inference_mode():
        made = torch.ones(6).as_subclass(OnGpu)
    plain = torch.ones(6).as_subclass(OnGpu)
    for grads, out in (([made], [made]), ([plain], [made]), ([plain, made], [plain, made])):
        with pytest.raises(RuntimeError, match="inference"):
            grad_clip._clip(grads, out, _lib.NORM_2, 1.0, False)
    for grads, out in (([made], None), ([made], [plain])):
        with pytest.raises(Reached):
            grad_clip._clip(grads, out, _lib.NORM_2, 1.0, False)
    with torch.inference_mode(), pytest.raises(Reached):
        grad_clip._clip([made], [made], _lib.NORM_2, 1.0, False)


def test_gated_mlp_argument_checks():
    lib = _lib.load()
    sizes = (10, 64, 96, 72, _lib.DTYPE_BF16)
    kept, fwd, bwd = (getattr(lib, f"proteus_gated_mlp_{n}_bytes") for n in ("kept", "fwd", "bwd"))
    assert kept(*sizes) >= 10 * 3 * 96 * 2 and fwd(*sizes) >= 10 * 96 * 2 and bwd(*sizes) > 0
    for bad in ((0, 64, 96, 72, 1), (-1, 64, 96, 72, 1), (10, 60, 96, 72, 1), (10, 64, 92, 72, 1), (10, 64, 96, 0, 1), (10, 64, 96, 72, 2), (10, 64, 96, 72, 7), (10, 62, 96, 72, 0),
                (1 << 20, 64, 1024, 72, 0), (10, 1 << 15, 1 << 15, 8, 1), (1 << 29, 8, 8, 8, 1)):
        assert kept(*bad) == fwd(*bad) == bwd(*bad) == 0, bad

    def forward(x=P, params=(P, P, P, P), y=P, k=P, k_bytes=1 << 30, ws=None, ws_bytes=0, act=0, s=sizes):
        return lib.proteus_gated_mlp_fwd(x, None if params is None else (ctypes.c_void_p * 4)(*params), y, k, k_bytes, ws, ws_bytes, *s[:4], act, s[4], None)
    for kw, code in ((dict(x=None), -1), (dict(params=None), -1), (dict(params=(None, P, P, P)), -1), (dict(params=(P, P, None, P)), -1), (dict(y=None), -1), (dict(k=None), -1),
                     (dict(params=(P, P + 8, P, P)), -5), (dict(x=P + 8), -5), (dict(y=P + 2), -5), (dict(k=P + 16), -5), (dict(k_bytes=64), -8), (dict(act=4), -7), (dict(act=-1), -7),
                     (dict(k=None, ws=P, ws_bytes=64), -8), (dict(k=None, ws=P + 16, ws_bytes=1 << 20), -5), (dict(s=(0, 64, 96, 72, 1)), -2), (dict(s=(10, 64, 96, 71, 1)), -2),
                     (dict(s=(10, 64, 96, 72, 2)), -9)):
        assert forward(**kw) == code, kw

    def backward(grads=(P, P, P, P), dx=P, k=P, ws=P, ws_bytes=1 << 30):
        return lib.proteus_gated_mlp_bwd(P, (ctypes.c_void_p * 4)(P, P, P, P), P, dx, None if grads is None else (ctypes.c_void_p * 4)(*grads), k, 1 << 30, ws, ws_bytes, *sizes[:4], 0, sizes[4], None)
    for kw, code in ((dict(grads=None), -1), (dict(k=None), -1), (dict(ws=None), -1), (dict(ws_bytes=bwd(*sizes) - 1), -8), (dict(dx=P + 4), -5), (dict(grads=(P, P, P + 8, P)), -5), (dict(ws=P + 128), -5)):
        assert backward(**kw) == code, kw


def test_gated_mlp_keeps_the_bytes_it_documents():
    """7 bytes of bf16 or 12 of fp32 for each of rows * hidden, in up to three regions of whole 256 bytes."""
    lib = _lib.load()
    for rows in (1, 5, 300, 5003, 32768):
        for d_in, hidden, d_out in ((8, 8, 8), (512, 2048, 512), (712, 1912, 712)):
            for dtype, each in ((_lib.DTYPE_BF16, 7), (_lib.DTYPE_F32, 12)):
                n = lib.proteus_gated_mlp_kept_bytes(rows, d_in, hidden, d_out, dtype)
                assert 0 <= n - each * rows * hidden < 3 * 256 and n % 256 == 0, (rows, hidden, dtype)


def test_gated_mlp_refusals():
    x, w, b, wo, bo = torch.zeros(3, 64), torch.zeros(192, 64), torch.zeros(192), torch.zeros(72, 96), torch.zeros(72)
    with pytest.raises(_lib.ProteusError, match="on the GPU"):
        pa.gated_mlp(x, w, b, wo, bo)
    with pytest.raises(NotImplementedError, match="act"):
        pa.gated_mlp(x, w, b, wo, bo, act="tanh")
    with pytest.raises(NotImplementedError, match="act"):
        pa.GatedMLP(act="tanh")
    for args in ((x[:, :32], w, b, wo, bo), (x, w[:191], b, wo, bo), (x, w[0], b, wo, bo), (x, w, b, wo[:, :95], bo), (x, w, b[:96], wo, bo), (x, w, b, wo, bo[:71]), (x[0, 0], w, b, wo, bo)):
        with pytest.raises(AssertionError):
            pa.gated_mlp(*args)
    # the module on the CPU is the expression, as MLP is
    m = pa.GatedMLP(16, 8, 24, dropout=0.0)
    t = torch.randn(5, 16)
    gate, value = (t @ m.in_proj.weight.t() + m.in_proj.bias).chunk(2, -1)
    assert torch.allclose(m(t), (gate * torch.sigmoid(gate) * value) @ m.out_proj.weight.t() + m.out_proj.bias, atol=1e-5)
