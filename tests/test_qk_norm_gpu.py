"""GPU tests of the norm and rotation of queries and keys against the formulas in float64 on the CPU.

Bars, from the roundings: u = x r w has r from a sum of d <= 128 squares (16 in a row, then 3 steps) and a square root, and two products: below 16 steps of
2^-24; its rotation has a cosine and a sine off by at most 2^-22 (the angle within a turn rounded to fp32, times 2 pi, and two ulp of the function) and three
roundings.  Together below 32 * 2^-24 of |a| + |b| of the pair: 2^-19, beside half a step of the result's type.  The gradient adds the sums of the norm's own
derivative, whose terms are at most |m| of the head: 2^-17 r |m|.  The weights' gradients are sums in chains of at most a few hundred terms: 2^-16 of the sum
of the terms' sizes."""
import decimal
import math

import pytest
import torch

import proteusai_amd as pa
from proteusai_amd import qk_norm

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


def half(t):
    return torch.finfo(t).eps / 2


def pairs(x, inter):
    return (x[..., 0::2], x[..., 1::2]) if inter else x.chunk(2, -1)


def joined(a, b, inter):
    return torch.stack((a, b), -1).flatten(-2) if inter else torch.cat((a, b), -1)


def reference(x, w, pos, mask, base, eps, inter, dy=None):
    """(y, bar of y, dx, bar of dx, dw terms' sums, their bars) of one [Z,H,N,d], in float64; w [H,d]."""
    x = x.detach().double().cpu()
    Z, H, N, d = x.shape
    if mask is not None:
        x = torch.where(mask.cpu()[:, None, :, None], 0.0, x)
    pos = (torch.arange(N) if pos is None else pos.cpu()).double().expand(Z, N)
    angle = pos[:, None, :, None] * base ** (-2.0 * torch.arange(d // 2, dtype=torch.float64) / d)
    c, s = angle.cos(), angle.sin()
    r = (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    n, w = x * r, w.detach().double().cpu()[:, None]
    a, b = pairs(n * w, inter)
    y = joined(a * c - b * s, b * c + a * s, inter)
    size = a.abs() + b.abs()
    bar = joined(size, size, inter) * 2.0 ** -19
    if dy is None:
        return y, bar
    dy = dy.detach().double().cpu()
    if mask is not None:
        dy = torch.where(mask.cpu()[:, None, :, None], 0.0, dy)
    a, b = pairs(dy, inter)
    t = joined(a * c + b * s, b * c - a * s, inter)
    m = t * w
    dx = r * (m - n * (m * n).mean(-1, keepdim=True))
    dx_bar = (r * m.norm(dim=-1, keepdim=True)).expand_as(dx) * 2.0 ** -17
    return y, bar, dx, dx_bar, (t * n).sum((0, 2)), (t * n).abs().sum((0, 2)) * 2.0 ** -16


def close(got, want, bar, what):
    off = (got.detach().double().cpu() - want).abs()
    limit = bar + half(got.dtype) * want.abs() + torch.finfo(got.dtype).tiny * half(got.dtype) * 2
    assert torch.isfinite(got).all(), what
    assert (off <= limit).all(), (what, float((off - limit).max()), int((off > limit).sum()))


def weights(H, d, how, dtype, g, gpu):
    if how == "none":
        return None, None
    shape = [(h, d) if how == "head" else (d,) for h in H]
    return tuple((1.0 + 0.3 * torch.randn(*s, generator=g)).to(dtype).to(gpu).requires_grad_() for s in shape)


def tail_mask(Z, N, g):
    lens = torch.randint(0, N + 1, (Z,), generator=g)
    lens[0] = 0                                   # one batch item without a token
    return torch.arange(N)[None, :] >= lens[:, None]


CASES = [
    # Z, Hq, Hk, N, d, x, out, interleaved, weights, weight type, positions, masked
    (1, 1, 1, 1, 32, BF, None, False, "shared", BF, None, False),
    (3, 8, 8, 1, 64, HF, None, False, "head", HF, "far", False),
    (2, 8, 8, 70, 64, BF, None, True, "shared", BF, None, True),
    (2, 4, 2, 129, 64, FL, BF, False, "head", FL, "batch", True),
    (1, 3, 5, 33, 128, FL, None, True, "none", FL, "far", False),
    (2, 16, 16, 65, 128, BF, None, False, "head", FL, "batch", True),
    (1, 40, 24, 19, 128, FL, HF, True, "shared", HF, "row", True),
    (1, 70, 1, 5, 64, HF, None, False, "shared", FL, "far", False),
    (4, 6, 6, 300, 32, FL, FL, False, "head", BF, "negative", True),
    (1, 8, 8, 2049, 64, BF, None, False, "shared", BF, None, False),
    (1, 2, 2, 40001, 32, FL, BF, True, "shared", FL, "far", False),
]


def positions_of(how, Z, N, g):
    if how is None:
        return None
    if how == "row":
        return torch.randint(0, 5000, (N,), generator=g, dtype=torch.int32)
    low, high = {"far": (10 ** 6, 2 * 10 ** 6), "batch": (0, 3000), "negative": (-4000, 4000)}[how]
    return torch.randint(low, high, (Z, N), generator=g)


@pytest.mark.parametrize("Z,Hq,Hk,N,d,x,out,inter,how,wtype,pos,masked", CASES)
def test_operator_and_gradients(gpu, Z, Hq, Hk, N, d, x, out, inter, how, wtype, pos, masked):
    g = torch.Generator().manual_seed(N + Hq)
    q, k = ((torch.randn(Z, h, N, d, generator=g) * torch.exp(torch.randn(1, h, 1, 1, generator=g))).to(x).to(gpu).requires_grad_() for h in (Hq, Hk))
    qw, kw = weights((Hq, Hk), d, how, wtype, g, gpu)
    positions = positions_of(pos, Z, N, g)
    mask = tail_mask(Z, N, g).to(gpu) if masked else None
    got = pa.qk_norm_rotate(q, k, qw, kw, positions=None if positions is None else positions.to(gpu), base=500.0, eps=1e-5, interleaved=inter, mask=mask, out_dtype=out)
    dy = [torch.randn(t.shape, generator=g).to(got[0].dtype).to(gpu) for t in (q, k)]
    leaves = [t for t in (q, k, qw, kw) if t is not None]
    grads = torch.autograd.grad(got, leaves, dy)
    with torch.no_grad():
        again = pa.qk_norm_rotate(q, k, qw, kw, positions=None if positions is None else positions.to(gpu), base=500.0, eps=1e-5, interleaved=inter, mask=mask, out_dtype=out)
    for i, (t, w) in enumerate(((q, qw), (k, kw))):
        full = torch.ones(t.shape[1], d) if w is None else w.detach().cpu().expand(t.shape[1], d)
        y, bar, dx, dx_bar, dw, dw_bar = reference(t, full, positions, mask, 500.0, 1e-5, inter, dy[i])
        assert got[i].dtype == (out or x) and grads[i].dtype == x
        close(got[i], y, bar, f"y{i}")
        close(grads[i], dx, dx_bar, f"dx{i}")
        assert torch.equal(got[i], again[i])
        if w is not None:
            if how == "shared":
                dw, dw_bar = dw.sum(0), dw_bar.sum(0)
            assert grads[2 + i].dtype == wtype
            close(grads[2 + i], dw, dw_bar, f"dw{i}")
        if mask is not None:
            assert not got[i].transpose(1, 2)[mask].any() and not grads[i].transpose(1, 2)[mask].any()


@pytest.mark.parametrize("Z,N,H,d,x,out,inter,masked", [(2, 70, 8, 64, FL, BF, False, True), (1, 1, 2, 32, BF, None, True, False), (3, 33, 24, 128, BF, None, False, True),
                                                         (2, 129, 4, 64, FL, None, True, True), (1, 1500, 8, 64, BF, None, False, False)])
def test_fused_projection_equals_the_separate_call(gpu, Z, N, H, d, x, out, inter, masked):
    g = torch.Generator().manual_seed(N)
    qkv = torch.randn(Z, N, 3, H, d, generator=g).to(x).to(gpu).requires_grad_()
    qw, kw = weights((H, H), d, "head", FL, g, gpu)
    mask = tail_mask(Z, N, g).to(gpu) if masked else None
    got = pa.qk_norm_rotate_qkv(qkv, qw, kw, interleaved=inter, mask=mask, out_dtype=out)
    dy = torch.randn(got.shape, generator=g).to(got.dtype).to(gpu)
    grads = torch.autograd.grad(got, [qkv, qw, kw], dy)
    q, k, v = (qkv.detach()[:, :, i].permute(0, 2, 1, 3).requires_grad_() for i in range(3))
    want = pa.qk_norm_rotate(q, k, qw, kw, interleaved=inter, mask=mask, out_dtype=out)
    wgrads = torch.autograd.grad(want, [q, k, qw, kw], [dy[:, :, i].permute(0, 2, 1, 3) for i in range(2)])
    assert got.shape == qkv.shape and got.is_contiguous() and got.dtype == (out or x)
    for i in range(2):
        assert torch.equal(got[:, :, i].permute(0, 2, 1, 3), want[i]) and torch.equal(grads[0][:, :, i].permute(0, 2, 1, 3), wgrads[i])
        # (the workgroups' shares of the tokens differ with the number of rows: another order of the sums)
        assert (grads[1 + i] - wgrads[2 + i]).abs().max() <= 2.0 ** -15 * wgrads[2 + i].abs().max() + 1e-5
    keep = torch.ones(Z, N, 1, 1, dtype=torch.bool, device=gpu) if mask is None else ~mask[:, :, None, None]
    assert torch.equal(got[:, :, 2], torch.where(keep, qkv[:, :, 2], 0.0).to(got.dtype))
    assert torch.equal(grads[0][:, :, 2], torch.where(keep, dy[:, :, 2], 0.0).to(x))


def test_layouts(gpu):
    """Views with other strides, orders and alignments give what dense copies give, in the views' memory order."""
    g = torch.Generator().manual_seed(1)
    base = torch.randn(2, 50, 3, 4, 64, generator=g).bfloat16().to(gpu)
    q, k = base[:, :, 0].permute(0, 2, 1, 3), base[:, :, 1].permute(0, 2, 1, 3)
    want = pa.qk_norm_rotate(q.contiguous(), k.contiguous())
    got = pa.qk_norm_rotate(q, k)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].permute(0, 2, 1, 3).is_contiguous()
    odd = torch.empty(2 * 4 * 50 * 64 + 1, dtype=torch.bfloat16, device=gpu)[1:].view(2, 4, 50, 64)
    odd.copy_(q)
    assert torch.equal(pa.qk_norm_rotate(odd, k)[0], want[0])                            # off 16 bytes
    wide = torch.zeros(2, 4, 50, 65, dtype=torch.bfloat16, device=gpu)
    wide[..., :64] = q
    assert torch.equal(pa.qk_norm_rotate(wide[..., :64], k)[0], want[0])                 # rows that are no multiples of 16 bytes apart
    features = q.permute(3, 2, 1, 0).contiguous().permute(3, 2, 1, 0)
    assert torch.equal(pa.qk_norm_rotate(features, k)[0], want[0])                       # features not contiguous
    one = q[:, :1].expand(2, 4, 50, 64)
    assert torch.equal(pa.qk_norm_rotate(one, k)[0], pa.qk_norm_rotate(one.contiguous(), k)[0])      # one head for all
    one = q[:, :1].detach().requires_grad_()
    dy = torch.randn(2, 4, 50, 64, generator=g).bfloat16().to(gpu)
    out = pa.qk_norm_rotate(one.expand(2, 4, 50, 64), k)
    got, = torch.autograd.grad(out[0], one, dy)
    leaf = one.detach().expand(2, 4, 50, 64).contiguous().requires_grad_()
    each, = torch.autograd.grad(pa.qk_norm_rotate(leaf, k)[0], leaf, dy)
    assert torch.equal(got, each.sum(1, keepdim=True))
    # gradients that are views themselves: of a sum (no stride at all), and of another memory order
    leaf = q.detach().clone().requires_grad_()
    got, = torch.autograd.grad(pa.qk_norm_rotate(leaf, k)[0].sum(), leaf)
    want, = torch.autograd.grad(pa.qk_norm_rotate(leaf, k)[0], leaf, torch.ones_like(leaf))
    assert torch.equal(got, want)
    rows = torch.randint(0, 3000, (50, 2), generator=g).to(gpu).t()                      # positions of another order
    assert torch.equal(pa.qk_norm_rotate(q, k, positions=rows)[0], pa.qk_norm_rotate(q, k, positions=rows.contiguous())[0])


def test_offsets_beyond_32_bits(gpu):
    wide = torch.zeros(1, 70_000, 2, 32_768, dtype=torch.bfloat16, device=gpu)           # 9 GB
    g = torch.Generator(device=gpu).manual_seed(0)
    wide[..., :64] = torch.randn(1, 70_000, 2, 64, generator=g, device=gpu)
    q = wide[..., :64].permute(0, 2, 1, 3)
    got = pa.qk_norm_rotate(q, q)
    want = pa.qk_norm_rotate(q.contiguous(), q.contiguous())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_padding_hides_what_is_not_finite(gpu):
    g = torch.Generator().manual_seed(2)
    q, k = (torch.randn(2, 4, 20, 64, generator=g).to(gpu) for _ in range(2))
    w = torch.ones(64, device=gpu)
    mask = torch.arange(20)[None, :] >= torch.tensor([13, 20])[:, None]
    dirty, dy = q.clone(), torch.randn(2, 4, 20, 64, generator=g).to(gpu)
    dirty[0, :, 13:] = float("nan")
    dirty[0, :, 15:] = float("inf")
    bad = dy.clone()
    bad[0, :, 13:] = float("nan")
    results = []
    for x, d in ((q, dy), (dirty, bad)):
        x, v = x.clone().requires_grad_(), w.clone().requires_grad_()
        y, _ = pa.qk_norm_rotate(x, k, v, w, mask=mask.to(gpu))
        results.append([y.detach(), *torch.autograd.grad(y, [x, v], d)])
    for a, b in zip(*results):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    # without a mask they stay in their own head
    y, _ = pa.qk_norm_rotate(dirty, k)
    assert torch.isfinite(y[0, :, :13]).all() and torch.isfinite(y[1]).all() and y[0, :, 13:].isnan().all()


def test_zero_rows_and_extremes(gpu):
    q = torch.zeros(1, 1, 3, 64, device=gpu)
    q[0, 0, 1, 5] = 1e18
    q[0, 0, 2] = 1e-30
    q.requires_grad_()
    y, _ = pa.qk_norm_rotate(q, q, eps=1e-6)
    d, = torch.autograd.grad(y.sum(), q)
    assert torch.isfinite(y).all() and torch.isfinite(d).all() and not y[0, 0, 0].any()
    assert abs(float(y[0, 0, 1].norm()) - 8.0) < 1e-5


def test_gradient_against_differences(gpu):
    g = torch.Generator().manual_seed(3)
    x0, w0, d = torch.randn(1, 2, 5, 32, generator=g).to(gpu), (1 + 0.2 * torch.randn(32, generator=g)).to(gpu), torch.randn(1, 2, 5, 32, generator=g).to(gpu)

    def loss(x, w):
        return (pa.qk_norm_rotate(x, x, w, w, interleaved=True)[0].double() * d).sum()
    x, w = x0.clone().requires_grad_(), w0.clone().requires_grad_()
    gx, gw = torch.autograd.grad(loss(x, w), [x, w])
    for v in (torch.randn(1, 2, 5, 32, generator=g).to(gpu),):
        h = 2.0 ** -7
        slope = (loss(x0 + h * v, w0) - loss(x0 - h * v, w0)) / (2 * h)
        # (third derivatives of order ten times the value's size, times h^2 / 6; the values' own roundings over h: 2^-19 * 2^7)
        assert abs(float(slope - (gx.double() * v).sum())) <= 2.0 ** -9 * float(gx.norm() * v.norm())
    v = torch.randn(32, generator=g).to(gpu)
    slope = (loss(x0, w0 + v) - loss(x0, w0 - v)) / 2                                    # linear in the weight
    assert abs(float(slope - (gw.double() * v).sum())) <= 2.0 ** -14 * float(gw.norm() * v.norm())


def test_recorded_backward_and_transforms_take_the_expression(gpu):
    g = torch.Generator().manual_seed(4)
    x, w = torch.randn(1, 2, 4, 32, generator=g).to(gpu).requires_grad_(), torch.ones(32, device=gpu, requires_grad=True)

    def second(f):
        y = f(x, x, w, w)[0]
        dx, = torch.autograd.grad((y ** 3).sum(), x, create_graph=True)
        return torch.autograd.grad((dx ** 2).sum(), [x, w])
    got = second(pa.qk_norm_rotate)
    want = second(lambda *a: qk_norm._expression(*a, None, None, 10000.0, 1e-6, False, torch.float32))
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= 1e-4 * b.abs().max()
    with torch.no_grad():
        xs = torch.randn(3, 1, 2, 4, 32, generator=g).to(gpu)
        rows = torch.func.vmap(lambda t: pa.qk_norm_rotate(t, t)[0])(xs)
        for i in range(3):
            assert (rows[i] - pa.qk_norm_rotate(xs[i], xs[i])[0]).abs().max() <= 1e-5


def test_saved_tensors_changed_in_place_are_an_error(gpu):
    x = torch.randn(1, 1, 4, 32, device=gpu).requires_grad_()
    h = x * 1.0
    y, _ = pa.qk_norm_rotate(h, h)
    h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


def test_same_bits_and_another_stream(gpu):
    g = torch.Generator().manual_seed(5)
    q = torch.randn(4, 8, 1000, 64, generator=g).bfloat16().to(gpu).requires_grad_()
    w = torch.ones(8, 64, device=gpu, requires_grad=True)
    d = torch.randn(4, 8, 1000, 64, generator=g).bfloat16().to(gpu)

    def step():
        y, _ = pa.qk_norm_rotate(q, q, w, w)
        return [y.detach(), *torch.autograd.grad(y, [q, w], d)]
    first = step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = step()
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


def test_captured_step_replays(gpu):
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(2, 100, 3, 4, 64, generator=g).to(gpu).requires_grad_()
    w = torch.ones(64, device=gpu, requires_grad=True)
    d = torch.randn(2, 100, 3, 4, 64, generator=g).bfloat16().to(gpu)

    def step():
        y = pa.qk_norm_rotate_qkv(qkv, w, w, out_dtype=torch.bfloat16)
        return [y.detach(), *torch.autograd.grad(y, [qkv, w], d)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(3):
        with torch.no_grad():
            qkv.copy_(torch.randn(qkv.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b), i


def test_empty_calls(gpu):
    for shape in ((0, 4, 10, 64), (2, 4, 0, 64)):
        q = torch.zeros(shape, device=gpu, requires_grad=True)
        w = torch.ones(64, device=gpu, requires_grad=True)
        y, z = pa.qk_norm_rotate(q, q, w, w)
        assert y.shape == z.shape == shape
        dx, dw = torch.autograd.grad(y.sum(), [q, w])
        assert dx.shape == shape and not dw.any()


@pytest.mark.parametrize("eps", [0.0, 1e-6])
@pytest.mark.parametrize("how", ["shared", "head"])
def test_recorded_backward_of_a_padded_batch_agrees_with_the_kernel(gpu, how, eps):
    """The expression's gradients and the kernel's, padded tokens and the gradients at their places not finite; both are within the bars above, of which 2^-14 of the
    largest element is more than two."""
    g = torch.Generator().manual_seed(8)
    Z, H, N, d = 3, 4, 21, 64
    mask = torch.arange(N)[None, :] >= torch.tensor([13, 21, 0])[:, None]
    x, dy = torch.randn(Z, H, N, d, generator=g), torch.randn(Z, H, N, d, generator=g)
    x.transpose(1, 2)[mask], dy.transpose(1, 2)[mask] = float("nan"), float("inf")
    x, dy = x.to(gpu).requires_grad_(), dy.to(gpu)
    w, _ = weights((H, H), d, how, FL, g, gpu)
    k = torch.randn(Z, H, N, d, generator=g).to(gpu)
    y, _ = pa.qk_norm_rotate(x, k, w, torch.ones_like(w), eps=eps, mask=mask.to(gpu))
    want = torch.autograd.grad(y, [x, w], dy, retain_graph=True)
    got = torch.autograd.grad(y, [x, w], dy, create_graph=True)
    for a, b in zip(got, want):
        assert torch.isfinite(b).all() and float((a.detach() - b).abs().max()) <= 2.0 ** -14 * float(b.abs().max())
    for t in (y, got[0], *torch.autograd.grad(sum(t.square().sum() for t in got), [x])):
        assert not t.detach().transpose(1, 2)[mask.to(gpu)].any() and torch.isfinite(t).all()


@pytest.mark.parametrize("base", [10000.0, 500.0, 0.3])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_angles_of_the_furthest_positions(gpu, d, base):
    """Angles against 60 decimal digits: off by at most 2^-52 of their number of turns (half a step of fp64 each for the frequency and for its product with the
    position), times 2 pi, and 2^-22 for what comes behind; two roundings of the pair's size, 2^-23, on top."""
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        two_pi = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494")
        D = decimal.Decimal
        turns = [D(base) ** (D(-2 * i) / D(d)) / two_pi for i in range(d // 2)]
        positions = [2 ** 40 + 12345, -(2 ** 41) - 77, 2 ** 42 - 1, 3 ** 26, 10 ** 7, -5, 0]
        rest = torch.tensor([[float(p * t - (p * t).to_integral_value()) for t in turns] for p in positions], dtype=torch.float64)
        size = torch.tensor([[float(abs(p * t)) for t in turns] for p in positions], dtype=torch.float64)
    for inter in (False, True):
        x = torch.zeros(1, 1, len(positions), d)
        pairs(x, inter)[0].fill_(1.0)                              # normed: (sqrt 2, 0) in every pair
        y, _ = pa.qk_norm_rotate(x.to(gpu), x.to(gpu), positions=torch.tensor(positions, device=gpu), base=base, eps=0.0, interleaved=inter)
        c, s = pairs(y[0, 0].double().cpu(), inter)
        bar = 2.0 ** 0.5 * (size * 2.0 ** -52 * 2 * math.pi + 2.0 ** -22 + 2.0 ** -23)
        for got, want in ((c, torch.cos(2 * math.pi * rest)), (s, torch.sin(2 * math.pi * rest))):
            off = (got - 2.0 ** 0.5 * want).abs()
            assert (off <= bar).all(), (float((off / bar).max()), int((off / bar).argmax()))
