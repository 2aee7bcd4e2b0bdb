"""GPU tests of the gated feed-forward block against its formulas in float64.

fp32 bars: products of K terms whose sums are at or below fp32's error, 2^-24 per step with signs at random over at most some 10^4 terms: 2-norms of the errors below 4e-6
(dz adds the activation's few roundings).
bf16 bars, element by element: the kernel rounds h and dz, each by at most 2^-8 of its size, z by 2^-12 of its, and its result by 2^-8.  An output is a sum over such numbers
times exact ones, so its error is a sum of independent terms bounded by b_i; it passes t sqrt(sum b_i^2) with a probability below 2 exp(-t^2 / 2), 5e-11 for
t = 7.  What the rounding of z does to dz: the value's part is off by 2^-12, act' by |act''(g) g| 2^-12 <= 0.6 * 2^-12 (all four functions), act by |act'(g) g| 2^-12."""
import copy
import ctypes
import math

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

import proteusai_amd as pa
from proteusai_amd import gated_mlp as gm_module  # noqa: F401
from proteusai_amd import train_ops

pytestmark = pytest.mark.gpu

BF, FL = torch.bfloat16, torch.float32
ACTS = {"silu": F.silu, "gelu": F.gelu, "relu": F.relu, "sigmoid": torch.sigmoid}


def make(rows, D, H, O, dtype, bias, gpu, seed=0, shape=None):
    g = torch.Generator().manual_seed(seed + rows)
    x = torch.randn(*(shape or (rows,)), D, generator=g)
    w, wo = torch.randn(2 * H, D, generator=g) * D ** -0.5, torch.randn(O, H, generator=g) * H ** -0.5
    b, bo = (torch.randn(2 * H, generator=g) * 0.3, torch.randn(O, generator=g) * 0.3) if bias else (None, None)
    d = torch.randn(*(shape or (rows,)), O, generator=g)
    return [None if t is None else t.to(dtype).to(gpu) for t in (x, w, b, wo, bo, d)]


def reference(x, w, b, wo, bo, d, act):
    """Outputs and the bf16 bars of each, in float64 on the GPU."""
    x, w, b, wo, bo, d = (None if t is None else t.detach().double() for t in (x, w, b, wo, bo, d))
    H = wo.shape[1]
    z = F.linear(x, w, b)
    g = z[..., :H].requires_grad_()
    a = ACTS[act](g)
    slope, = torch.autograd.grad(a.sum(), g)
    g, a, u = g.detach(), a.detach(), z[..., H:]
    h = a * u
    y = F.linear(h, wo, bo)
    dh = d @ wo
    dg, du = dh * u * slope, dh * a
    dz = torch.cat((dg, du), -1)
    outs = {"y": y, "dx": dz @ w, "dw": dz.t() @ x, "db": dz.sum(0), "dwo": d.t() @ h, "dbo": d.sum(0)}
    half = 2.0 ** -8
    bz = half * dz.abs() + 2.0 ** -12 * torch.cat((dh.abs() * u.abs() * (slope.abs() + 0.6), dh.abs() * (slope * g).abs()), -1)
    sq = {"y": (h * half).square() @ wo.square().t(), "dx": bz.square() @ w.square(), "dw": bz.square().t() @ x.square(), "db": bz.square().sum(0),
          "dwo": d.square().t() @ (h * half).square(), "dbo": torch.zeros(wo.shape[0], dtype=torch.float64, device=x.device)}
    bars = {k: 7 * sq[k].sqrt() + half * outs[k].abs() + 2.0 ** -20 * outs[k].abs().max() for k in outs}
    return outs, bars


def check(got, outs, bars, dtype):
    for k, v in got.items():
        assert v.dtype == dtype and v.shape == outs[k].shape, k
        off = (v.double() - outs[k]).abs()
        if dtype == BF:
            assert (off <= bars[k]).all(), (k, float((off / bars[k].clamp_min(1e-30)).max()))
        else:
            assert float(off.norm()) <= 4e-6 * float(outs[k].norm()) + 1e-30, (k, float(off.norm() / outs[k].norm()))


SIZES = [(1, 8, 8, 8), (1, 512, 2048, 512), (3, 64, 24, 40), (8, 512, 2048, 512), (16, 72, 200, 136), (17, 128, 64, 256), (33, 264, 136, 72), (64, 512, 1024, 512), (129, 96, 160, 64),
         (300, 32, 520, 40), (511, 512, 2048, 512), (1000, 712, 1912, 712), (2049, 256, 128, 248), (5003, 136, 264, 520), (9000, 64, 64, 64), (70_001, 8, 16, 8)]


@pytest.mark.parametrize("dtype", [BF, FL], ids=["bf16", "f32"])
@pytest.mark.parametrize("rows,D,H,O", SIZES)
def test_forward_and_gradients(gpu, rows, D, H, O, dtype):
    acts = list(ACTS)
    i = SIZES.index((rows, D, H, O))
    for act, bias in ((acts[i % 4], True), (acts[(i + 1) % 4], False)):
        x, w, b, wo, bo, d = make(rows, D, H, O, dtype, bias, gpu)
        leaves = [None if t is None else t.requires_grad_() for t in (x, w, b, wo, bo)]
        y = pa.gated_mlp(*leaves, act=act)
        names = [n for n, t in zip(("dx", "dw", "db", "dwo", "dbo"), leaves) if t is not None]
        got = dict(zip(names, torch.autograd.grad(y, [t for t in leaves if t is not None], d)), y=y.detach())
        outs, bars = reference(x, w, b, wo, bo, d, act)
        check(got, {k: outs[k] for k in got}, bars, dtype)
        with torch.no_grad():
            check({"y": pa.gated_mlp(*leaves, act=act)}, outs, bars, dtype)


@pytest.mark.parametrize("D,H", [(512, 2048), (1000, 136), (2056, 1096)])
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65])
def test_few_rows(gpu, rows, D, H):
    """Where a kernel of its own reads the weights once for all rows, and around its ends."""
    for i, act in enumerate(ACTS):
        x, w, b, wo, bo, d = make(rows, D, H, D, BF, i % 2 == 0, gpu, seed=i)
        outs, bars = reference(x, w, b, wo, bo, d, act)
        check({"y": pa.gated_mlp(x, w, b, wo, bo, act=act)}, outs, bars, BF)
        leaves = [t for t in (x.requires_grad_(), w.requires_grad_(), b, wo, bo)]
        y = pa.gated_mlp(*leaves, act=act)
        got = torch.autograd.grad(y, [x, w], d)
        check({"y": y.detach(), "dx": got[0], "dw": got[1]}, outs, bars, BF)


@pytest.mark.parametrize("dtype", [BF, FL], ids=["bf16", "f32"])
def test_gradients_left_out(gpu, dtype):
    x, w, b, wo, bo, d = make(130, 64, 96, 72, dtype, True, gpu)
    everything = [t.clone().requires_grad_() for t in (x, w, b, wo, bo)]
    want = torch.autograd.grad(pa.gated_mlp(*everything), everything, d)
    for keep in range(1, 32):
        leaves = [t.clone().requires_grad_(bool(keep >> i & 1)) for i, t in enumerate((x, w, b, wo, bo))]
        got = iter(torch.autograd.grad(pa.gated_mlp(*leaves), [t for t in leaves if t.requires_grad], d))
        for i in range(5):
            if keep >> i & 1:
                assert torch.equal(next(got), want[i]), (keep, i)


def test_gradient_against_differences(gpu):
    x, w, b, wo, bo, d = make(5, 16, 24, 12, FL, True, gpu)
    leaves = [t.requires_grad_() for t in (x, w, b, wo, bo)]
    for act in ("silu", "gelu", "sigmoid"):
        grads = torch.autograd.grad(pa.gated_mlp(*leaves, act=act), leaves, d)
        g = torch.Generator().manual_seed(1)
        for i, grad in enumerate(grads):
            v, h = torch.randn(leaves[i].shape, generator=g).to(gpu), 2.0 ** -7

            def loss(s):
                with torch.no_grad():
                    return float((pa.gated_mlp(*[t + s * v if j == i else t for j, t in enumerate(leaves)], act=act).double() * d).sum())
            slope = (loss(h) - loss(-h)) / (2 * h)
            # (the third derivative's part is of order h^2 of the slope's terms; rounding of the two sums: 2^-21 of their size over h)
            assert abs(slope - float((grad.double() * v).sum())) <= 2.0 ** -8 * float(grad.norm() * v.norm()) + 2e-3, (act, i)


def test_layouts_and_leading_shapes(gpu):
    for dtype in (BF, FL):
        x, w, b, wo, bo, _ = make(60, 64, 96, 72, dtype, True, gpu)
        want = pa.gated_mlp(x, w, b, wo, bo)
        assert torch.equal(pa.gated_mlp(x.view(3, 4, 5, 64), w, b, wo, bo), want.view(3, 4, 5, 72))
        assert torch.equal(pa.gated_mlp(x[7], w, b, wo, bo), pa.gated_mlp(x[7:8], w, b, wo, bo)[0])
        wide = torch.empty(60, 3, 64, dtype=dtype, device=gpu)
        wide[:, 1] = x
        assert torch.equal(pa.gated_mlp(wide[:, 1], w, b, wo, bo), want)
        odd = torch.empty(60 * 64 + 1, dtype=dtype, device=gpu)[1:].view(60, 64)
        odd.copy_(x)
        assert torch.equal(pa.gated_mlp(odd, w, b, wo, bo), want)
        assert torch.equal(pa.gated_mlp(x, w.t().contiguous().t(), b, wo.t().contiguous().t(), bo), want)
        one = x[:1].expand(60, 64).detach().requires_grad_()
        y = pa.gated_mlp(one, w, b, wo, bo)
        dx, = torch.autograd.grad(y.sum(), one)                        # (a gradient without strides)
        leaf = one.detach().contiguous().requires_grad_()
        want_dx, = torch.autograd.grad(pa.gated_mlp(leaf, w, b, wo, bo), leaf, torch.ones_like(y))
        assert torch.equal(dx, want_dx)


def test_not_finite_values_stay_in_their_rows(gpu):
    for dtype in (BF, FL):
        x, w, b, wo, bo, _ = make(300, 64, 96, 72, dtype, True, gpu)
        want = pa.gated_mlp(x, w, b, wo, bo)
        x[17], x[255, 3] = float("nan"), float("inf")
        got = pa.gated_mlp(x, w, b, wo, bo)
        keep = torch.ones(300, dtype=torch.bool, device=gpu)
        keep[17] = keep[255] = False
        assert torch.equal(got[keep], want[keep]) and got[17].isnan().all() and not torch.isfinite(got[255]).all()
        large = torch.full((4, 64), 100.0, dtype=dtype, device=gpu)    # saturated gates on either side
        for act in ACTS:
            y = pa.gated_mlp(large, torch.cat((w[:96].abs(), w[96:])), None, wo, None, act=act)
            z = pa.gated_mlp(large, torch.cat((-w[:96].abs(), w[96:])), None, wo, None, act=act)
            assert torch.isfinite(y).all() and float(z.abs().max()) <= 1e-2 * float(y.abs().max())


def test_same_bits_another_stream_and_replays(gpu):
    for dtype in (BF, FL):
        x, w, b, wo, bo, d = make(3000, 128, 256, 128, dtype, True, gpu)
        leaves = [t.requires_grad_() for t in (x, w, b, wo, bo)]

        def step():
            y = pa.gated_mlp(*leaves)
            return [y.detach(), *torch.autograd.grad(y, leaves, d)]
        first = step()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            second = step()
        torch.cuda.current_stream().wait_stream(stream)
        assert all(torch.equal(a, b_) for a, b_ in zip(first, second))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        g = torch.Generator().manual_seed(2)
        for i in range(3):
            with torch.no_grad():
                x.copy_(torch.randn(x.shape, generator=g))
                w.mul_(1.1)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b_) for a, b_ in zip(held, step())), i


def test_what_takes_the_expression(gpu):
    x, w, b, wo, bo, _ = make(9, 16, 24, 16, FL, True, gpu)
    xd = x.clone().requires_grad_()

    def second(f):
        dx, = torch.autograd.grad((f(xd) ** 3).sum(), xd, create_graph=True)
        return torch.autograd.grad((dx ** 2).sum(), xd)[0]
    want = second(lambda t: pa.gated_mlp.__globals__["_expression"](t, w, b, wo, bo, "silu"))
    got = second(lambda t: pa.gated_mlp(t, w, b, wo, bo))
    assert float((got - want).norm()) <= 1e-4 * float(want.norm())
    rows = torch.func.vmap(lambda t: pa.gated_mlp(t, w, b, wo, bo))(x.view(3, 3, 16))
    assert float((rows.reshape(9, 16) - pa.gated_mlp(x, w, b, wo, bo)).abs().max()) <= 1e-5
    with torch.autocast("cuda", dtype=BF):
        assert pa.gated_mlp(x, w, b, wo, bo).dtype == BF
    y = pa.gated_mlp(xd, w, b, wo, bo)
    with torch.autocast("cuda", dtype=BF):                              # (a backward called inside)
        inside, = torch.autograd.grad(y.sum(), xd)
    outside, = torch.autograd.grad(pa.gated_mlp(xd, w, b, wo, bo).sum(), xd)
    assert torch.equal(inside, outside)
    assert pa.gated_mlp(x[:0], w, b, wo, bo).shape == (0, 16)


@pytest.mark.parametrize("dtype", [BF, FL], ids=["bf16", "f32"])
@pytest.mark.parametrize("bias", [True, False])
def test_module(gpu, dtype, bias):
    torch.manual_seed(0)
    m = pa.GatedMLP(64, 72, 96, dropout=0.0, act="gelu", bias=bias).to(gpu, dtype)
    if bias:
        with torch.no_grad():
            for p in (m.in_proj.bias, m.out_proj.bias):
                p.normal_(0, 0.3)
    x, d = torch.randn(2, 65, 64, device=gpu).to(dtype).requires_grad_(), torch.randn(2, 65, 72, device=gpu).to(dtype)
    y = m(x)
    got = torch.autograd.grad(y, [x, *m.parameters()], d)
    assert torch.equal(y, pa.gated_mlp(x, m.in_proj.weight, m.in_proj.bias, m.out_proj.weight, m.out_proj.bias, act="gelu"))
    other = copy.deepcopy(m)
    other.out_proj.register_forward_hook(lambda *a: None)               # (a hook: the expression)
    ref = other(x)
    want = torch.autograd.grad(ref, [x, *other.parameters()], d)
    for a, b in zip((y, *got), (ref, *want)):
        assert a.shape == b.shape and float((a - b).norm()) <= (2.0 ** -6 if dtype == BF else 4e-6) * float(b.norm())
    m.dropout.p = 0.5
    assert (m(x) != y).any()
    m.eval()
    assert torch.equal(m(x), y)
    assert isinstance(nn.Sequential(m, nn.Linear(72, 3).to(gpu, dtype))(x), torch.Tensor)
    assert m.half()(x.half()).dtype == torch.float16                    # (another type: the expression)


def test_saved_tensors_given_back_otherwise(gpu):
    x, w, b, wo, bo, d = make(40, 64, 96, 72, BF, True, gpu)
    leaves = [t.requires_grad_() for t in (x, w, b, wo, bo)]
    want = torch.autograd.grad(pa.gated_mlp(*leaves), leaves, d)

    def pack(t):
        return t.cpu()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(gpu)):
        y = pa.gated_mlp(*leaves)
    assert all(torch.equal(a, b_) for a, b_ in zip(torch.autograd.grad(y, leaves, d), want))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:-1]):
        y = pa.gated_mlp(*leaves)
    with pytest.raises(RuntimeError, match="came back"):
        torch.autograd.grad(y, leaves, d)
    y = pa.gated_mlp(*leaves)
    with torch.no_grad():
        w.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(y, leaves, d)


def test_workspaces_are_asked_for_as_documented(gpu):
    lib = train_ops._lib.load()
    assert lib.proteus_gated_mlp_kept_bytes(10, 64, 96, 72, 0) > 0 and lib.proteus_gated_mlp_kept_bytes(10, 62, 96, 72, 0) == 0


LARGE = [(8192, 512, 2048, 512, BF), (20_000, 264, 1000, 520, BF), (12_345, 1032, 2056, 1032, BF), (40_001, 520, 1048, 512, BF), (2048, 4096, 2048, 4096, BF), (65_537, 136, 264, 136, BF),
         (2048, 512, 2048, 512, FL), (4099, 516, 1100, 520, FL), (700, 1028, 2052, 512, FL), (1000, 2048, 1236, 128, FL)]


@pytest.mark.parametrize("rows,D,H,O,dtype", LARGE, ids=lambda v: str(v).replace("torch.", ""))
def test_many_tiles(gpu, rows, D, H, O, dtype):
    """Sizes of several tiles for each workgroup, of ragged last ones, of shares of K, and the ones from which fp32's gate is in the product's launch."""
    for act, bias in ((list(ACTS)[LARGE.index((rows, D, H, O, dtype)) % 4], True), ("silu", False)):
        x, w, b, wo, bo, d = make(rows, D, H, O, dtype, bias, gpu)
        leaves = [t.requires_grad_() for t in (x, w, b, wo, bo) if t is not None]
        y = pa.gated_mlp(x, w, b, wo, bo, act=act)
        names = [n for n, t in zip(("dx", "dw", "db", "dwo", "dbo"), (x, w, b, wo, bo)) if t is not None]
        got = dict(zip(names, torch.autograd.grad(y, leaves, d)), y=y.detach())
        outs, bars = reference(x, w, b, wo, bo, d, act)
        check(got, {k: outs[k] for k in got}, bars, dtype)
        with torch.no_grad():
            assert torch.equal(pa.gated_mlp(x, w, b, wo, bo, act=act), y)


@pytest.mark.parametrize("dtype", [BF, FL], ids=["bf16", "f32"])
def test_not_finite_values_among_many_tiles(gpu, dtype):
    """A row and a feature that are not finite: what reads neither keeps its bits."""
    x, w, b, wo, bo, d = make(4100, 512, 1100 if dtype == FL else 1104, 64, dtype, True, gpu)
    F_ = wo.shape[1]
    leaves = [t.requires_grad_() for t in (x, w, wo)]

    def run():
        y = pa.gated_mlp(x, w, b, wo, bo)
        return [y.detach(), *torch.autograd.grad(y, leaves, d)]
    want = run()
    with torch.no_grad():
        x[1234, 5] = float("inf")
        x[4099] = float("nan")
    got = run()
    rows = torch.ones(4100, dtype=torch.bool, device=gpu)
    rows[1234] = rows[4099] = False
    assert torch.equal(got[0][rows], want[0][rows]) and torch.equal(got[1][rows], want[1][rows])
    assert got[0][4099].isnan().all() and got[1][4099].isnan().all() and not torch.isfinite(got[0][1234]).any()
    assert got[2].isnan().all() and got[3].isnan().all()
    with torch.no_grad():
        x[1234], x[4099] = 0.0, 0.0
        d[:, 7] = 0.0
        wo[:, 300], wo[:, F_ - 1] = 0.0, 0.0
    want = run()
    with torch.no_grad():
        w[300, 3], w[2 * F_ - 1, 4] = float("nan"), float("inf")
    got = run()
    features = torch.ones(F_, dtype=torch.bool, device=gpu)
    features[300] = features[F_ - 1] = False
    assert torch.equal(got[2][features.repeat(2)], want[2][features.repeat(2)]) and torch.equal(got[3][:, features], want[3][:, features])
    assert got[0].isnan().any(1).all() and got[3][:, 300].isnan().any()


def test_offsets_beyond_32_bits(gpu):
    """z of 4.9 GB: rows from either end against the formula, the gradients of the weights against its sums over shares of the rows."""
    rows, D, H, O, act = 600_011, 64, 2048, 64, "silu"
    x, w, b, wo, bo, d = make(rows, D, H, O, BF, True, gpu)
    leaves = [t.requires_grad_() for t in (x, w, b, wo, bo)]
    y = pa.gated_mlp(*leaves, act=act)
    got = dict(zip(("dx", "dw", "db", "dwo", "dbo"), torch.autograd.grad(y, leaves, d)), y=y.detach())
    step, sums, bars = 60_000, {}, {}
    half = 2.0 ** -8
    for r in range(0, rows, step):
        at = slice(r, min(rows, r + step))
        outs, bar = reference(x[at], w, b, wo, bo, d[at], act)
        check({"y": got["y"][at], "dx": got["dx"][at]}, outs, bar, BF)
        for k in ("dw", "db", "dwo", "dbo"):
            # (of a share's bar the part that is not of its own rounding and size, in squares)
            own = ((bar[k] - half * outs[k].abs() - 2.0 ** -20 * outs[k].abs().max()) / 7).clamp_min(0.0).square()
            sums[k], bars[k] = sums.get(k, 0.0) + outs[k], bars.get(k, 0.0) + own
    bars = {k: 7 * bars[k].sqrt() + half * sums[k].abs() + 2.0 ** -20 * sums[k].abs().max() for k in bars}
    check({k: got[k] for k in sums}, sums, bars, BF)


@pytest.mark.parametrize("rows", [5, 300, 9000])
@pytest.mark.parametrize("bits", [0x7fc0, 0x7fff, 0xffff - 0x10000, 0x7f81], ids=hex)
def test_every_kind_of_nan_comes_back(gpu, rows, bits):
    """A NaN of any payload in x is one in what is kept for the backward."""
    x, w, b, wo, bo, d = make(rows, 64, 2048, 64, BF, True, gpu)
    x.view(torch.int16)[rows // 2, 7] = bits
    x.requires_grad_()
    y = pa.gated_mlp(x, w, b, wo, bo)
    dx, = torch.autograd.grad(y, x, d)
    keep = torch.arange(rows, device=gpu) != rows // 2
    assert y[rows // 2].isnan().all() and dx[rows // 2].isnan().all()
    assert torch.isfinite(y[keep]).all() and torch.isfinite(dx[keep]).all()


@pytest.mark.parametrize("rows,D,H,O", [(5, 16, 128, 16), (100, 64, 256, 64), (300, 64, 2056, 64), (1000, 64, 2056, 64)])
def test_bias_gradients_beside_an_infinite_weight(gpu, rows, D, H, O):
    """An infinite weight of the way down makes the gradients of its feature's biases infinite, whatever the number of rows: what a tile has beyond the last row
    (zeros, whose product with it is NaN) is not among them.  All the terms are positive."""
    x, w, b, wo, bo, d = make(rows, D, H, O, BF, True, gpu)
    w.mul_(0.01)
    b.fill_(2.0)
    d.abs_().add_(0.125)
    leaves = [t.requires_grad_() for t in (x, w, b, wo, bo)]
    want = torch.autograd.grad(pa.gated_mlp(*leaves), leaves, d)[2]
    with torch.no_grad():
        wo[3, 7] = float("inf")
    got = torch.autograd.grad(pa.gated_mlp(*leaves), leaves, d)[2]
    assert got[7] == float("inf") and got[H + 7] == float("inf")
    keep = torch.arange(2 * H, device=gpu) % H != 7
    assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("rows", [40, 1500, 20_000])
def test_gelu_far_below_zero(gpu, rows):
    """GELU of a bf16 gate down to -12.5, where its tail is 10^-35, and its slope: what they are off by beside the rounding of the result (half a step, 2^-8) stays
    below 2^-12 of the tail's terms.  One feature of the block is the function itself: gate x, value 1, passed on by weights of one."""
    g = torch.exp(torch.linspace(math.log(0.01), math.log(12.5), rows)).neg().to(BF)
    x = torch.zeros(rows, 8)
    x[:, 0], x[:, 1] = g.float(), 1.0
    w, wo = torch.zeros(16, 8), torch.zeros(8, 8)
    w[0, 0] = w[8, 1] = wo[0, 0] = 1.0
    x, w, wo = (t.to(BF).to(gpu).requires_grad_() for t in (x, w, wo))
    with torch.no_grad():
        alone = pa.gated_mlp(x, w, None, wo, None, act="gelu")
    y = pa.gated_mlp(x, w, None, wo, None, act="gelu")
    d = torch.zeros_like(y)
    d[:, 0] = 1.0
    dx, = torch.autograd.grad(y, x, d)
    g = g.double()
    tail, bell = 0.5 * torch.special.erfc(-g / 2 ** 0.5), torch.exp(-0.5 * g * g) / (2 * math.pi) ** 0.5
    half, more = 2.0 ** -8, 2.0 ** -12
    for got, want, terms in ((y, g * tail, (g * tail).abs()), (alone, g * tail, (g * tail).abs()), (dx, tail + g * bell, tail + (g * bell).abs())):
        off = (got[:, 0].detach().double().cpu() - want).abs()
        bar = half * want.abs() + (1 + half) * more * terms
        assert (off <= bar).all(), (float((off / bar).max()), float(g[(off / bar).argmax()]))


# (few rows; tiles of 64 x 128, 128 x 128 and 256 x 256; the three products behind dz together and apart; fp32 with the gate in the product and behind it)
EXACT_BYTES = [(1, 8, 8, 8, BF), (5, 512, 2048, 512, BF), (40, 512, 2048, 512, BF), (33, 264, 136, 72, BF), (300, 512, 2048, 512, BF), (1000, 712, 1912, 712, BF), (5003, 712, 1912, 712, BF),
               (9000, 64, 64, 64, BF), (32_768, 1024, 4096, 1024, BF), (70_001, 8, 16, 8, BF), (3, 64, 24, 40, FL), (700, 1028, 2052, 512, FL), (2048, 512, 2048, 512, FL), (4099, 516, 1100, 520, FL)]


@pytest.mark.parametrize("rows,D,H,O,dtype", EXACT_BYTES, ids=lambda v: str(v).replace("torch.", ""))
def test_nothing_is_written_beside_the_bytes_asked_for(gpu, rows, D, H, O, dtype):
    """The library's own entry points with everything they write in the middle of a buffer of a pattern, of exactly the bytes that they ask for: the results are the operator's
    bit for bit, and the pattern around them stays."""
    lib, beside = train_ops._lib.load(), 1 << 16
    x, w, b, wo, bo, d = make(rows, D, H, O, dtype, True, gpu)
    leaves = [t.requires_grad_() for t in (x, w, b, wo, bo)]
    y = pa.gated_mlp(*leaves)
    want = [y.detach(), *torch.autograd.grad(y, leaves, d)]
    leaves = [t.detach() for t in leaves]
    held = []

    def room(n):
        t = torch.full((n + 2 * beside,), 0xA5, dtype=torch.uint8, device=gpu)
        assert t.data_ptr() % 256 == 0
        held.append((t, n))
        return t[beside:beside + n]

    def pointers(ts):
        return (ctypes.c_void_p * 4)(*[t.data_ptr() for t in ts])
    sizes = rows, D, H, O, train_ops._lib.DTYPE_BF16 if dtype == BF else train_ops._lib.DTYPE_F32
    kept, forward, train, backward = (room(getattr(lib, f"proteus_gated_mlp_{n}_bytes")(*sizes)) for n in ("kept", "fwd", "train_fwd", "bwd"))
    out, alone = room(y.numel() * y.element_size()), room(y.numel() * y.element_size())
    grads = [room(t.numel() * t.element_size()) for t in leaves]
    params, stream = pointers(leaves[1:]), torch.cuda.current_stream().cuda_stream
    assert lib.proteus_gated_mlp_fwd(x.data_ptr(), params, out.data_ptr(), kept.data_ptr(), kept.numel(), train.data_ptr(), train.numel(), *sizes[:4], 0, sizes[4], stream) == 0
    assert lib.proteus_gated_mlp_fwd(x.data_ptr(), params, alone.data_ptr(), None, 0, forward.data_ptr(), forward.numel(), *sizes[:4], 0, sizes[4], stream) == 0
    assert lib.proteus_gated_mlp_bwd(x.data_ptr(), params, d.data_ptr(), grads[0].data_ptr(), pointers(grads[1:]), kept.data_ptr(), kept.numel(), backward.data_ptr(), backward.numel(),
                                     *sizes[:4], 0, sizes[4], stream) == 0
    for got, t in zip((out, alone, *grads), (want[0], *want)):
        assert torch.equal(got.view(dtype).view(t.shape), t)
    for t, n in held:
        assert (t[:beside] == 0xA5).all() and (t[beside + n:] == 0xA5).all()
