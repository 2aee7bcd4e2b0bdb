"""GPU tests of the cross entropy from features against its definition in float64.

Bars.  u = 2^-24, h = half a step of the type (2^-9 relative to the next power of two for bf16: eps / 2).  A logit is a sum of D products, exact ones for 16-bit operands and off by 2^-24 of their size in fp32, in
fp32 accumulators: off by e = (D / 8 + 16) u of the sum of their sizes (a matrix instruction adds 16 products; twice that for the order inside it).  The loss is off by 2 e and 16 u of the
logarithm and its terms.  P by 4 e + 32 u of itself for its exponential and factor, and h for its rounding (fp32: 4 u); a gradient by that of the sum of sizes |P| |W|, by (n / 8 + 16) u of it for its own sums over n
terms, and by its own rounding h.  fp16's P ends at 2^-25 / 2^15 of the largest weight."""
import math

import pytest
import torch

import proteusai_amd as pa

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def make(M, D, V, dtype, gpu, seed=0, bias=True, left_out=0.2, spread=2.0):
    g = torch.Generator(device=gpu).manual_seed(seed)
    w = torch.randn(V, D, generator=g, device=gpu) * spread * D ** -0.5
    target = torch.randint(0, V, (M,), generator=g, device=gpu)
    x = torch.randn(M, D, generator=g, device=gpu) + w[target] * (4 / spread * torch.rand(M, 1, generator=g, device=gpu))
    if left_out:
        target[torch.rand(M, generator=g, device=gpu) < left_out] = -100
    b = torch.randn(V, generator=g, device=gpu).to(dtype) if bias else None
    return x.to(dtype), w.to(dtype), b, target


def exact(x, w, b, target, smoothing=0.0, reduction="mean", d=None, ignore=-100, fine=False):
    """Loss, gradients and their bars in float64, tokens in pieces.  fine: P of 16-bit operands in two pieces, each off by h of what is left for it (and 2^-9 of an fp16 step's end, above)."""
    V, D = w.shape
    dtype = x.dtype
    h = torch.finfo(dtype).eps / 2
    w64, b64 = w.detach().double(), None if b is None else b.detach().double()
    counts = target != ignore
    n = int(counts.sum())
    weight = counts.double() * (d.double() if reduction == "none" else 1.0 / max(n, 1) if reduction == "mean" else 1.0)
    losses, bars, dxs, dx_bars = [], [], [], []
    dw, dw_bar = torch.zeros_like(w64), torch.zeros_like(w64)
    db, db_bar = torch.zeros(V, dtype=torch.float64, device=w.device), torch.zeros(V, dtype=torch.float64, device=w.device)
    for i in range(0, len(target), 4096):
        xs = x.detach()[i:i + 4096].double()
        xs = torch.where(counts[i:i + 4096, None], xs, 0.0)
        at = torch.where(counts, target, 0)[i:i + 4096]
        wt = weight[i:i + 4096, None]
        l = xs @ w64.t() + (0.0 if b is None else b64)
        sizes = xs.abs() @ w64.abs().t() + (0.0 if b is None else b64.abs())
        e = (D / 8 + 16) * U * sizes.nan_to_num(0.0, 0.0, 0.0).amax(1)
        lp = torch.log_softmax(l, 1)
        hot = torch.zeros_like(lp).scatter_(1, at[:, None], 1.0)
        own = -lp.gather(1, at[:, None])[:, 0]
        losses.append(torch.where(counts[i:i + 4096], (1 - smoothing) * own - (smoothing * lp.mean(1) if smoothing else 0.0), 0.0))
        bars.append(2 * e + 16 * U * (l.logsumexp(1).abs() + l.abs().nan_to_num(0.0, 0.0, 0.0).amax(1) + own))
        p = lp.exp()
        missed = 1 - hot * 1.0
        miss = torch.where(hot > 0, (p * missed).sum(1, keepdim=True), p)     # of the own word what it lacks
        P = (torch.where(hot > 0, -miss, p) + smoothing * (hot - 1.0 / V)) * wt
        term = (miss + smoothing * (hot + 1.0 / V)) * wt.abs()
        off = term * (4 * e[:, None] + 32 * U) + P.abs() * (4 * U if dtype == F32 else h * h + 4 * U if fine else h)
        if dtype == F16:
            off = off + 2.0 ** -40 * weight.abs().max()
        dxs.append(P @ w64)
        dx_bars.append(off @ w64.abs() + (V / 8 + 16) * U * (P.abs() @ w64.abs()))
        dw += P.t() @ xs
        dw_bar += off.t() @ xs.abs() + (n / 8 + 16) * U * (P.abs().t() @ xs.abs())
        db += P.sum(0)
        db_bar += off.sum(0) + (n / 8 + 16) * U * P.abs().sum(0)
    loss, bar = torch.cat(losses), torch.cat(bars)
    if reduction != "none":
        k = (n if n else math.nan) if reduction == "mean" else 1.0
        loss, bar = loss.sum() / k, (bar * counts).sum() / k + U * loss.sum().abs() / k
    else:
        bar = torch.where(counts, bar, 0.0)
    grads = [torch.cat(dxs), dw] + ([] if b is None else [db])
    gbars = [torch.cat(dx_bars), dw_bar] + ([] if b is None else [db_bar])
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return loss, bar, grads, [q * 1.001 + (g.abs() + q) * (h + 4 * U) + tiny for g, q in zip(grads, gbars)]


def off(got, want, bar, what):
    assert got.shape == want.shape
    d = (got.double() - want).abs()
    assert bool((d <= bar).all()), f"{what}: {float((d / bar.clamp_min(1e-300)).max()):.3g} of the bar"


def check(x, w, b, target, smoothing=0.0, reduction="mean", seed=5):
    d = torch.rand(len(target), generator=torch.Generator(device=x.device).manual_seed(seed), device=x.device) - 0.3 if reduction == "none" else None
    loss, bar, grads, bars = exact(x, w, b, target, smoothing, reduction, d)
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b) if t is not None]
    got = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2] if b is not None else None, label_smoothing=smoothing, reduction=reduction)
    assert got.dtype == F32 and got.requires_grad
    off(got.detach(), loss, bar, "loss")
    with torch.no_grad():
        assert torch.equal(pa.linear_cross_entropy(x, w, target, b, label_smoothing=smoothing, reduction=reduction), got.detach())
    for name, g, want, q, leaf in zip(("dx", "dw", "db"), torch.autograd.grad(got, leaves, d), grads, bars, leaves):
        assert g.dtype == leaf.dtype
        off(g, want, q, name)


SIZES = [(1, 8, 1), (1, 8, 2), (3, 24, 2), (20, 512, 20), (64, 64, 33), (65, 40, 127), (127, 72, 128), (130, 512, 129), (33, 8, 1000), (300, 128, 257), (1000, 712, 1003), (2, 1032, 8001), (5003, 64, 20), (700, 2048, 60),
         (1, 64, 70_001), (30_000, 16, 5), (33, 48, 32), (31, 24, 64), (95, 136, 63), (64, 264, 65), (8200, 520, 31), (700, 2048, 90)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
def test_sizes(gpu, size, dtype):
    check(*make(*size, dtype, gpu, seed=sum(size), left_out=0.0 if size[0] < 3 else 0.2))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("V", [300, 20])
def test_forms(gpu, dtype, reduction, smoothing, bias, V):
    check(*make(150, 64, V, dtype, gpu, seed=3, bias=bias), smoothing, reduction)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("size", [(1, 64, 70), (2, 136, 30_693), (2, 1136, 111), (17, 40, 1001), (64, 264, 5003), (5, 2048, 300)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("reduction", ["none", "mean"])
def test_few_tokens(gpu, size, dtype, reduction):
    """Up to 64 of them: gradients are off by their own rounding, not by that of the logits' gradient, which nothing averages out."""
    x, w, b, target = make(*size, dtype, gpu, seed=sum(size), left_out=0.2 if size[0] > 4 else 0.0)
    d = torch.rand(size[0], device=gpu) + 0.1 if reduction == "none" else None
    loss, bar, grads, bars = exact(x, w, b, target, 0.1, reduction, d, fine=True)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], label_smoothing=0.1, reduction=reduction)
    off(got.detach(), loss, bar, "loss")
    for name, g, want, q in zip(("dx", "dw", "db"), torch.autograd.grad(got, leaves, d), grads, bars):
        off(g, want, q, name)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("size,bias", [((4100, 512, 8200), True), ((9000, 256, 2048), False), ((2100, 72, 20_011), True)], ids=str)
def test_large_tiles(gpu, size, bias, dtype):
    check(*make(*size, dtype, gpu, seed=7, bias=bias, left_out=0.1), 0.1 if bias else 0.0)


@pytest.mark.parametrize("dtype", [BF16, F32], ids=lambda t: str(t).split(".")[-1])
def test_several_pieces_of_the_vocabulary(gpu, dtype):
    """20000 x 30011 gradients of logits: over 1 GB in either type, so in pieces."""
    check(*make(20_000, 64, 30_011, dtype, gpu, seed=8, left_out=0.3), 0.1, "none")


def test_few_tokens_and_several_pieces(gpu):
    """64 x 4.3 million gradients of logits, two numbers each: over 1 GB."""
    x, w, b, target = make(64, 8, 4_300_000, BF16, gpu, seed=2)
    loss, bar, grads, bars = exact(x, w, b, target, fine=True)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
    off(got.detach(), loss, bar, "loss")
    for name, g, want, q in zip(("dx", "dw", "db"), torch.autograd.grad(got, leaves), grads, bars):
        off(g, want, q, name)


def test_fp32_columns_that_are_no_multiple_of_8(gpu):
    for D in (4, 12, 508):
        check(*make(70, D, 90, F32, gpu, seed=D))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("which", ["all", "first", "last", "all but one", "in blocks"])
@pytest.mark.parametrize("V", [100, 20])
def test_tokens_that_are_left_out(gpu, dtype, which, V):
    """What lies in their features and (by token) in the gradient of their loss is not read."""
    x, w, b, target = make(600, 64, V, dtype, gpu, seed=9, left_out=0.0)
    gone = torch.zeros(600, dtype=torch.bool, device=gpu)
    gone[{"all": slice(None), "first": slice(0, 300), "last": slice(300, None), "all but one": slice(1, None), "in blocks": slice(0, 512)}[which]] = True
    target = torch.where(gone, -100, target)
    for reduction in ("mean", "sum", "none"):
        d = torch.rand(600, device=gpu) if reduction == "none" else None
        loss, bar, grads, bars = exact(x, w, b, target, 0.1, reduction, d)
        bad = torch.where(gone[:, None], float("nan"), x.float()).to(dtype)
        bad[::2] = torch.where(gone[::2, None], float("inf"), x[::2].float()).to(dtype)
        leaves = [t.clone().requires_grad_() for t in (bad, w, b)]
        got = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], label_smoothing=0.1, reduction=reduction)
        if d is not None:
            d = torch.where(gone, float("nan"), d)
            assert bool((got[gone] == 0).all())
        if which == "all" and reduction == "mean":
            assert math.isnan(float(got.detach()))
        else:
            off(got.detach(), loss, bar, "loss")
        dx, dw, db = torch.autograd.grad(got, leaves, d)
        assert bool((dx[gone] == 0).all())
        for g, want, q in zip((dx, dw, db), grads, bars):
            off(g, want, q, "gradient")


@pytest.mark.parametrize("V", [30, 130])
def test_ignore_index(gpu, V):
    x, w, b, target = make(100, 64, V, BF16, gpu, left_out=0.0)
    target[40] = 3
    for ignore in (3, -1, 2 ** 40):
        t = target.clone()
        if ignore != 3:
            t[::3] = ignore
        keep = t != ignore
        got = pa.linear_cross_entropy(x, w, t, b, ignore_index=ignore, reduction="none")
        want = pa.linear_cross_entropy(x[keep], w, t[keep], b, reduction="none")
        assert torch.equal(got[keep], want) and bool((got[~keep] == 0).all()) and 0 < int(keep.sum()) < 100
        leaf = w.clone().requires_grad_()
        mean = pa.linear_cross_entropy(x, leaf, t, b, ignore_index=ignore)
        loss, bar, grads, bars = exact(x, w, b, t, ignore=ignore)
        off(mean.detach(), loss, bar, "loss")
        off(torch.autograd.grad(mean, leaf)[0], grads[1], bars[1], "dw")


@pytest.mark.parametrize("V", [30, 130, 300])
def test_targets_outside_of_the_vocabulary(gpu, V):
    """NaN for that token and what it goes into, nothing else, and no access outside."""
    for dtype in (BF16, F16, F32):
        x, w, b, target = make(100, 64, V, dtype, gpu, left_out=0.0)
        for bad in (V, V + 1, -1, 2 ** 40, -2 ** 62):
            t = target.clone()
            t[7] = bad
            leaf = x.clone().requires_grad_()
            loss = pa.linear_cross_entropy(leaf, w, t, b, reduction="none")
            dx, = torch.autograd.grad(loss, leaf, torch.ones(100, device=gpu))
            rest = torch.arange(100, device=gpu) != 7
            assert torch.isnan(loss[7]) and torch.isfinite(loss[rest]).all() and torch.isnan(dx[7]).all() and torch.isfinite(dx[rest]).all()
            assert math.isnan(float(pa.linear_cross_entropy(x, w, t, b)))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("V", [200, 62])
def test_words_that_are_shut_out(gpu, dtype, V):
    """A bias of -infinity for words that cannot be: no gradient for them, and only an infinite loss where one is wanted all the same.  A bias at the type's lowest value does the same."""
    for low in (-math.inf, torch.finfo(dtype).min):
        x, w, b, target = make(300, 64, V, dtype, gpu, seed=4, left_out=0.1)
        b[50:] = low
        target = torch.where(target >= 0, target % 50, target)
        loss, bar, grads, bars = exact(x, w[:50], b[:50], target)
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        got = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
        off(got.detach(), loss, bar, "loss")
        dx, dw, db = torch.autograd.grad(got, leaves)
        off(dx, grads[0], bars[0] * 4, "dx")          # (sums over four times as many words)
        off(dw[:50], grads[1], bars[1], "dw")
        assert bool((dw[50:] == 0).all()) and bool((db[50:] == 0).all())
        target[3] = 60
        one = pa.linear_cross_entropy(x, w, target, b, reduction="none")
        assert (float(one[3]) == math.inf or float(one[3]) > 1e4) and torch.isfinite(one[4:]).all()
        b[:50] = -math.inf                             # a single word that can be, and only it
        b[60] = 0.0
        b[50:60] = b[61:] = -math.inf
        sure = pa.linear_cross_entropy(x, w, torch.full_like(target, 60), b, reduction="none")
        assert bool((sure == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("size", [(300, 64, 62), (300, 64, 200), (4100, 512, 8200)], ids=str)
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_infinite_logits(gpu, dtype, size, smoothing):
    """One at +infinity: NaN for every token, whichever word is wanted.  One at -infinity: an infinite loss for those that want it and, smoothed, for all."""
    x, w, b, target = make(*size, dtype, gpu, seed=4, left_out=0.1)
    target[:5] = torch.tensor([7, 8, 9, 7, -100], device=gpu)
    kept = target >= 0
    for value in (math.inf, -math.inf):
        b[7] = value
        loss = pa.linear_cross_entropy(x, w, target, b, label_smoothing=smoothing, reduction="none")
        want = torch.nn.functional.cross_entropy(x.float() @ w.float().t() + b.float(), target, label_smoothing=smoothing, reduction="none")
        assert torch.equal(torch.isnan(loss), torch.isnan(want)) and torch.equal(loss == math.inf, want == math.inf)
        assert bool((torch.isnan(loss) if value > 0 else loss == math.inf)[kept & ((target == 7) | (value > 0) | (smoothing > 0))].all())


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("V", [40, 140])
def test_words_that_are_all_but_certain(gpu, dtype, V):
    """Losses of 3e-10 (among 140 words 9e-9) to 1, and their gradients, to a share of themselves: 4 e + 32 u for the exponentials' arguments (logits of at most 40, so 64 u more), not to a share of the logits."""
    g = torch.Generator(device=gpu).manual_seed(1)
    M, D = 200, 32
    w = (torch.randn(V, D, generator=g, device=gpu) * 0.1).to(dtype)
    target = torch.randint(0, V, (M,), generator=g, device=gpu)
    x = torch.randn(M, D, generator=g, device=gpu)
    b = torch.zeros(V, device=gpu).to(dtype)
    x = (x + w.float()[target] * (torch.linspace(5, 30, M, device=gpu) / w.float()[target].square().sum(1))[:, None]).to(dtype)
    e = 2 * (4 * (D / 8 + 16) * U * float((x.float().abs() @ w.float().abs().t()).max()) + 128 * U)
    leaf = x.clone().requires_grad_()
    loss = pa.linear_cross_entropy(leaf, w, target, b, reduction="none")
    l = x.double() @ w.double().t()
    others = l.scatter(1, target[:, None], -math.inf).logsumexp(1) - l.gather(1, target[:, None])[:, 0]
    want = torch.log1p(torch.exp(others))
    assert float(want.min()) < (1e-9 if V == 40 else 1e-8) and bool(((loss.detach().double() - want).abs() <= e * want).all())
    dx, = torch.autograd.grad(loss, leaf, torch.ones(M, device=gpu))
    p = torch.softmax(l, 1).scatter(1, target[:, None], 0.0)
    P = p.scatter(1, target[:, None], -p.sum(1, keepdim=True))
    bar = (P.abs() @ w.double().abs()) * (e + 4 * torch.finfo(dtype).eps) + (2.0 ** -40 * V * float(w.abs().max()) + 2.0 ** -25 if dtype == F16 else 0.0)
    assert bool(((dx.double() - P @ w.double()).abs() <= bar).all())


def test_against_differences(gpu):
    """The gradient along random directions against differences of the loss in float64 of the same function, and the loss's own over steps that fp32 resolves (2^-24 of a loss of about 5 against a step's 0.01: 1e-4)."""
    x, w, b, target = make(60, 32, 50, F32, gpu, seed=2)
    for reduction in ("mean", "sum"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        grads = torch.autograd.grad(pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], label_smoothing=0.1, reduction=reduction), leaves)
        for i in range(3):
            way = [torch.zeros_like(t) for t in leaves]
            way[i] = torch.randn_like(way[i])
            t = 0.01

            def at(k):
                return float(pa.linear_cross_entropy(x + k * way[0], w + k * way[1], target, b + k * way[2], label_smoothing=0.1, reduction=reduction))
            slope = float((grads[i].double() * way[i].double()).sum())
            got = (8 * (at(t) - at(-t)) - (at(2 * t) - at(-2 * t))) / (12 * t)
            size = at(0)
            assert abs(got - slope) <= 2e-3 * abs(slope) + 4 * U * 18 * abs(size) / (12 * t) + 1e-4 * abs(size)


@pytest.mark.parametrize("V", [90, 20])
def test_layouts(gpu, V):
    """Batches of sequences, strided and unaligned tensors, an expanded gradient, parts that need no gradient."""
    x, w, b, target = make(240, 64, V, BF16, gpu, seed=6)
    want = [pa.linear_cross_entropy(x, w, target, b, reduction=r) for r in ("none", "mean", "sum")]
    wide = torch.zeros(4, 60, 130, dtype=BF16, device=gpu)
    wide[..., 1:65] = x.view(4, 60, 64)
    views = (wide[..., 1:65], w.t().contiguous().t(), target.view(4, 60), torch.cat((b[:1], b))[1:])
    assert not views[0].is_contiguous() and not views[1].is_contiguous() and views[3].data_ptr() % 16
    for r, q in zip(("none", "mean", "sum"), want):
        got = pa.linear_cross_entropy(views[0], views[1], views[2], views[3], reduction=r)
        assert torch.equal(got, q.view(got.shape))
    strided = torch.stack((target, target + 1), 1)[:, 0]
    assert torch.equal(pa.linear_cross_entropy(x, w, strided, b), want[1])
    grads = None
    for need in ((1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1)):
        leaves = [t.detach().clone().requires_grad_(bool(n)) for t, n in zip((views[0], views[1], views[3]), need)]
        leaves[0] = views[0].detach().requires_grad_(bool(need[0]))
        loss = pa.linear_cross_entropy(leaves[0], leaves[1], views[2], leaves[2], reduction="none")
        got = torch.autograd.grad(loss.sum(), [t for t in leaves if t.requires_grad])         # (the gradient of the sum: one number, expanded)
        grads = grads or got
        for g, q in zip(got, [q for q, n in zip(grads, need) if n]):
            assert torch.equal(g, q)
        leaves[0].requires_grad_(False)
    one = pa.linear_cross_entropy(x[3], w, target[3].clone(), b)                             # a single token without a batch
    assert one.dim() == 0 and torch.equal(one.view(1), pa.linear_cross_entropy(x[3:4], w, target[3:4].clone(), b).view(1))


def test_same_tensor_twice_and_shared_weights(gpu):
    """Features that are the words' own vectors (a tied embedding): both gradients go into one tensor."""
    g = torch.Generator(device=gpu).manual_seed(1)
    w = torch.randn(64, 32, generator=g, device=gpu).requires_grad_()
    t = torch.randint(0, 64, (64,), generator=g, device=gpu)
    got, = torch.autograd.grad(pa.linear_cross_entropy(w, w, t), w)
    a, b = w.detach().clone().requires_grad_(), w.detach().clone().requires_grad_()
    da, db = torch.autograd.grad(pa.linear_cross_entropy(a, b, t), (a, b))
    assert torch.equal(got, da + db)


def test_gradient_of_the_gradient_and_transforms(gpu):
    """These differentiate the torch expression."""
    x, w, b, target = make(20, 8, 10, F32, gpu, left_out=0.0)
    x.requires_grad_()
    loss = pa.linear_cross_entropy(x, w, target, b, label_smoothing=0.1)
    first, = torch.autograd.grad(loss, x, create_graph=True)
    second, = torch.autograd.grad(first.square().sum(), x)
    y = x.detach().requires_grad_()
    want = torch.nn.functional.cross_entropy(torch.nn.functional.linear(y, w, b), target, label_smoothing=0.1)
    wf, = torch.autograd.grad(want, y, create_graph=True)
    ws, = torch.autograd.grad(wf.square().sum(), y)
    assert (first - wf).abs().max() <= 1e-5 * wf.abs().max() and (second - ws).abs().max() <= 1e-4 * ws.abs().max()
    per = torch.func.vmap(lambda q, t: pa.linear_cross_entropy(q, w, t, b))(x.detach()[:, None], target[:, None])
    assert (per - pa.linear_cross_entropy(x.detach(), w, target, b, reduction="none")).abs().max() <= 1e-5
    with torch.autocast("cuda", dtype=BF16):
        again, = torch.autograd.grad(pa.linear_cross_entropy(x, w, target, b, label_smoothing=0.1), x)
        want, = torch.autograd.grad(torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w, b).float(), target, label_smoothing=0.1), x)
    assert torch.equal(again, want)


def test_saved_tensors_elsewhere(gpu):
    """Hooks that keep saved tensors on the CPU, and checkpoints, give the same gradients; a weight changed in place in between is noticed."""
    x, w, b, target = make(50, 32, 40, BF16, gpu)
    w.requires_grad_()
    want, = torch.autograd.grad(pa.linear_cross_entropy(x, w, target, b), w)
    with torch.autograd.graph.save_on_cpu():
        loss = pa.linear_cross_entropy(x, w, target, b)
    got, = torch.autograd.grad(loss, w)
    assert torch.equal(got, want)
    loss = torch.utils.checkpoint.checkpoint(lambda q: pa.linear_cross_entropy(x, q, target, b), w, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(loss, w)[0], want)
    loss = pa.linear_cross_entropy(x, w, target, b)
    with torch.no_grad():
        w.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(loss, w)


@pytest.mark.parametrize("size", [(300, 64, 500), (3000, 128, 20)], ids=str)
def test_graphs_and_streams(gpu, size):
    """A captured forward and backward replays on new inputs with other tokens left out; on another stream the bits are the same."""
    for dtype in (BF16, F32):
        cases = [make(*size, dtype, gpu, seed=s, left_out=q) for s, q in ((1, 0.5), (2, 0.0), (3, 0.9))]

        def go(x, w, b, target):
            leaves = [t.detach().requires_grad_() for t in (x, w, b)]
            loss = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2])
            return [loss.detach(), *torch.autograd.grad(loss, leaves)]
        want = [[t.clone() for t in go(*c)] for c in cases]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            there = go(*cases[0])
        torch.cuda.current_stream().wait_stream(stream)
        assert all(torch.equal(a, b) for a, b in zip(there, want[0]))
        held = [t.clone() for t in cases[0]]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go(*held)
        for _ in range(2):
            for c, q in zip(cases, want):
                for a, b in zip(held, c):
                    a.copy_(b)
                graph.replay()
                torch.cuda.synchronize()
                torch.randn(1000, device=gpu).sum()
                assert all(torch.equal(a, b) for a, b in zip(out, q))


def test_calls_at_once_on_two_streams(gpu):
    """Losses and gradients of different heads on two streams at once are those of each alone."""
    cases = [make(*size, dtype, gpu, seed=s) for s, (size, dtype) in enumerate([((2500, 256, 4100), BF16), ((3000, 128, 20), F32), ((900, 320, 9000), F32), ((2000, 64, 50), F16)])]

    def go(x, w, b, target):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        loss = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], label_smoothing=0.1)
        return [loss.detach(), *torch.autograd.grad(loss, leaves)]
    want = [go(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(3):
        for k, c in enumerate(cases):
            with torch.cuda.stream(streams[k % 2]):
                got.append((k, go(*c)))
    torch.cuda.synchronize()
    for k, g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want[k])), k


def test_nothing_beside_its_results_is_written(gpu):
    """Guarded gradients and workspaces of exactly the bytes asked for, through the C interface."""
    import ctypes
    from proteusai_amd import _lib
    lib = _lib.load()
    for dtype, code in ((BF16, 1), (F16, 2), (F32, 0)):
        for M, D, V in ((77, 40, 45), (100, 40, 20), (300, 64, 1003)):
            x, w, b, target = make(M, D, V, dtype, gpu, seed=M)
            a = _lib.CeArgs(x=x.data_ptr(), weight=w.data_ptr(), bias=b.data_ptr(), target=target.data_ptr(), ignore_index=-100, rows=M, d=D, vocab=V, dtype=code, reduction=1, label_smoothing=0.1)
            st = torch.cuda.current_stream().cuda_stream

            def guarded(n):
                t = torch.full((n + 512,), 0xA5, dtype=torch.uint8, device=gpu)
                return t, t[256:256 + n]
            parts = {}
            sizes = dict(loss=4, kept=lib.proteus_linear_ce_kept_bytes(ctypes.byref(a)), f=lib.proteus_linear_ce_fwd_bytes(ctypes.byref(a)), g=lib.proteus_linear_ce_bwd_bytes(ctypes.byref(a)),
                         dx=x.numel() * x.element_size(), dw=w.numel() * w.element_size(), db=V * b.element_size(), one=4)
            for k, n in sizes.items():
                parts[k] = guarded(n)
            p = {k: v[1].data_ptr() for k, v in parts.items()}
            parts["one"][1].view(F32).fill_(1.0)
            assert lib.proteus_linear_ce_fwd(ctypes.byref(a), p["loss"], p["kept"], sizes["kept"], p["f"], sizes["f"], st) == 0
            assert lib.proteus_linear_ce_bwd(ctypes.byref(a), p["one"], p["kept"], sizes["kept"], p["dx"], p["dw"], p["db"], p["g"], sizes["g"], st) == 0
            torch.cuda.synchronize()
            for k, (t, inner) in parts.items():
                assert bool((t[:256] == 0xA5).all()) and bool((t[256 + sizes[k]:] == 0xA5).all()), k
            leaves = [t.clone().requires_grad_() for t in (x, w, b)]
            loss = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], label_smoothing=0.1)
            for k, g in zip(("loss", "dx", "dw", "db"), (loss.detach(), *torch.autograd.grad(loss, leaves))):
                assert torch.equal(parts[k][1].view(g.dtype), g.reshape(-1)), k


def test_offsets_beyond_32_bits(gpu):
    """1.2 million tokens (gradients of their logits: 2.5e9 elements), and weights of 2.2e9 elements."""
    M, D, V = 1_200_000, 16, 2050
    x, w, b, target = make(M, D, V, BF16, gpu, seed=3)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    loss = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], reduction="none")
    d = torch.rand(M, device=gpu)
    grads = torch.autograd.grad(loss, leaves, d)
    pick = torch.cat((torch.arange(2000), torch.arange(1_048_000, 1_050_000), torch.arange(M - 2000, M))).to(gpu)
    wl, bar, wg, wb = exact(x[pick], w, b, target[pick], 0.0, "none", d[pick])
    off(loss.detach()[pick], wl, bar, "loss")
    off(grads[0][pick], wg[0], wb[0], "dx")
    _, _, wg, wb = exact(x, w, b, target, 0.0, "none", d)
    off(grads[1], wg[1], wb[1], "dw")
    off(grads[2], wg[2], wb[2], "db")
    del x, leaves, grads, loss, wg, wb
    M, D, V = 40, 4104, 540_000
    g = torch.Generator(device=gpu).manual_seed(1)
    w = torch.empty(V, D, dtype=BF16, device=gpu).normal_(0.0, 0.03, generator=g)
    x = torch.randn(M, D, generator=g, device=gpu).to(BF16)
    target = torch.randint(0, V, (M,), generator=g, device=gpu)
    target[:3] = torch.tensor([0, V - 1, 523_300], device=gpu)
    w.requires_grad_()
    loss = pa.linear_cross_entropy(x, w, target, reduction="none")
    l = torch.cat([x.double() @ c.double().t() for c in w.detach().split(60_000)], 1)
    e = 2 * (D / 8 + 16) * U * float(x.float().abs().sum(1).max()) * float(w.detach().abs().max())
    assert float((loss.detach() - (l.logsumexp(1) - l.gather(1, target[:, None])[:, 0])).abs().max()) <= e
    dw, = torch.autograd.grad(loss.sum(), w)
    p = torch.softmax(l, 1)
    p[torch.arange(M), target] -= 1.0
    for row in (0, 1, 523_299, 523_300, 523_301, V - 1, *target[3:6].tolist()):
        want = p[:, row] @ x.double()
        assert float((dw[row].double() - want).abs().max()) <= float((p[:, row].abs() @ x.double().abs()).max()) * (2.0 ** -7 + 4 * e)


@pytest.mark.parametrize("V", [30, 130])
def test_the_torch_expression_is_as_the_kernels_about_tokens(gpu, V):
    """Under autocast and in a backward that is recorded: targets that are no words, and features of tokens that are left out."""
    x, w, b, target = make(60, 32, V, F32, gpu, seed=3, left_out=0.0)
    target[5:20] = -100
    dirty = x.clone()
    dirty[5:20] = float("nan")

    def go(features, t, reduction="mean"):
        leaves = [q.detach().clone().requires_grad_() for q in (features, w, b)]
        loss = pa.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], label_smoothing=0.1, reduction=reduction)
        return [loss.detach(), *torch.autograd.grad(loss.sum(), leaves)]
    with torch.autocast("cuda", dtype=BF16):
        assert all(torch.equal(p, q) for p, q in zip(go(dirty, target), go(x, target)))
        for bad in (V, -1, 2 ** 40):
            t = target.clone()
            t[30] = bad
            loss, dx, *_ = go(dirty, t, "none")
            rest = torch.arange(60, device=gpu) != 30
            assert loss[30].isnan() and torch.isfinite(loss[rest]).all() and dx[30].isnan().all() and torch.isfinite(dx[rest]).all() and bool((dx[5:20] == 0).all())
            assert go(dirty, t)[0].isnan()
    firsts = []
    for features in (x, dirty):
        leaf = features.clone().requires_grad_()
        first, = torch.autograd.grad(pa.linear_cross_entropy(leaf, w, target, b), leaf, create_graph=True)
        firsts.append([first.detach(), *torch.autograd.grad(first.square().sum(), leaf)])
    assert all(torch.equal(p, q) and bool(torch.isfinite(p).all()) for p, q in zip(*firsts))
    with pytest.raises(ValueError, match="no words"):
        pa.linear_cross_entropy(x, w[:0], target)


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("size", [(70, 64, 1), (300, 64, 62), (300, 64, 200), (40, 64, 200), (4100, 512, 8200)], ids=str)
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_tokens_whose_words_are_all_shut_out(gpu, dtype, size, smoothing):
    """Nothing to be a share of: NaN as torch's expression gives it, for the loss and the gradients, and not a loss of 0."""
    x, w, b, target = make(*size, dtype, gpu, seed=4, left_out=0.1)
    target[:3] = torch.tensor([0, size[2] - 1, -100], device=gpu)
    leaves = [t.clone().requires_grad_() for t in (x, w, torch.full_like(b, -math.inf))]
    loss = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], label_smoothing=smoothing, reduction="none")
    want = torch.nn.functional.cross_entropy(torch.nn.functional.linear(*leaves).detach().float(), target, label_smoothing=smoothing, reduction="none")
    assert torch.equal(torch.isnan(loss), target >= 0) and torch.equal(torch.isnan(want), target >= 0) and bool((loss[target < 0] == 0).all())
    dx, dw, db = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
    assert bool(dx[target >= 0].isnan().all()) and bool((dx[target < 0] == 0).all()) and bool(dw.isnan().all()) and bool(db.isnan().all())
    if dtype == F16:                                    # (whose products stay below fp32's infinity)
        return
    clean = x.clone()                                   # one token alone, by its features; powers of two are exact in every type
    clean[:, 0] = 0.0
    w[:, 0] = -2.0 ** 100
    one = clean.clone()
    one[1, 0] = 2.0 ** 100
    got = [pa.linear_cross_entropy(t, w, target, b, label_smoothing=smoothing, reduction="none") for t in (clean, one)]
    rest = torch.arange(size[0], device=gpu) != 1
    assert got[1][1].isnan() and torch.equal(got[0][rest], got[1][rest]) and bool(torch.isfinite(got[0]).all())


def test_more_tiles_than_a_grid_may_have(gpu):
    """2^20 tokens of 16 features and 2^17 words: 2^37 logits.  The words are 64 different ones over and over, so that a token's loss is log(2^11) more than it is among those; the sum over 1024 groups of 128
    words rounds once for each."""
    M, D, V, R = 1 << 20, 16, 64, 1 << 11
    x, w, _, target = make(M, D, V, BF16, gpu, seed=1, bias=False)
    kept = target >= 0
    words = w.repeat(R, 1)
    loss = pa.linear_cross_entropy(x, words, torch.where(kept, target + V * (torch.arange(M, device=gpu) % R), target), reduction="none")
    want, bar, _, _ = exact(x, w, None, target, 0.0, "none", torch.ones(M, device=gpu))
    want, bar = torch.where(kept, want + math.log(R), want), bar + (16 * math.log(R) + 1024) * U
    off(loss, want, bar, "loss")
    mean = pa.linear_cross_entropy(x, words, target)
    assert abs(float(mean) - float(want[kept].mean())) <= float(bar[kept].mean()) + U * float(mean)


@pytest.mark.parametrize("dtype", [BF16, F16], ids=lambda t: str(t).split(".")[-1])
@pytest.mark.parametrize("size,left", [((65, 136, 3001), 1), ((4096, 136, 3001), 10), ((64, 136, 3001), 1)], ids=str)
def test_few_tokens_that_count_among_many(gpu, dtype, size, left):
    """The gradients' bars are those of all tokens' number: up to 64, left out or not, the logits' gradient is two numbers of its type, beyond that one."""
    x, w, b, target = make(*size, dtype, gpu, seed=left, left_out=0.0)
    target[torch.randperm(size[0], generator=torch.Generator().manual_seed(1))[left:].to(gpu)] = -100
    loss, bar, grads, bars = exact(x, w, b, target, 0.1, fine=size[0] <= 64)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    got = pa.linear_cross_entropy(leaves[0], leaves[1], target, leaves[2], label_smoothing=0.1)
    off(got.detach(), loss, bar, "loss")
    for name, g, want, q in zip(("dx", "dw", "db"), torch.autograd.grad(got, leaves), grads, bars):
        off(g, want, q, name)


def test_the_torch_expression_in_a_captured_graph(gpu):
    """Under autocast: replays on other tokens, some left out and one of them no word, are the eager call's."""
    x, w, b, target = make(200, 32, 60, F32, gpu, seed=3)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    held = target.clone()

    def go():
        with torch.autocast("cuda", dtype=BF16):
            loss = pa.linear_cross_entropy(leaves[0], leaves[1], held, leaves[2], reduction="none")
        return [loss.detach(), *torch.autograd.grad(loss, leaves, torch.ones_like(loss))]
    targets = [target, target.roll(7), torch.where(torch.arange(200, device=gpu) == 90, 60, target)]
    want = []
    for t in targets:
        held.copy_(t)
        want.append([q.clone() for q in go()])
    assert int(want[2][0].isnan().sum()) == 1
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        go()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = go()
    for _ in range(2):
        for t, q in zip(targets, want):
            held.copy_(t)
            graph.replay()
            torch.cuda.synchronize()
            torch.randn(1000, device=gpu).sum()
            for a, c in zip(out, q):
                assert torch.equal(a.isnan(), c.isnan()) and bool(((a - c).abs().nan_to_num(0.0) <= 1e-5 * (1 + c.abs().nan_to_num(0.0).max())).all())
