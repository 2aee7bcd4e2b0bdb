"""GPU tests of the norm over gradients and their clipping against float64 on the CPU.

Bars: the norm is an fp64 sum rounded to fp32 once (half a step, 2^-24; the sum's own error over 10^8 terms is below 2^-26).  The factor takes four more roundings
to fp32, a scaled element one of its own type."""
import math

import pytest
import torch

import proteusai_amd as pa

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.bfloat16, torch.float16)


def make(sizes, dtypes, gpu, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * math.exp(float(torch.randn((), generator=g)))).to(dtypes[i % len(dtypes)]).to(gpu) for i, n in enumerate(sizes)]


def exact_norm(grads, p):
    flat = torch.cat([t.detach().double().cpu().reshape(-1) for t in grads])
    return float(torch.linalg.vector_norm(flat, p)) if flat.numel() else 0.0


def check(got, grads, norm, max_norm):
    factor = min(1.0, max_norm / (norm + 1e-6))
    for o, g in zip(got, grads):
        want = g.double().cpu() * factor
        bar = want.abs() * (5 * 2.0 ** -24 + (0 if factor == 1.0 and o.dtype == g.dtype else torch.finfo(o.dtype).eps / 2)) + torch.finfo(o.dtype).smallest_normal * torch.finfo(o.dtype).eps
        assert ((o.double().cpu() - want).abs() <= bar).all()


SIZES = [
    [1], [1, 2, 3], [5, 0, 7], [4096, 4097, 4095, 8191], [100_003, 1, 17, 2_000_001], list(range(1, 330)), [37] * 700, [3_000_000, 5, 64],
]


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_norm_and_clipping(gpu, sizes, p):
    for dtypes in (TYPES[:1], TYPES[1:2], TYPES):
        grads = make(sizes, dtypes, gpu, seed=len(sizes))
        norm = exact_norm(grads, p)
        got = float(pa.grad_norm(grads, p))
        assert abs(got - norm) <= 2.0 ** -23 * norm
        for ratio in (0.3, 3.0):
            for out_dtype in (None, torch.float32, torch.bfloat16):
                out = None if out_dtype is None else [torch.full_like(t, float("nan"), dtype=out_dtype) for t in grads]
                n, out = pa.clip_grad_norm(grads, ratio * norm, p, out=out)
                assert float(n) == got and n.dtype == torch.float32 and n.dim() == 0
                check(out, grads, norm, ratio * norm)
            params = [torch.nn.Parameter(torch.empty_like(t)) for t in grads] + [torch.nn.Parameter(torch.zeros(3, device=gpu))]     # (the last without a gradient)
            for q, t in zip(params, grads):
                q.grad = t.clone()
            versions = [q.grad._version for q in params[:-1]]
            n = pa.clip_grad_norm_(params, ratio * norm, p)
            assert float(n) == got and params[-1].grad is None
            check([q.grad for q in params[:-1]], grads, norm, ratio * norm)
            assert all(q.grad._version > v for q, v in zip(params, versions))
            if ratio > 1:
                assert all(torch.equal(q.grad, t) for q, t in zip(params, grads))


def test_bucket_of_odd_sizes(gpu):
    """Tensors one behind the other at every alignment: nothing beside them is written."""
    sizes = [1, 3, 8, 17, 4099, 2, 5, 40_001, 64]
    for dtype in TYPES:
        g = torch.Generator().manual_seed(1)
        flat = torch.randn(sum(sizes) + 2 * len(sizes), generator=g).to(dtype).to(gpu)
        parts, at, gaps = [], 0, torch.ones(flat.numel(), dtype=torch.bool)
        for n in sizes:
            parts.append(flat[at + 1:at + 1 + n])
            gaps[at + 1:at + 1 + n] = False
            at += n + 2
        before = flat.clone()
        norm = exact_norm(parts, 2.0)
        grads = [t.clone() for t in parts]
        n, out = pa.clip_grad_norm(parts, 0.25 * norm, out=parts)
        check(parts, grads, norm, 0.25 * norm)
        assert torch.equal(flat.cpu()[gaps], before.cpu()[gaps])
        apart = torch.full_like(flat, 7.0)
        views, at = [], 0
        for k in sizes:
            views.append(apart[at:at + k])
            at += k
        pa.clip_grad_norm(grads, 0.25 * norm, out=views)
        assert all(torch.equal(a, b) for a, b in zip(views, parts)) and (apart[at:] == 7.0).all()


def test_extremes(gpu):
    big, small = torch.full((1000,), 3e38, device=gpu), torch.full((999,), 1e-42, device=gpu)
    assert float(pa.grad_norm([big])) == math.inf                                # beyond fp32 as a number, not as a sum
    big = torch.full((1000,), 1e30, device=gpu)
    n, out = pa.clip_grad_norm([big], 1.0)
    assert abs(float(n) - 1e30 * 1000 ** 0.5) <= 2.0 ** -22 * float(n) and abs(float(out[0].double().norm()) - 1.0) <= 1e-5
    assert abs(float(pa.grad_norm([small])) - float(small.double().norm())) <= 2.0 ** -149
    for bad, p in ((math.nan, 2.0), (math.nan, 1.0), (math.nan, math.inf)):
        g = [torch.ones(5000, device=gpu), torch.ones(3, device=gpu)]
        g[1][2] = bad
        n, out = pa.clip_grad_norm(g, 1.0, p)
        assert math.isnan(float(n)) and all(o.isnan().all() for o in out)
    g = [torch.ones(5000, device=gpu), torch.ones(3, device=gpu)]
    g[1][2] = math.inf
    want = [t.clone() for t in g]
    params = [torch.nn.Parameter(t.clone()) for t in g]
    for q, t in zip(params, want):
        q.grad = t
    torch.nn.utils.clip_grad_norm_(params, 1.0)
    n, out = pa.clip_grad_norm(g, 1.0)
    assert float(n) == math.inf and all(torch.equal(a, b) or (a.isnan() == b.isnan()).all() for a, b in zip(out, want))
    with pytest.raises(RuntimeError, match="cannot be clipped"):
        pa.clip_grad_norm(g, 1.0, out=g, error_if_nonfinite=True)
    assert (g[0] == 1).all()                                                     # not touched
    n, out = pa.clip_grad_norm([torch.ones(4, device=gpu)], 0.0)
    assert float(n) == 2.0 and not out[0].any()
    n, out = pa.clip_grad_norm([torch.zeros(4, device=gpu)], 1.0)
    assert float(n) == 0.0 and not out[0].any()
    assert float(pa.grad_norm([torch.ones(16, device=gpu)], error_if_nonfinite=True)) == 4.0
    assert float(pa.clip_grad_norm_([], 1.0)) == 0.0 and float(pa.clip_grad_norm_([torch.nn.Parameter(torch.ones(2))], 1.0)) == 0.0
    n, out = pa.clip_grad_norm([torch.empty(0, device=gpu)], 1.0)
    assert float(n) == 0.0


def test_matches_torch(gpu):
    model = torch.nn.Sequential(torch.nn.Linear(100, 333), torch.nn.Linear(333, 7)).to(gpu)
    model(torch.randn(50, 100, device=gpu)).square().sum().backward()
    grads = [q.grad.clone() for q in model.parameters()]
    for p in (1.0, 2.0, math.inf):
        for q, t in zip(model.parameters(), grads):
            q.grad.copy_(t)
        want = torch.nn.utils.clip_grad_norm_(model.parameters(), 0.1, p)
        expected = [q.grad.clone() for q in model.parameters()]
        for q, t in zip(model.parameters(), grads):
            q.grad.copy_(t)
        got = pa.clip_grad_norm_(model.parameters(), 0.1, p)
        assert abs(float(got) - float(want)) <= 1e-5 * float(want)
        for q, t in zip(model.parameters(), expected):
            assert (q.grad - t).abs().max() <= 1e-5 * t.abs().max()
    one = torch.nn.Parameter(torch.zeros(3, device=gpu))
    one.grad = torch.tensor([3.0, 0.0, 4.0], device=gpu)
    assert float(pa.clip_grad_norm_(one, 1.0)) == 5.0


def test_layouts(gpu):
    g = torch.Generator().manual_seed(2)
    base = torch.randn(40, 60, generator=g).to(gpu)
    norm = float(base.double().norm())
    n, out = pa.clip_grad_norm([base.t()], 0.5 * norm)                           # dense in another order
    assert torch.equal(out[0], pa.clip_grad_norm([base], 0.5 * norm)[1][0].t())
    apart = torch.empty(60, 40, device=gpu)                                      # ... into this one
    pa.clip_grad_norm([base.t()], 0.5 * norm, out=[apart])
    assert torch.equal(apart, out[0])
    part = base[:, ::3]                                                          # not dense
    want = part.double().cpu() * (1.0 / (float(part.double().norm()) + 1e-6))
    rest = base.clone()
    q = torch.nn.Parameter(torch.empty_like(part))
    q.grad = rest[:, ::3]
    pa.clip_grad_norm_([q], 1.0)
    assert (rest[:, ::3].double().cpu() - want).abs().max() <= 1e-6 and torch.equal(rest[:, 1::3], base[:, 1::3])
    assert abs(float(pa.grad_norm([base[:1].expand(40, 60)])) - float(base[:1].expand(40, 60).double().norm())) <= 1e-4


def test_shared_memory_is_refused(gpu):
    flat = torch.randn(1000, device=gpu)
    keep = flat.clone()
    q = torch.nn.Parameter(torch.zeros(500, device=gpu))
    q.grad = flat[:500]
    with pytest.raises(ValueError, match="share memory"):
        pa.clip_grad_norm_([q, q], 1e-3)
    with pytest.raises(ValueError, match="share memory"):
        pa.clip_grad_norm([flat[:500], flat[400:900]], 1e-3, out=[flat[:500], flat[400:900]])
    with pytest.raises(ValueError, match="share memory"):
        pa.clip_grad_norm([flat[:500]], 1e-3, out=[flat[1:501]])
    with pytest.raises(ValueError, match="share memory"):
        pa.clip_grad_norm([flat[:500], flat[500:]], 1e-3, out=[flat[500:], flat[:500]])
    assert torch.equal(flat, keep)
    assert abs(float(pa.grad_norm([flat, flat])) - 2 ** 0.5 * float(flat.double().norm())) <= 1e-4      # the norm alone may count one twice


def test_same_bits_other_streams_and_replays(gpu):
    grads = make([70_001, 5, 300_000, 1 << 20] + [33] * 400, TYPES, gpu, seed=3)
    max_norm = 0.1 * exact_norm(grads, 2.0)
    n0, first = pa.clip_grad_norm(grads, max_norm)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        n1, second = pa.clip_grad_norm(grads, max_norm)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(n0, n1) and all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n2, out = pa.clip_grad_norm(grads, max_norm)
    for i in range(3):
        for t in grads:
            t.mul_(-0.5)
        graph.replay()
        torch.cuda.synchronize()
        n3, want = pa.clip_grad_norm(grads, max_norm)
        assert torch.equal(n2, n3) and all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_large(gpu):
    g = torch.Generator(device=gpu).manual_seed(4)
    big = torch.randn(300_000_007, generator=g, device=gpu).bfloat16()           # 16-bit elements beyond 2^28, an odd number of them
    norm = float(torch.stack([c.double().square().sum() for c in big.split(1 << 26)]).sum().sqrt())
    n, out = pa.clip_grad_norm([big], 0.5 * norm, out=[torch.empty_like(big, dtype=torch.float32)])
    assert abs(float(n) - norm) <= 2.0 ** -23 * norm
    factor = 0.5 * norm / (norm + 1e-6)
    for a, b in zip(out[0].split(1 << 26), big.split(1 << 26)):
        assert float((a.double() - b.double() * factor).abs().max()) <= 6 * 2.0 ** -24 * float(b.double().abs().max())


def test_a_gradient_scaled_in_place_and_read_for_another_is_refused(gpu):
    a, b = torch.randn(100_000, device=gpu), torch.randn(100_000, device=gpu)
    before = a.clone(), b.clone()
    for grads, out in (([a, a], [a, b]), ([a, a], [b, a]), ([a[:60_000], a[50_000:]], [a[:60_000], b[50_000:]])):
        with pytest.raises(ValueError, match="share memory"):
            pa.clip_grad_norm(grads, 1e-3, out=out)
    assert torch.equal(a, before[0]) and torch.equal(b, before[1])
    norm, (c, d) = pa.clip_grad_norm([a, a], 1.0)                                # (read twice and written nowhere: two results)
    assert torch.equal(c, d) and torch.equal(a, before[0])


def test_tensors_made_in_inference_mode(gpu):
    """Outside of it they can be read and not written, as with torch's own operators; inside everything goes."""
    with torch.inference_mode():
        made = torch.full((100,), 3.0, device=gpu)
    apart = torch.zeros(100, device=gpu)
    n, out = pa.clip_grad_norm([made], 3.0, out=[apart])
    assert abs(float(n) - 30.0) <= 1e-5 and float(pa.grad_norm([made])) == float(n)
    p = torch.nn.Parameter(torch.zeros(100, device=gpu))
    p.grad = made
    for call in (lambda: pa.clip_grad_norm([made], 3.0, out=[made]), lambda: pa.clip_grad_norm([apart], 3.0, out=[made]), lambda: pa.clip_grad_norm_([p], 3.0),
                 lambda: pa.clip_grad_norm([made], 3.0, out=[made], error_if_nonfinite=True), lambda: pa.clip_grad_norm([apart.view(10, 10).t()], 3.0, out=[made.view(10, 10)])):
        with pytest.raises(RuntimeError, match="inference"):
            call()
    assert (made == 3.0).all()
    with torch.inference_mode():
        pa.clip_grad_norm([made], 3.0, out=[made])
    assert abs(float(made.double().norm()) - 3.0) <= 1e-5
