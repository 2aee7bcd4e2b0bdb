"""GPU tests of AdamW's step against the formula in float64 on the CPU, with moments in 32 and in 8 bits, and of the optimizer around it.

Bars, in units of u = 2^-24 (half a step of fp32, relative).  m: b1, 1 - b1, the two products and their sum round once each, the gradient's factor and its product 5 times more: 9 u of |b1 m| + |(1 - b1) g|.
v: as m, the gradient's error twice: 15 u of itself.  The update: m's 9 u of its terms, and of itself half of v's, root, two coefficients, products, sum and division: 16 u.  The parameter: its own
product and sum 3 u, and half a step of its type."""
import copy
import math

import pytest
import torch

import proteusai_amd as pa

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24
HOW = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [[1], [1, 2, 3, 511, 512, 513], [5, 0, 7], [2047, 2048, 2049, 8191], [100_003, 1, 17, 2_000_001], list(range(1, 330)), [37] * 500]


def make(sizes, ptype, gtype, gpu, seed=0, master=False):
    g = torch.Generator().manual_seed(seed)
    p = [torch.randn(n, generator=g) for n in sizes]
    s = dict(params=[x.to(ptype).to(gpu) for x in p], masters=[x.to(gpu) for x in p] if master else None,
             grads=[(torch.randn(n, generator=g) * 10.0 ** float(torch.randint(-3, 2, (1,), generator=g))).to(gtype).to(gpu) for n in sizes])
    s["m"] = [0.3 * x.float() * torch.randn(x.shape, generator=g).to(gpu) for x in s["grads"]]
    s["v"] = [(x.float() * (0.5 + torch.rand(x.shape, generator=g).to(gpu))).square() for x in s["grads"]]
    return s


def formula(p, g, m, v, t, factor=1.0, lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1):
    """(p, m, v, the bars of each without the parameter's own rounding), in float64."""
    p, g, m, v = (x.double().cpu() for x in (p, g, m, v))
    g = g * factor
    b1, b2 = betas
    terms = (b1 * m).abs() + ((1 - b1) * g).abs()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    scale = lr / (1 - b1 ** t) / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    kept = p * (1 - lr * weight_decay)
    return kept - scale * m, m, v, 3 * U * (kept.abs() + (scale * m).abs()) + scale * 9 * U * terms + 16 * U * (scale * m).abs(), 9 * U * terms + 2.0 ** -149, 15 * U * v + 2.0 ** -148


def off(got, want, bar):
    d = (got.double().cpu() - want).abs()
    assert (d <= bar).all(), f"{(d / bar.clamp_min(1e-300)).max():.3g} of the bar"


def half_step(x, dtype):
    return x.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


KINDS = [(F32, F32, False), (F32, BF16, False), (F32, F16, False), (BF16, BF16, False), (BF16, BF16, True), (BF16, F32, True), (BF16, F32, False), (F16, F16, True), (F16, F32, False)]


def check32(s, before, t, factor=1.0, how=HOW):
    for i in range(len(s["params"])):
        start = before["masters"][i] if s["masters"] else before["params"][i]
        p, m, v, bp, bm, bv = formula(start, before["grads"][i], before["m"][i], before["v"][i], t, factor, **how)
        off(s["m"][i], m, bm)
        off(s["v"][i], v, bv)
        if s["masters"]:
            off(s["masters"][i], p, bp)
            assert torch.equal(s["params"][i], s["masters"][i].to(s["params"][i].dtype))
        else:
            off(s["params"][i], p, bp + (half_step(p.abs() + bp, s["params"][i].dtype) if s["params"][i].dtype != F32 else 0))
        assert torch.equal(s["grads"][i], before["grads"][i])


@pytest.mark.parametrize("ptype,gtype,master", KINDS, ids=lambda x: str(x).split(".")[-1])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_step(gpu, sizes, ptype, gtype, master):
    s = make(sizes, ptype, gtype, gpu, len(sizes), master)
    before = copy.deepcopy(s)
    versions = [x._version for x in s["params"]]
    assert pa.adamw_(s["params"], s["grads"], s["m"], s["v"], 3, masters=s["masters"], **HOW) is None
    check32(s, before, 3)
    assert all(x._version > v for x, v in zip(s["params"], versions))


@pytest.mark.parametrize("how", [dict(lr=0.0), dict(weight_decay=0.0), dict(betas=(0.0, 0.0)), dict(eps=1e-3), dict(lr=0.5, betas=(0.5, 0.999))], ids=str)
@pytest.mark.parametrize("t", [1, 2, 1000, 10 ** 9])
def test_hyperparameters(gpu, how, t):
    how = {**HOW, **how}
    for on_gpu in (False, True):
        s = make([700, 5], F32, F32, gpu, 4)
        before = copy.deepcopy(s)
        step = torch.full((), t - 1, dtype=torch.int64, device=gpu) if on_gpu else t
        lr = torch.full((1,), how["lr"], device=gpu) if on_gpu else how["lr"]
        pa.adamw_(s["params"], s["grads"], s["m"], s["v"], step, **{**how, "lr": lr})
        check32(s, before, t, how={**how, "lr": float(lr)})
        assert not on_gpu or int(step) == t


@pytest.mark.parametrize("ratio", [0.1, 5.0])
def test_norm(gpu, ratio):
    for eight in (False, True):
        s = make([3000, 17, 70_001], F32, BF16, gpu, 5)
        before = copy.deepcopy(s)
        norm = pa.grad_norm(s["grads"])
        max_norm = ratio * float(norm)
        if eight:
            states = [pa.adamw8_state(p) for p in s["params"]]
            other = [x.clone() for x in states], [x.clone() for x in s["params"]]
            _, clipped = pa.clip_grad_norm(s["grads"], max_norm, out=[torch.empty_like(x, dtype=F32) for x in s["grads"]])
            pa.adamw8_(s["params"], s["grads"], states, 1, norm=norm, max_norm=max_norm, **HOW)
            pa.adamw8_(other[1], clipped, other[0], 1, **HOW)
            assert all(torch.equal(a, b) for a, b in zip(states + s["params"], other[0] + other[1]))
        else:
            pa.adamw_(s["params"], s["grads"], s["m"], s["v"], 7, norm=norm, max_norm=max_norm, **HOW)
            check32(s, before, 7, min(1.0, max_norm / (float(norm) + 1e-6)))


def test_no_element_beside_them(gpu):
    """Tensors one behind the other at every alignment: nothing between them is written."""
    sizes = [1, 3, 8, 17, 4099, 2, 5, 40_001, 64]
    for ptype, gtype in ((F32, F32), (F32, BF16), (BF16, BF16)):
        for eight in (False, True):
            s = make(sizes, ptype, gtype, gpu, 6)

            def bucket(tensors):
                flat = torch.full((sum(x.numel() + 3 for x in tensors),), 7.0, dtype=tensors[0].dtype, device=gpu)
                inside, parts, at = torch.zeros(flat.numel(), dtype=torch.bool, device=gpu), [], 1
                for x in tensors:
                    parts.append(flat[at:at + x.numel()].copy_(x))
                    inside[at:at + x.numel()] = True
                    at += x.numel() + 3
                return flat, inside, parts
            packed = {k: bucket(s[k]) for k in ("params", "grads", "m", "v")}
            before = copy.deepcopy({k: s[k] for k in s})
            if eight:
                states = torch.full((sum(-(-n // 512) + 1 for n in sizes), 1056), 0, dtype=torch.uint8, device=gpu)
                parts, at = [], 0
                guard = torch.ones(len(states), dtype=torch.bool, device=gpu)
                for n in sizes:
                    rows = -(-n // 512)
                    parts.append(states[at:at + rows])
                    guard[at:at + rows] = False
                    at += rows + 1
                states[guard] = 99
                plain = [pa.adamw8_state(x) for x in s["params"]]
                pa.adamw8_(packed["params"][2], packed["grads"][2], parts, 2, seed=3, **HOW)
                pa.adamw8_(s["params"], s["grads"], plain, 2, seed=3, **HOW)
                assert (states[guard] == 99).all() and all(torch.equal(a, b) for a, b in zip(parts, plain))
                assert all(torch.equal(a, b) for a, b in zip(packed["params"][2], s["params"]))
            else:
                pa.adamw_(packed["params"][2], packed["grads"][2], packed["m"][2], packed["v"][2], 2, **HOW)
                check32(dict(params=packed["params"][2], grads=packed["grads"][2], m=packed["m"][2], v=packed["v"][2], masters=None), before, 2)
            for k in ("params", "grads", "m", "v"):
                flat, inside, _ = packed[k]
                assert (flat[~inside] == 7.0).all()


def test_layouts(gpu):
    """Parameters in other orders of memory, gradients in another order than theirs."""
    g = torch.Generator().manual_seed(8)
    p = torch.randn(33, 70, generator=g).to(gpu).t()
    conv = torch.randn(4, 6, 5, 3, generator=g).to(gpu).to(memory_format=torch.channels_last)
    for x in (p, conv):
        grad = torch.randn(x.shape, generator=g).to(gpu)
        assert grad.stride() != x.stride()
        m, v = torch.zeros_like(x), torch.zeros_like(x)
        assert m.stride() == x.stride()
        before = [t.clone().contiguous() for t in (x, m, v)]
        wanted = formula(before[0], grad, before[1], before[2], 1, **HOW)
        mine = x.clone(memory_format=torch.preserve_format)
        pa.adamw_([mine], [grad], [m], [v], 1, **HOW)
        off(mine, wanted[0], wanted[3])
        off(m, wanted[1], wanted[4])
        state, dense = pa.adamw8_state(x), pa.adamw8_state(x)
        mine = x.clone(memory_format=torch.preserve_format)
        pa.adamw8_([mine], [grad], [state], 1, **HOW)
        off(mine, wanted[0], wanted[3])
        m8, v8 = pa.adamw8_moments(x, state)
        assert m8.stride() == x.stride() and ((m8 - m).abs() <= 2.0 ** -3 * m.abs() + 1e-9).all()
        order = x.permute(*sorted(range(x.dim()), key=lambda i: -x.stride(i)))
        flat = order.clone().contiguous().view(-1)
        pa.adamw8_([flat], [grad.permute(*sorted(range(x.dim()), key=lambda i: -x.stride(i))).contiguous().view(-1)], [dense], 1, **HOW)
        assert torch.equal(state, dense)


def test_memory_that_is_shared_is_refused(gpu):
    """Whatever the order of the lists: views of one another, interleaved buffers, a gradient, a rate or a norm inside of what is written."""
    flat = torch.zeros(4000, device=gpu)
    half = torch.randn(100, device=gpu)

    def lists(p=None, g=None, m=None, v=None, **kw):
        z = lambda: torch.zeros(100, device=gpu)  # noqa: E731
        return [p or [z(), z()], g or [half, half], m or [z(), z()], v or [z(), z()], 1], kw
    fine = [flat[i * 200:i * 200 + 100] for i in range(16)]
    for args, kw in (lists(p=fine[0:2], m=fine[2:4], v=fine[4:6], g=fine[6:8]), lists(p=fine[0:4:2], m=fine[1:5:2], v=fine[5:9:2], g=[fine[9], fine[9]]), lists(p=fine[8:6:-1], m=fine[0:2], v=fine[15:13:-1])):
        pa.adamw_(*args, **kw)
    a, b = torch.zeros(100, device=gpu), torch.zeros(100, device=gpu)
    for args, kw in (lists(p=[a, a]), lists(p=[a, b], m=[b, torch.zeros(100, device=gpu)]), lists(p=[a, b], g=[half, a]), lists(p=[flat[:100], flat[99:199]]), lists(p=[flat[300:400], flat[0:100]], v=[flat[500:600], flat[50:150]]),
                     lists(m=[a, b], v=[b, a]), lists(p=[a, b], norm=a[5], max_norm=1.0), lists(p=[a, b], lr=b[7:8])):
        before = [x.clone() for x in (a, b, flat)]
        with pytest.raises(ValueError, match="share memory"):
            pa.adamw_(*args, **kw)
        assert all(torch.equal(x, y) for x, y in zip((a, b, flat), before))


# ---------------------------------------------------------------------------------------------------- moments in 8 bits

def mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def random_bits(n, tensor, step, seed):
    key = mix(torch.tensor((seed + step * 0x9e3779b1) & 0xffffffff))
    i = torch.arange(n)
    key = mix((key + tensor * 0x85ebca6b + (i >> 32) * 0xc2b2ae35) & 0xffffffff)
    return mix(key ^ (i & 0xffffffff))


def grid(x, random, least):
    """(values, the distance of two codes there) of x in float64, rounded by 16 random bits; a scale for every 32."""
    n = len(x)
    x = torch.nn.functional.pad(x, (0, -n % 32)).view(-1, 32)
    random = torch.nn.functional.pad(random, (0, -n % 32)).view(-1, 32).double() / 65536
    most = x.abs().amax(1)
    e = torch.where(most > 0, torch.ceil(torch.log2(most.clamp_min(1e-300) / 448)), -127.0).clamp_min(-127.0)
    y = x.abs() * torch.exp2(-e)[:, None]
    step = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
    q = torch.floor(y / step + random) * step
    if least:
        q = torch.where((x > 0) & (q == 0), 2.0 ** -9, q)
    scale = torch.exp2(e)[:, None]
    return (torch.sign(x) * q * scale).view(-1)[:n], (step * scale).view(-1)[:n]


@pytest.mark.parametrize("ptype,gtype,master", KINDS, ids=lambda x: str(x).split(".")[-1])
@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{max(s)}")
def test_step_of_8_bits(gpu, sizes, ptype, gtype, master):
    """Two steps.  A code is the oracle's but where the fp32 moment (16 u off at most) lies on the other side of the border drawn for it, one in 2^16 of the distance of two codes apart from the next: in
    2^23 u / 8 of that distance (the least for its size) the chance of that is 2^-15 an element; then it is the neighbour."""
    s = make(sizes, ptype, gtype, gpu, 20 + len(sizes), master)
    states = [pa.adamw8_state(p) for p in s["params"]]
    differ = total = 0
    for t in (1, 2):
        before, moments = copy.deepcopy(s), [pa.adamw8_moments(p, st) for p, st in zip(s["params"], states)]
        pa.adamw8_(s["params"], s["grads"], states, t, masters=s["masters"], seed=77, **HOW)
        for i, p in enumerate(s["params"]):
            n = p.numel()
            start = before["masters"][i] if master else before["params"][i]
            wp, wm, wv, bp, _, _ = formula(start, before["grads"][i], *moments[i], t, **HOW)
            if master:
                off(s["masters"][i], wp, bp)
                assert torch.equal(p, s["masters"][i].to(ptype))
            else:
                off(p, wp, bp + (half_step(wp.abs() + bp, ptype) if ptype != F32 else 0))
            r = random_bits(n, i, t, 77)
            m, v = pa.adamw8_moments(p, states[i])
            for got, want, bits, least in ((m, wm, r & 0xffff, False), (v.sqrt(), wv.sqrt(), r >> 16, True)):
                q, step = grid(want, bits, least)
                d = (got.double().cpu() - q).abs()
                assert (d <= step * 1.0001).all()
                differ += int((d > step * 0.01).sum())
                total += n
            rest = states[i].view(-1, 1056)[-1:]
            if n % 512:
                assert (rest[0, n % 512:512] == 0).all() and (rest[0, 512 + n % 512:1024] == 0).all()
    assert differ <= 4 + total * 2.0 ** -15


def test_rounding_is_unbiased(gpu):
    """The mean of 4096 roundings of a moment is within 5 of its deviations (at most half a distance of two codes over 64) of it."""
    n = 320
    g = torch.Generator().manual_seed(1)
    grad = (torch.randn(n, generator=g) * torch.exp(2 * torch.randn(n, generator=g))).to(gpu)
    sums = torch.zeros(2, n, dtype=torch.float64, device=gpu)
    p = torch.zeros(n, device=gpu)
    for seed in range(4096):
        state = pa.adamw8_state(p)
        pa.adamw8_([p.clone()], [grad], [state], 1, seed=seed, **HOW)
        m, v = pa.adamw8_moments(p, state)
        sums += torch.stack((m, v.sqrt())).double()
    for got, want in zip((sums / 4096).cpu(), (0.1 * grad.double().cpu(), 0.1 * grad.double().cpu().abs())):
        _, step = grid(want, torch.zeros(n, dtype=torch.int64), False)
        big = want.abs() > 8 * step                       # (beside the lowest codes of the root, which never become zero)
        assert ((got - want).abs() <= 5 * 0.5 / 64 * step)[big].all()


def test_a_decaying_moment_leaves_its_code(gpu):
    """300 steps of gradients of zero: the second moment falls to 0.999^300 = 0.74 of itself, its root to 0.861 (the mean of 4096 elements: a step moves a root by 0.0005 of itself and rounds it with a variance
    of at most that times the distance of two codes, an eighth: a deviation of sqrt(300 * 0.0005 / 8) = 0.14 an element, 0.0022 of the mean); rounded to nearest it would not move at all."""
    p = torch.zeros(4096, device=gpu)
    grad, state = torch.ones_like(p), pa.adamw8_state(p)
    how = dict(lr=0.0, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    pa.adamw8_([p], [grad], [state], 1, **how)
    first = float(pa.adamw8_moments(p, state)[1].sqrt().double().mean())
    for t in range(2, 302):
        pa.adamw8_([p], [torch.zeros_like(p)], [state], t, **how)
    last = float(pa.adamw8_moments(p, state)[1].sqrt().double().mean())
    assert abs(last / first - 0.999 ** 150) <= 5 * 0.0022


@pytest.mark.parametrize("scale", [1e-38, 1e-30, 1e-12, 1e12])
def test_small_and_large_moments(gpu, scale):
    """Scales of every size; what lies far under the largest of its 32 rounds to zero or a lowest code."""
    n = 1000
    g = torch.Generator().manual_seed(3)
    grad = (torch.randn(n, generator=g) * torch.exp(6 * torch.randn(n, generator=g)) * scale).to(gpu)
    p, state = torch.zeros(n, device=gpu), pa.adamw8_state(torch.zeros(n))
    state = state.to(gpu)
    pa.adamw8_([p], [grad], [state], 1, seed=5, **HOW)
    m, _ = pa.adamw8_moments(p, state)
    q, step = grid((1 - 0.9) * grad.double().cpu(), random_bits(n, 0, 1, 5) & 0xffff, False)
    d = (m.double().cpu() - q).abs()
    assert (d <= step * 1.0001 + 2.0 ** -148).all() and int((d > 0.01 * step + 2.0 ** -148).sum()) <= 4


def test_values_that_are_not_finite(gpu):
    for eight in (False, True):
        for bad in (math.inf, -math.inf, math.nan):
            g = torch.ones(1000, device=gpu)
            g[5] = bad
            p = torch.zeros(1000, device=gpu)
            if eight:
                state = pa.adamw8_state(p)
                for t in (1, 2):
                    pa.adamw8_([p], [g], [state], t, **HOW)
                m, v = pa.adamw8_moments(p, state)
            else:
                m, v = torch.zeros_like(p), torch.zeros_like(p)
                for t in (1, 2):
                    pa.adamw_([p], [g], [m], [v], t, **HOW)
            rest = torch.arange(1000, device=gpu) != 5
            assert not torch.isfinite(p[5]) and not torch.isfinite(m[5]) and not torch.isfinite(v[5])
            for x in (p, m, v):
                assert torch.isfinite(x[rest]).all() and (x[rest] == x[0]).all() if not eight else torch.isfinite(x[rest]).all()


def test_same_bits_whatever_the_launch(gpu):
    """A tensor alone, among others, on another stream and replayed from a graph."""
    s = make([5000, 300, 70_000], F32, F32, gpu, 9)
    for eight in (False, True):
        def fresh():
            return ([x.clone() for x in s["params"]], [pa.adamw8_state(x) for x in s["params"]]) if eight else ([x.clone() for x in s["params"]], [[x.clone() for x in s["m"]], [x.clone() for x in s["v"]]])

        def go(params, state, step, grads=s["grads"]):
            pa.adamw8_(params, grads, state, step, **HOW) if eight else pa.adamw_(params, grads, *state, step, **HOW)

        def all_of(params, state):
            return params + (state if eight else state[0] + state[1])
        a, sa = fresh()
        for t in range(1, 5):
            go(a, sa, t)
        b, sb = fresh()
        step = torch.zeros((), dtype=torch.int64, device=gpu)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            go(b, sb, step)
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            go(b, sb, step)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            torch.randn(1000, device=gpu).sum()
        assert int(step) == 4
        for x, y in zip(all_of(a, sa), all_of(b, sb)):
            if eight:
                same = float((x == y).double().mean())        # (coefficients in float64 on either side, rounded to fp32: a last bit may differ)
                assert same > 1 - 2.0 ** -10
            else:
                assert ((x - y).abs() <= 64 * U * (x.abs() + 0.02)).all()


# ---------------------------------------------------------------------------------------------------- the optimizer

def losses(model, opt, x, y, steps, clip=None):
    out = []
    for _ in range(steps):
        opt.zero_grad()
        loss = (model(x) - y).square().mean()
        loss.backward()
        if clip is not None:
            torch.nn.utils.clip_grad_norm_(model.parameters(), clip)
        opt.step()
        out.append(float(loss.detach()))
    return out


def network(gpu, dtype=F32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(19, 33), torch.nn.GELU(), torch.nn.Linear(33, 7)).to(gpu).to(dtype)


@pytest.mark.parametrize("max_norm", [None, 0.3])
def test_as_torchs(gpu, max_norm):
    """Ten steps beside torch.optim.AdamW's on the same gradients: a step's bar (19 u of terms of at most 10 lr, 3 u of the weight), ten times, and what it moves the gradients by."""
    ours, theirs = network(gpu), network(gpu)
    x, y = torch.randn(50, 19, device=gpu), torch.randn(50, 7, device=gpu)
    how = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=0.05)
    a, b = pa.AdamW(ours.parameters(), max_norm=max_norm, **how), torch.optim.AdamW(theirs.parameters(), **how)
    for _ in range(10):
        theirs.zero_grad()
        (theirs(x) - y).square().mean().backward()
        for p, q in zip(ours.parameters(), theirs.parameters()):
            p.grad = q.grad.clone()
        if max_norm is not None:
            norm = torch.nn.utils.clip_grad_norm_(theirs.parameters(), max_norm)
        b.step()
        a.step()
        if max_norm is not None:
            assert abs(float(a.norm) - float(norm)) <= 1e-6 * float(norm)
    for p, q in zip(ours.parameters(), theirs.parameters()):
        assert ((p - q).abs() <= 10 * 64 * U * (q.abs() + 0.1)).all()
        assert a.state[p]["step"] == 10 and (a.state[p]["exp_avg"] - b.state[q]["exp_avg"]).abs().max() <= 1e-5 * b.state[q]["exp_avg"].abs().max()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype,master", [(F32, False), (BF16, True), (BF16, False)])
def test_optimizer_resumes(gpu, bits, dtype, master):
    """Five steps, saved and loaded, five more: the bits of ten."""
    x, y = torch.randn(50, 19, device=gpu, dtype=dtype), torch.randn(50, 7, device=gpu, dtype=dtype)
    how = dict(lr=1e-2, bits=bits, master_weights=master, max_norm=1.0, seed=5)
    a = network(gpu, dtype)
    oa = pa.AdamW(a.parameters(), **how)
    losses(a, oa, x, y, 10)
    b = network(gpu, dtype)
    ob = pa.AdamW(b.parameters(), **how)
    losses(b, ob, x, y, 5)
    saved = copy.deepcopy((b.state_dict(), ob.state_dict()))
    c = network(gpu, dtype)
    oc = pa.AdamW(c.parameters(), **how)
    c.load_state_dict(saved[0])
    oc.load_state_dict(saved[1])
    losses(c, oc, x, y, 5)
    assert all(torch.equal(p, q) for p, q in zip(a.parameters(), c.parameters()))
    for p, q in zip(a.parameters(), c.parameters()):
        for k, v in oa.state[p].items():
            w = oc.state[q][k]
            assert (torch.equal(v, w) and v.dtype == w.dtype) if isinstance(v, torch.Tensor) else v == w
    other = pa.AdamW(network(gpu, dtype).parameters(), **{**how, "bits": 40 - bits})
    with pytest.raises(ValueError, match="keeps"):
        other.load_state_dict(saved[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_takes_over_from_torchs(gpu, dtype):
    """Five steps of torch.optim.AdamW, its state loaded, and five more beside its own: as far off as five steps are from them (16-bit moments are rounded at each of torch's: eps / 2 of a moment and step,
    so 8 eps of an update of lr; and the weights, half a step of theirs at each)."""
    ours, theirs = network(gpu, dtype), network(gpu, dtype)
    how = dict(lr=1e-2, betas=(0.9, 0.99), weight_decay=0.05)
    a, b = pa.AdamW(ours.parameters(), **how), torch.optim.AdamW(theirs.parameters(), **how)
    x, y = torch.randn(50, 19, device=gpu, dtype=dtype), torch.randn(50, 7, device=gpu, dtype=dtype)
    losses(theirs, b, x, y, 5)
    ours.load_state_dict(theirs.state_dict())
    a.load_state_dict(copy.deepcopy(b.state_dict()))
    for p, q in zip(ours.parameters(), theirs.parameters()):
        assert a.state[p]["step"] == 5 and a.state[p]["exp_avg"].dtype == F32 and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"].float())
    for _ in range(5):
        theirs.zero_grad()
        (theirs(x) - y).square().mean().backward()
        for p, q in zip(ours.parameters(), theirs.parameters()):
            p.grad = q.grad.clone()
        b.step()
        a.step()
    h = torch.finfo(dtype).eps / 2 if dtype == BF16 else 64 * U
    for p, q in zip(ours.parameters(), theirs.parameters()):
        assert a.state[p]["step"] == 10 and ((p - q).abs() <= 5 * (4 * h * (q.abs() + 0.05) + 16 * h * 1e-2)).all()
    state = b.state_dict()
    state["param_groups"][0]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        a.load_state_dict(state)


def test_parameters_that_begin_later(gpu):
    """A parameter without a gradient is left out of a step and its count; mixed types go together."""
    a, b = torch.nn.Parameter(torch.ones(700, device=gpu)), torch.nn.Parameter(torch.ones(300, device=gpu, dtype=BF16))
    for bits in (32, 8):
        opt = pa.AdamW([a, b], bits=bits, master_weights=True)
        a.grad, b.grad = torch.ones_like(a), None
        opt.step()
        assert b not in opt.state
        b.grad, start = torch.ones_like(b), float(b[0].detach())
        opt.step()
        # (0.00101 below 1 or the next lower number is less than half a step of bf16, 2^-9: the master weight holds it)
        assert opt.state[a]["step"] == 2 and opt.state[b]["step"] == 1 and "master" not in opt.state[a]
        assert opt.state[b]["master"].dtype == F32 and float((opt.state[b]["master"] - (start * (1 - 1e-5) - 1e-3)).abs().max()) <= 4 * U and bool((b == start).all())
        assert opt.step(lambda: torch.tensor(3.0)) == 3.0


@pytest.mark.parametrize("bits", [32, 8])
def test_driven_by_a_schedule_and_a_gradient_scaler(gpu, bits):
    """The same steps as with the rate set and the gradients divided by hand (by a power of two, so exactly); a step with an infinite gradient is left out."""
    a, b = network(gpu), network(gpu)
    oa, ob = (pa.AdamW(m.parameters(), lr=0.02, bits=bits, seed=1) for m in (a, b))
    schedule = torch.optim.lr_scheduler.LambdaLR(oa, lambda t: 0.5 ** t)
    scaler = torch.amp.GradScaler("cuda", init_scale=1024.0)
    x, y = torch.randn(50, 19, device=gpu), torch.randn(50, 7, device=gpu)
    for t in range(4):
        oa.zero_grad()
        scaler.scale((a(x) - y).square().mean()).backward()
        before = [p.detach().clone() for p in a.parameters()]
        if t == 2:
            next(a.parameters()).grad[0, 0] = math.inf
        else:
            ob.param_groups[0]["lr"] = 0.02 * 0.5 ** t
            for p, q in zip(a.parameters(), b.parameters()):
                q.grad = p.grad / scaler.get_scale()
            ob.step()
        scaler.step(oa)
        scaler.update()
        schedule.step()
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))
        assert t != 2 or all(torch.equal(p, q) for p, q in zip(a.parameters(), before))
    assert all(s["step"] == 3 for s in oa.state.values())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_optimizer(gpu, bits):
    """A captured step with clipping and a rate that a schedule fills, replayed, beside eager steps; the norm's kernels and the step's are in the graph."""
    results = []
    for captured in (False, True):
        p = [torch.nn.Parameter(x.clone()) for x in make([4000, 33, 999], F32, F32, gpu, 11)["params"]]
        lr = torch.full((), 1e-2, device=gpu)
        opt = pa.AdamW([{"params": p[:2]}, {"params": p[2:], "weight_decay": 0.0}], lr=lr, bits=bits, max_norm=0.5, capturable=True, seed=3)
        for q in p:
            q.grad = torch.ones_like(q)

        def set_gradients(t):
            for i, q in enumerate(p):
                g = torch.Generator().manual_seed(100 * t + i)
                q.grad.copy_(torch.randn(q.shape, generator=g).to(gpu))
            lr.fill_(1e-2 / (t + 1))
        set_gradients(0)
        opt.step()
        graph = torch.cuda.CUDAGraph()
        if captured:
            with torch.cuda.graph(graph):
                opt.step()
        for t in range(1, 4):
            set_gradients(t)
            graph.replay() if captured else opt.step()
            torch.cuda.synchronize()
        assert [int(g["steps"]) for g in opt.param_groups] == [4, 4]
        results.append([q.detach().clone() for q in p] + [x for q in p for x in opt.state[q].values()])
    for x, y in zip(*results):
        assert torch.equal(x, y)
    q = torch.nn.Parameter(torch.ones(5, device=gpu))
    opt.add_param_group({"params": [q]})
    q.grad = torch.ones_like(q)
    opt.step()
    p[0].grad = None
    with pytest.raises(RuntimeError, match="together"):
        opt.step()


def test_offsets_beyond_32_bits(gpu):
    """A tensor of 2^31 + 4099 bf16 elements with moments in 8 bits: its first and last elements, and those about 2^31, as the formula has them."""
    n = 2 ** 31 + 4099
    p = torch.zeros(n, dtype=BF16, device=gpu)
    g = torch.zeros(n, dtype=BF16, device=gpu)
    places = [0, 511, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 513, n - 1]
    for k, at in enumerate(places):
        g[at] = 0.5 + k
    state = pa.adamw8_state(p)
    pa.adamw8_([p], [g], [state], 1, **HOW)
    rows = [at // 512 for at in places]
    for k, (at, row) in enumerate(zip(places, rows)):
        assert abs(float(p[at]) + 3e-3) <= 3e-3 * 2.0 ** -8
        m, _ = pa.adamw8_moments(p[:512], state[row:row + 1])
        assert abs(float(m[at % 512]) - 0.1 * (0.5 + k)) <= 0.1 * (0.5 + k) / 8
    assert int((p != 0).sum()) == len(places)


@pytest.mark.parametrize("bits", [32, 8])
def test_capture_without_capturable_is_refused(gpu, bits):
    """After an eager step as before one: nothing of the step goes into the graph, and the optimizer goes on as if it had not been called."""
    results = []
    for tried in (False, True):
        p = torch.nn.Parameter(make([700], F32, F32, gpu, 4)["params"][0].clone())
        opt = pa.AdamW([p], lr=1e-2, bits=bits, max_norm=1.0)
        p.grad = torch.linspace(-1, 1, 700, device=gpu)
        opt.step()
        torch.cuda.synchronize()
        if tried:
            before = [x.clone() for x in (p.detach(), *[v for v in opt.state[p].values() if isinstance(v, torch.Tensor)])]
            count = torch.zeros(1, device=gpu)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                count += 1
                with pytest.raises(RuntimeError, match="capturable=True"):
                    opt.step()
            for _ in range(3):
                graph.replay()
            torch.cuda.synchronize()
            assert int(count) == 3 and opt.state[p]["step"] == 1
            assert all(torch.equal(a, b) for a, b in zip(before, (p.detach(), *[v for v in opt.state[p].values() if isinstance(v, torch.Tensor)])))
        opt.step()
        assert opt.state[p]["step"] == 2
        results.append([p.detach().clone()] + [v for v in opt.state[p].values() if isinstance(v, torch.Tensor)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("counted", [False, True])
def test_an_error_that_an_earlier_call_left(gpu, bits, counted):
    """It is not this step's, which is taken, and once."""
    from proteusai_amd import _lib
    lib = _lib.load()
    results = []
    for left in (False, True):
        c = make([3000, 77], F32, F32, gpu, 6)
        states = [pa.adamw8_state(p) for p in c["params"]] if bits == 8 else None
        step = torch.zeros((), dtype=torch.int64, device=gpu) if counted else 1
        torch.cuda.synchronize()
        if left:
            assert lib.hipSetDevice(100_000) != 0                            # (no such device: the host's own answer)
        if bits == 8:
            pa.adamw8_(c["params"], c["grads"], states, step, **HOW)
        else:
            pa.adamw_(c["params"], c["grads"], c["m"], c["v"], step, **HOW)
        lib.hipGetLastError()
        torch.cuda.synchronize()
        assert not counted or int(step) == 1
        results.append([*c["params"], *(states or c["m"] + c["v"])])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_captured_optimizer_resumes(gpu, bits, dtype):
    """Saved after three of eight steps: a fresh optimizer that loads it, steps, is captured and replayed, and one whose step was captured before it loads it, have the bits of the one that went on."""
    def optimizer(seed=11):
        p = [torch.nn.Parameter(x.clone()) for x in make([4000, 33, 999], dtype, dtype, gpu, seed)["params"]]
        rate = torch.full((), 1e-2, device=gpu)
        for q in p:
            q.grad = torch.ones_like(q)
        return p, rate, pa.AdamW([{"params": p[:2]}, {"params": p[2:], "weight_decay": 0.0}], lr=rate, bits=bits, max_norm=0.5, master_weights=True, capturable=True, seed=3)

    def prepare(p, rate, t):
        for i, q in enumerate(p):
            q.grad.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(100 * t + i)).to(gpu))
        rate.fill_(1e-2 / (t + 1))

    def captured(opt):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        return graph

    def run(p, rate, step, first, end):
        for t in range(first, end):
            prepare(p, rate, t)
            step()
            torch.cuda.synchronize()

    def load(p, opt):
        with torch.no_grad():
            for q, x in zip(p, saved[0]):
                q.copy_(x)
        opt.load_state_dict(saved[1])

    def result(p, opt):
        assert [int(g["steps"]) for g in opt.param_groups] == [8, 8]
        return [q.detach() for q in p] + [x for q in p for x in opt.state[q].values()]
    p, rate, opt = optimizer()
    run(p, rate, opt.step, 0, 3)
    saved = copy.deepcopy(([q.detach() for q in p], opt.state_dict()))
    run(p, rate, opt.step, 3, 8)
    want = result(p, opt)
    p, rate, opt = optimizer(12)                                            # fresh: its own rate tensor is filled, and read
    load(p, opt)
    assert opt.param_groups[0]["lr"] is rate
    run(p, rate, opt.step, 3, 4)
    run(p, rate, captured(opt).replay, 4, 8)
    assert all(torch.equal(a, b) for a, b in zip(want, result(p, opt)))
    p, rate, opt = optimizer(13)                                            # captured before
    run(p, rate, opt.step, 0, 1)
    graph = captured(opt)
    run(p, rate, graph.replay, 1, 3)
    load(p, opt)
    run(p, rate, graph.replay, 3, 8)
    assert all(torch.equal(a, b) for a, b in zip(want, result(p, opt)))
    p[0].grad = None
    with pytest.raises(RuntimeError, match="together"):
        opt.step()


@pytest.mark.parametrize("beta2", [0.999, 0.5])
@pytest.mark.parametrize("exponent", [-20, -60, -74, -76, -100, -118])
def test_roots_whose_squares_are_below_fp32(gpu, exponent, beta2):
    """Steps of gradients of zero from roots of 1 to 15/8 times 2^exponent, with eps = 0: none becomes zero, each is within a distance of two codes (an eighth; a root that fp32's subnormal squares stand for, half
    of itself) of sqrt(beta2) times what it was, and the update, of first moments of zero, is zero and not NaN."""
    n = 512
    p, grad = torch.ones(n, device=gpu), torch.zeros(n, device=gpu)
    state = pa.adamw8_state(p)
    state[0, 512:1024] = (0x38 + torch.arange(n, device=gpu) % 8).to(torch.uint8)
    state[0, 1024:] = 127 + exponent

    def roots():
        codes = state[0, 512:1024].view(torch.float8_e4m3fn).double().view(16, 32)
        return (codes * torch.exp2(state[0, 1040:].double() - 127)[:, None]).view(-1)
    for t in range(1, 6):
        before = roots()
        pa.adamw8_([p], [grad], [state], t, lr=1e-3, betas=(0.9, beta2), eps=0.0, weight_decay=0.0)
        after, want = roots(), before * math.sqrt(beta2)
        assert bool((after > 0).all()) and bool((p == 1).all())
        squares = exponent < -55                                             # (of 2^-126 and less)
        assert bool(((after - want).abs() <= want * (0.5 if squares else 0.125) + 2.0 ** -136).all())


@pytest.mark.parametrize("ptype,gtype,master", [(F16, F16, False), (F16, F32, True)], ids=lambda x: str(x).split(".")[-1])
def test_the_other_kinds_of_tensors(gpu, ptype, gtype, master):
    for sizes in SIZES[:6]:
        test_step(gpu, sizes, ptype, gtype, master)
        test_step_of_8_bits(gpu, sizes, ptype, gtype, master)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("t", [2 ** 32, 2 ** 32 + 1, 2 ** 40])
def test_steps_whose_number_passes_32_bits(gpu, bits, t):
    """Given as a number or on the GPU, with a rate that is a number or on the GPU."""
    c = make([700], F32, F32, gpu, 8)
    start = c["params"][0]
    m, v = torch.zeros_like(start), torch.zeros_like(start)
    want, _, _, bar = formula(start, c["grads"][0], m, v, t, **{**HOW, "lr": 2.0 ** -8})[:4]
    for on_gpu in (False, True):
        for lr in (2.0 ** -8, torch.full((), 2.0 ** -8, device=gpu)):
            p, step = start.clone(), torch.full((), t - 1, dtype=torch.int64, device=gpu) if on_gpu else t
            if bits == 8:
                pa.adamw8_([p], c["grads"], [pa.adamw8_state(p)], step, **{**HOW, "lr": lr})
            else:
                pa.adamw_([p], c["grads"], [m.clone()], [v.clone()], step, **{**HOW, "lr": lr})
            off(p, want, bar)
            assert not on_gpu or int(step) == t
