"""The two ends of a training step, what is timed, and their plain forms: the loss of the encoder's head and the optimizer.

  ce      pa.linear_cross_entropy: softmax cross entropy of x W' + b over a vocabulary, forward or forward + backward
  adamw   pa.adamw_: an AdamW step over many tensors, moments in 32 bits
  adamw8  pa.adamw8_: the same, moments in 8 bits: rows of 1056 bytes for 512 elements of a tensor, 512 codes (e4m3) of the first moment, 512 of the root of the second,
          16 + 16 scales (powers of two, e8m0), each for 32 elements

A case's sizes are fixed; the seed gives the values, which tokens are left out and the rounding.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
IGNORED = -100
BETAS, EPS, DECAY, LR = (0.9, 0.999), 1e-8, 0.01, 3e-4
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
ROW, CODES, GROUP = 1056, 512, 32                           # bytes and elements of a row of 8-bit moments, elements of a scale


# ---------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # twenty residues of one sequence scored: a launch-latency-sized call
        dict(name="ce_20x20", kind="ce", M=20, D=512, V=20, dtype="bf16", bias=True, smoothing=0.0, reduction="none", left_out=0.0, train=False),
        # the encoder's head on a padded training batch of 8 x 1024 residues, fp32 weights
        dict(name="ce_8192x20_f32_train", kind="ce", M=8192, D=512, V=20, dtype="f32", bias=True, smoothing=0.0, reduction="mean", left_out=0.44, train=True),
        # the small training batch (4 x 512 residues) against 1000 structure tokens, fp32 weights
        dict(name="ce_2048x1000_f32_train", kind="ce", M=2048, D=512, V=1000, dtype="f32", bias=True, smoothing=0.1, reduction="mean", left_out=0.1, train=True),
        # 2000 masked residues against a vocabulary of residue triplets, each token with a weight of its own
        dict(name="ce_2000x8001_f16_train", kind="ce", M=2000, D=768, V=8001, dtype="f16", bias=True, smoothing=0.1, reduction="none", left_out=0.0, train=True),
        # a ragged batch packed without padding, sizes that are no multiples of a tile
        dict(name="ce_5003x20011_train", kind="ce", M=5003, D=712, V=20011, dtype="bf16", bias=True, smoothing=0.0, reduction="sum", left_out=0.05, train=True),
        # a large batch of a wide model and a large vocabulary without bias
        dict(name="ce_16384x65536_train", kind="ce", M=16384, D=2048, V=65536, dtype="bf16", bias=False, smoothing=0.0, reduction="mean", left_out=0.0, train=True),
        # the encoder of four layers (d_model 512, 8 heads, feed-forward 2048) in fp32, gradients scaled by the clipping's factor, the number of steps on the GPU
        dict(name="adamw_encoder", kind="adamw", layers=4, D=512, F=2048, count=0, numel=0, dtype="f32", grad="f32", master=False, clip=True, on_gpu=True),
        # 500 odd-sized small tensors in bf16 with fp32 master weights
        dict(name="adamw_500_small", kind="adamw", layers=0, D=0, F=0, count=500, numel=600_000, dtype="bf16", grad="bf16", master=True, clip=False, on_gpu=False),
        # 350 million fp32 parameters of a large model, gradients in bf16
        dict(name="adamw_350m", kind="adamw", layers=0, D=0, F=0, count=140, numel=350_000_000, dtype="f32", grad="bf16", master=False, clip=True, on_gpu=False),
        # one head's weight and bias
        dict(name="adamw8_head", kind="adamw8", layers=0, D=0, F=0, count=2, numel=10_260, dtype="f32", grad="f32", master=False, clip=False, on_gpu=False),
        # the encoder again, moments in 8 bits
        dict(name="adamw8_encoder", kind="adamw8", layers=4, D=512, F=2048, count=0, numel=0, dtype="f32", grad="f32", master=False, clip=True, on_gpu=True),
        # 350 million bf16 parameters with fp32 master weights, moments in 8 bits
        dict(name="adamw8_350m", kind="adamw8", layers=0, D=0, F=0, count=140, numel=350_000_000, dtype="bf16", grad="bf16", master=True, clip=True, on_gpu=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["ce", "ce", "ce", "adamw", "adamw8"])
    if kind == "ce":
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        D, V = 8 * _log_int(rng, 8, 256), _log_int(rng, 2, 65536)
        M = _log_int(rng, 1, max(1, min(16384, (2 ** 38 if dtype != "f32" else 2 ** 35) // (D * V))))
        return dict(kind=kind, M=M, D=D, V=V, dtype=dtype, bias=rng.random() < 0.6, smoothing=rng.choice([0.0, 0.0, 0.1]), reduction=rng.choice(["mean", "mean", "sum", "none"]),
                    left_out=rng.choice([0.0, 0.1, 0.5]) if M > 8 else 0.0, train=rng.random() < 0.7)
    dtype = rng.choice(["f32", "f32", "bf16", "f16"])
    grad = rng.choice(["f32", "bf16", "f16"]) if dtype == "f32" else rng.choice([dtype, dtype, "f32"])
    numel = _log_int(rng, 1000, 2 * 10 ** 8)
    return dict(kind=kind, layers=0, D=0, F=0, count=_log_int(rng, 1, min(600, max(1, numel // 100))), numel=numel, dtype=dtype, grad=grad,
                master=dtype != "f32" and rng.random() < 0.6, clip=rng.random() < 0.5, on_gpu=rng.random() < 0.5)


def _sizes(case):
    """Numbers of elements of the tensors: the encoder's, or spread over three decades about their mean."""
    if case["layers"]:
        D, F = case["D"], case["F"]
        layer = 4 * [D * D] + 3 * [D] + [8] + 4 * [D] + [F * D, F, D * F, D]
        return case["layers"] * layer + [D // 2, 33 * D, 20 * D, 20]
    rng = np.random.default_rng(case["count"])
    weight = np.exp(rng.uniform(0.0, math.log(1000.0), case["count"]))
    return [max(1, int(n)) for n in weight / weight.sum() * case["numel"]]


def _counted(case):
    """Tokens that count."""
    return case["M"] - int(case["M"] * case["left_out"])


# ---------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)
    s = dict(case=case)
    if case["kind"] == "ce":
        M, D, V, t = case["M"], case["D"], case["V"], TYPES[case["dtype"]]
        # normed features, logits of a deviation of 2; every token's own word stands out, by nothing to plenty
        w = randn(V, D) * (2.0 * D ** -0.5)
        target = torch.randint(0, V, (M,), generator=g, device=DEV)
        x = randn(M, D) + w[target] * (2.5 * torch.rand(M, 1, generator=g, device=DEV))
        if case["left_out"]:
            target[torch.randperm(M, generator=g, device=DEV)[_counted(case):]] = IGNORED
        s["x"], s["w"], s["b"], s["target"] = x.to(t), w.to(t), randn(V).to(t) if case["bias"] else None, target
        s["leaves"] = [p for p in (s["x"], s["w"], s["b"]) if p is not None]
        if case["train"]:
            for p in s["leaves"]:
                p.requires_grad_()
            if case["reduction"] == "none":
                s["d"] = torch.rand(M, generator=g, device=DEV) / M
        return s
    sizes = _sizes(case)
    # the tensors lie one behind the other; those whose moments are in 8 bits begin at a multiple of 512 elements (nothing but zeros lies between)
    spans = [-(-n // CODES) * CODES for n in sizes] if case["kind"] == "adamw8" else sizes
    # gradients of trained layers: sizes of their elements differ by orders of magnitude from tensor to tensor, and within one
    scale = np.exp(np.random.default_rng(seed).normal(-7.0, 1.5, len(sizes)))
    counts = torch.tensor(spans, device=DEV)
    per = torch.repeat_interleave(torch.tensor(scale, dtype=torch.float32, device=DEV), counts, output_size=sum(spans))
    if spans != sizes:
        inside = torch.arange(sum(spans), device=DEV) - torch.repeat_interleave(torch.cumsum(counts, 0) - counts, counts, output_size=sum(spans))
        per = torch.where(inside < torch.repeat_interleave(torch.tensor(sizes, device=DEV), counts, output_size=sum(spans)), per, 0.0)
        del inside
    n = sum(spans)
    per = per * torch.exp(randn(n))
    grad = (per * randn(n)).to(TYPES[case["grad"]])
    first, second = 0.3 * per * randn(n), per * (0.5 + torch.rand(n, generator=g, device=DEV))          # the moment and the root of the second
    weight = torch.where(per > 0.0, 0.05 * randn(n), 0.0)
    s["p"], s["g"] = weight.to(TYPES[case["dtype"]]), grad
    s["master"] = weight if case["master"] else None

    def parts(flat):
        return [c[:k] for c, k in zip(flat.split(spans), sizes)]
    s["params"], s["grads"], s["masters"] = parts(s["p"]), parts(grad), parts(weight) if case["master"] else None
    if case["kind"] == "adamw":
        s["m"], s["v"] = first, second.square_()
        s["ms"], s["vs"] = parts(s["m"]), parts(s["v"])
    else:
        s["state"] = torch.zeros(n // CODES, ROW, dtype=torch.uint8, device=DEV)
        _pack(s["state"], first, second, torch.full((1,), 1 << 15, dtype=torch.int32, device=DEV), torch.full((1,), 1 << 15, dtype=torch.int32, device=DEV))
        s["states"] = list(s["state"].split([k // CODES for k in spans]))
        s["rows"] = torch.tensor([k // CODES for k in spans], device=DEV)
        s["seed"] = seed
    s["norm"] = 2.0 * torch.linalg.vector_norm(grad.float()) if case["clip"] else None      # (as if there were others)
    s["max_norm"] = 1.0 if case["clip"] else None
    s["step"] = torch.full((), 99, dtype=torch.int64, device=DEV) if case["on_gpu"] else 100         # steps done, or the number of this one
    return s


# ---------------------------------------------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    return _plain_ce(s, case) if case["kind"] == "ce" else _plain_adamw(s, case)


def _run_own(s, case):
    import proteusai_amd as pa
    if case["kind"] == "ce":
        loss = pa.linear_cross_entropy(s["x"], s["w"], s["target"], s["b"], ignore_index=IGNORED, label_smoothing=case["smoothing"], reduction=case["reduction"])
        return [loss, *torch.autograd.grad(loss, s["leaves"], s.get("d"))] if case["train"] else [loss]
    how = dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, masters=s["masters"], norm=s["norm"], max_norm=s["max_norm"])
    if case["kind"] == "adamw":
        pa.adamw_(s["params"], s["grads"], s["ms"], s["vs"], s["step"], **how)
    else:
        pa.adamw8_(s["params"], s["grads"], s["states"], s["step"], seed=s["seed"], **how)
    return _results(s, case)


def _results(s, case):
    got = [s["p"]] + ([s["master"]] if case["master"] else [])
    if case["kind"] == "adamw":
        return got + [s["m"], s["v"]]
    c8, s8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    st = s["state"]
    return got + [st[:, :CODES].view(c8), st[:, CODES:2 * CODES].view(c8), st[:, 2 * CODES:2 * CODES + 16].view(s8), st[:, 2 * CODES + 16:].view(s8)]


def _plain_ce(s, case):
    t, eps = TYPES[case["dtype"]], case["smoothing"]
    x, w, b = (None if p is None else p.detach().float() for p in (s["x"], s["w"], s["b"]))
    V, counts = case["V"], s["target"] != IGNORED
    at = torch.where(counts, s["target"], 0)[:, None]
    logits = x @ w.t() if b is None else x @ w.t() + b
    wanted = logits.gather(1, at)
    loss = eps * wanted[:, 0] - eps / V * logits.sum(1) if eps else 0.0
    # the other words apart: next to a word that is all but certain their sum is what counts
    p = logits.scatter_(1, at, -math.inf)
    most = p.amax(1, keepdim=True)
    p = torch.exp(p - most)
    total = p.sum(1, keepdim=True)
    ahead = most + torch.log(total) - wanted
    loss = loss + (torch.clamp_min(ahead, 0.0) + torch.log1p(torch.exp(-ahead.abs())))[:, 0]
    loss = torch.where(counts, loss, 0.0)
    number = counts.sum()
    if case["reduction"] != "none":
        loss = loss.double().sum()
        loss = (loss / number if case["reduction"] == "mean" else loss).float()
    if not case["train"]:
        return [loss]
    missed = torch.sigmoid(ahead)                           # 1 - the probability of the wanted word
    p *= missed / total
    p -= eps / V
    p.scatter_(1, at, eps - eps / V - missed)
    d = counts.float()
    d = d * s["d"] if case["reduction"] == "none" else d / number if case["reduction"] == "mean" else d
    p *= d[:, None]
    return [loss, (p @ w).to(t), (p.t() @ x).to(t)] + ([] if b is None else [p.sum(0).to(t)])


def _mix(x):
    """A mix of 32 bits (xor and shift, two products), on whole numbers of 64."""
    x = x ^ (x >> 16)
    x = (x * 0x7feb352d) & 0xffffffff
    x = x ^ (x >> 15)
    x = (x * 0x846ca68b) & 0xffffffff
    return x ^ (x >> 16)


def _random(s, step):
    """32 random bits for each element: of the seed, the step, the tensor's number and the element's in it."""
    rows = s["rows"]
    n = s["state"].shape[0]
    tensor = torch.repeat_interleave(torch.arange(len(rows), device=DEV), rows, output_size=n)
    row = torch.arange(n, device=DEV) - torch.repeat_interleave(torch.cumsum(rows, 0) - rows, rows, output_size=n)
    element = row[:, None] * CODES + torch.arange(CODES, device=DEV)
    step = torch.as_tensor(step, device=DEV)
    key = _mix((s["seed"] + (step & 0xffffffff) * 0x9e3779b1) & 0xffffffff)
    key = _mix((key + tensor[:, None] * 0x85ebca6b + (element >> 32) * 0xc2b2ae35) & 0xffffffff)
    return _mix(key ^ (element & 0xffffffff))


def _round8(x, random):
    """Codes (e4m3) and scales (e8m0) of x [rows, 512], each |x| rounded up with the probability of what is cut off (random: 16 bits)."""
    size = x.abs()
    most = size.view(-1, CODES // GROUP, GROUP).amax(2).view(torch.int32)
    # the least power of two by which the largest is at most 448
    scale = torch.clamp_min((most >> 23) - 8 + ((most & 0x7fffff) > 0x600000).int(), 0)
    small = (size.view(-1, CODES // GROUP, GROUP).double() * torch.exp2((7 - scale).double())[:, :, None]).float()     # e4m3's exponents are fp32's lowest
    code = ((small.view(torch.int32).view(-1, CODES) + (random << 4)) >> 20)
    return torch.where(x < 0.0, code | 0x80, code).to(torch.uint8), scale.to(torch.uint8)


def _pack(state, first, second, random1, random2):
    state[:, :CODES], state[:, 2 * CODES:2 * CODES + 16] = _round8(first.view(-1, CODES), random1)
    second = second.view(-1, CODES)
    codes, state[:, 2 * CODES + 16:] = _round8(second, random2)
    state[:, CODES:2 * CODES] = torch.where(second > 0.0, torch.clamp_min(codes, 1), codes)              # (what has been seen is not forgotten altogether)


def _value8(codes, scales):
    """What codes and scales stand for."""
    return (codes.view(torch.float8_e4m3fn).double().view(-1, CODES // GROUP, GROUP) * torch.exp2(scales.double() - 127.0)[:, :, None]).float().view(-1, CODES)


def _plain_adamw(s, case):
    b1, b2 = BETAS
    if case["on_gpu"]:
        s["step"] += 1
    step = torch.as_tensor(s["step"], device=DEV)
    c1, c2 = ((1.0 - b ** step.double()).float() for b in (b1, b2))
    g = s["g"].float()
    if case["clip"]:
        g = g * torch.clamp_max(s["max_norm"] / (s["norm"] + 1e-6), 1.0)
    shape, st = g.shape, s.get("state")
    if st is None:
        m, v = s["m"], s["v"]
    else:
        m, v = _value8(st[:, :CODES], st[:, 2 * CODES:2 * CODES + 16]).view(shape), _value8(st[:, CODES:2 * CODES], st[:, 2 * CODES + 16:]).square().view(shape)
    m = b1 * m + (1.0 - b1) * g
    v = b2 * v + (1.0 - b2) * g * g
    root = torch.sqrt(v)
    p = s["master"] if case["master"] else s["p"].float()
    p = p * (1.0 - LR * DECAY) - (LR / c1) * m / (root / torch.sqrt(c2) + EPS)
    if case["master"]:
        s["master"].copy_(p)
    s["p"].copy_(p)
    if st is None:
        s["m"].copy_(m)
        s["v"].copy_(v)
    else:
        del p, g, v
        random = _random(s, step)
        _pack(st, m, root, (random & 0xffff).int(), (random >> 16).int())
    return _results(s, case)


# ---------------------------------------------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_ce(s, case) if case["kind"] == "ce" else _exact_adamw(s, case)


def _exact_ce(s, case):
    """The mean over pieces of tokens of cross entropies against the smoothed target distribution; gradients from the difference of the two distributions."""
    x, w, b = (None if p is None else p.detach().double() for p in (s["x"], s["w"], s["b"]))
    M, V, eps = case["M"], case["V"], case["smoothing"]
    number = float(_counted(case))
    losses, dx, dw, db = [], [], torch.zeros_like(w), torch.zeros(V, dtype=torch.float64, device=DEV)
    for i in range(0, M, 2048):
        at = s["target"][i:i + 2048]
        counts = (at >= 0).double()
        log_p = torch.log_softmax(x[i:i + 2048] @ w.t() + (0.0 if b is None else b), 1)
        wanted = torch.full_like(log_p, eps / V)
        wanted[torch.arange(len(at), device=DEV), at.clamp_min(0)] += 1.0 - eps
        losses.append(-(wanted * log_p).sum(1) * counts)
        if case["train"]:
            d = counts * (s["d"][i:i + 2048].double() if case["reduction"] == "none" else 1.0 / number if case["reduction"] == "mean" else 1.0)
            p = (log_p.exp_() - wanted) * d[:, None]
            dx.append(p @ w)
            dw += p.t() @ x[i:i + 2048]
            db += p.sum(0)
    losses = torch.cat(losses)
    loss = losses if case["reduction"] == "none" else losses.sum() / (number if case["reduction"] == "mean" else 1.0)
    return [loss, torch.cat(dx), dw] + ([] if b is None else [db]) if case["train"] else [loss]


def _exact_adamw(s, case):
    """Tensor by tensor; of moments in 8 bits the values, rounded by the same random bits."""
    (b1, b2), t = BETAS, 100
    factor = min(1.0, s["max_norm"] / (float(s["norm"]) + 1e-6)) if case["clip"] else 1.0
    random = _random(s, t) if case["kind"] == "adamw8" else None
    out = dict(p=[], m=[], v=[])
    at = 0
    for i, g in enumerate(s["grads"]):
        n = g.numel()
        g = g.double() * factor
        p = (s["masters"] if case["master"] else s["params"])[i].double()
        if random is None:
            m, v = s["ms"][i].double(), s["vs"][i].double()
        else:
            st = s["states"][i]

            def value(k):
                sign_exponent_mantissa = st[:, k * CODES:(k + 1) * CODES].long().view(-1, CODES // GROUP, GROUP)
                e, f = (sign_exponent_mantissa >> 3) & 15, (sign_exponent_mantissa & 7).double()
                size = torch.where(e > 0, (8.0 + f) * 2.0 ** (e - 10).double(), f * 2.0 ** -9)
                size = size * 2.0 ** (st[:, 2 * CODES + 16 * k:2 * CODES + 16 * (k + 1)].long() - 127).double()[:, :, None]
                return torch.where(sign_exponent_mantissa >= 128, -size, size).reshape(-1)[:n]
            m, v = value(0), value(1) ** 2
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
        out["p"].append(p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS))
        out["m"].append(m)
        out["v"].append(v if random is None else v.sqrt())
    if random is None:
        p, m, v = (torch.cat(out[k]) for k in "pmv")
        return [p] * (2 if case["master"] else 1) + [m, v]

    def spread(parts):
        return torch.cat([torch.nn.functional.pad(x, (0, -len(x) % CODES)) for x in parts]).view(-1, CODES // GROUP, GROUP)

    def codes(x, bits, least):
        size = x.abs()
        most = size.amax(2)
        e = torch.where(most > 0, torch.ceil(torch.log2(torch.clamp_min(most, 1e-300) / 448.0)).clamp_min(-127.0), -127.0)
        size = size * torch.exp2(-e)[:, :, None]
        step = torch.exp2(torch.floor(torch.log2(size.clamp_min(2.0 ** -6))) - 3)
        size = torch.floor(size / step + bits.view(x.shape).double() / 65536.0) * step
        size = torch.where((x > 0) & (size == 0), 2.0 ** -9, size) if least else size
        return (torch.sign(x) * size).view(-1, CODES), torch.exp2(e)
    m, ms = codes(spread(out["m"]), random & 0xffff, False)
    v, vs = codes(spread(out["v"]), random >> 16, True)
    p = spread(out["p"]).reshape(-1)
    return [p] * (2 if case["master"] else 1) + [m, v, ms, vs]


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "ce":
        n, D, V, b = _counted(case), case["D"], case["V"], SIZE[case["dtype"]]
        weights = V * D + (V if case["bias"] else 0)
        both = 2 if case["train"] else 1
        return {"bytes": b * both * (n * D + weights) + 8 * case["M"] + (4 * case["M"] if case["reduction"] == "none" else 4), "flops": (3 if case["train"] else 1) * 2 * n * D * V}
    n = sum(_sizes(case))
    moments = 16 if case["kind"] == "adamw" else 4 * (1 + 1 / GROUP)
    weights = SIZE[case["dtype"]] + 8 if case["master"] else 2 * SIZE[case["dtype"]]
    return {"bytes": n * (SIZE[case["grad"]] + weights + moments), "flops": 15 * n}
