"""The operators that an encoder layer with normed, rotated queries and keys and a gated feed-forward block adds, and the clipping of
its training step: what is timed, and their plain forms.

  qk      pa.qk_norm_rotate: root-mean-square norm of every head's queries and keys and the rotation by position, one pass
  qkv     pa.qk_norm_rotate_qkv: the same on a fused projection [Z,N,3,H,d], values passed on in the result's type
  ffn     pa.gated_mlp: (act(x Wg' + bg) * (x Wu' + bu)) Wd' + bd, forward or forward + backward
  clip    pa.clip_grad_norm / pa.clip_grad_norm_: the norm over all gradients, and the gradients scaled to at most `max_norm`

A case's sizes are fixed; the seed gives the values, the padding's order and the chain breaks.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
BASE, EPS = 10000.0, 1e-6
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # 64 chains that each got one more residue, queries and keys of that residue alone: a launch-latency-sized call
        dict(name="qk_64x1_f16", kind="qk", Z=64, H=8, N=1, min_len=1, d=64, dtype="f16", out="f16", per_head=False, interleaved=False, far=True, train=False),
        # one protein through the encoder's inference: views of the fused projection, residues numbered from 0
        dict(name="qk_512", kind="qk", Z=1, H=8, N=512, min_len=512, d=64, dtype="bf16", out="bf16", per_head=False, interleaved=False, far=False, train=False),
        # a padded training batch with fp32 weights: projection in fp32, the attention's operands in bf16, weights of the norm per head
        dict(name="qkv_8x1024_padded_train", kind="qkv", Z=8, H=8, N=1024, min_len=128, d=64, dtype="f32", out="bf16", per_head=True, interleaved=False, far=True, train=True),
        # long chains with wide heads in bf16 training, neighbouring features paired
        dict(name="qk_2x16384_d128_train", kind="qk", Z=2, H=8, N=16384, min_len=16384, d=128, dtype="bf16", out="bf16", per_head=False, interleaved=True, far=False, train=True),
        # eight residues through the block: bound by reading the weights
        dict(name="ffn_8", kind="ffn", M=8, D=512, F=2048, dtype="bf16", act="silu", bias=True, train=False),
        # one protein of 512 residues, inference
        dict(name="ffn_512", kind="ffn", M=512, D=512, F=2048, dtype="bf16", act="silu", bias=True, train=False),
        # the encoder's small training batch (4 x 512 residues) on fp32 weights
        dict(name="ffn_2048_f32_train", kind="ffn", M=2048, D=512, F=2048, dtype="f32", act="gelu", bias=True, train=True),
        # a ragged batch packed without padding, widths that are no multiples of a tile
        dict(name="ffn_5003_train", kind="ffn", M=5003, D=712, F=1912, dtype="bf16", act="gelu", bias=True, train=True),
        # a large training batch of a wide layer without biases
        dict(name="ffn_32768_train", kind="ffn", M=32768, D=1024, F=4096, dtype="bf16", act="silu", bias=False, train=True),
        # the gradients of an encoder of four layers (d_model 512, 8 heads, feed-forward 2048) clipped into buffers of their own
        dict(name="clip_encoder", kind="clip", layers=4, D=512, F=2048, count=0, numel=0, dtype="f32", out="f32", p=2.0, ratio=0.5, inplace=False),
        # late in training: 500 odd-sized small gradients in place, their norm within the bound
        dict(name="clip_500_small", kind="clip", layers=0, D=0, F=0, count=500, numel=600_000, dtype="bf16", out="bf16", p=2.0, ratio=4.0, inplace=True),
        # 350 million bf16 gradients of a large model, clipped into fp32 for the optimizer
        dict(name="clip_350m", kind="clip", layers=0, D=0, F=0, count=140, numel=350_000_000, dtype="bf16", out="f32", p=2.0, ratio=0.1, inplace=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["qk", "qkv", "ffn", "ffn", "ffn", "clip"])
    if kind in ("qk", "qkv"):
        d, H = rng.choice([32, 64, 64, 128]), rng.choice([2, 4, 8, 12, 16])
        N = _log_int(rng, 1, 16384)
        Z = _log_int(rng, 1, max(1, min(64, 2 ** 25 // (N * H * d))))
        dtype = rng.choice(["f32", "bf16", "bf16", "f16"])
        padded = N > 1 and Z > 1 and rng.random() < 0.5
        return dict(kind=kind, Z=Z, H=H, N=N, min_len=max(1, N // rng.choice([2, 4, 8])) if padded else N, d=d, dtype=dtype,
                    out=rng.choice(["bf16", "f32"]) if dtype == "f32" else dtype, per_head=rng.random() < 0.5, interleaved=rng.random() < 0.4,
                    far=rng.random() < 0.5, train=rng.random() < 0.5)
    if kind == "ffn":
        dtype = rng.choice(["bf16", "bf16", "f32"])
        D, F = 8 * _log_int(rng, 8, 160), 8 * _log_int(rng, 16, 512)
        cost = 2 ** 37 if dtype == "bf16" else 2 ** 34
        M = _log_int(rng, 1, max(1, min(32768, cost // (D * F))))
        return dict(kind=kind, M=M, D=D, F=F, dtype=dtype, act=rng.choice(["silu", "silu", "gelu", "relu", "sigmoid"]), bias=rng.random() < 0.6, train=rng.random() < 0.6)
    dtype = rng.choice(["f32", "bf16", "f16"])
    inplace = rng.random() < 0.3
    numel = _log_int(rng, 2000, 2 * 10 ** 8)
    return dict(kind="clip", layers=0, D=0, F=0, count=_log_int(rng, 1, min(600, numel // 100)), numel=numel, dtype=dtype,
                out="f32" if not inplace and rng.random() < 0.5 else dtype, p=rng.choice([2.0, 2.0, 1.0, math.inf]),
                ratio=4.0 if inplace else rng.choice([0.01, 0.3, 2.0]), inplace=inplace)


def _lengths(case):
    Z, N, lo = case["Z"], case["N"], case["min_len"]
    return np.array([int(round(n)) for n in np.linspace(lo, N, Z)] if Z > 1 else [N])


def _sizes(case):
    """Numbers of elements of the gradients of a clip case: the encoder's tensors, or spread over three decades about their mean."""
    if case["layers"]:
        D, F = case["D"], case["F"]
        layer = 4 * [D * D] + 3 * [D] + [8] + 4 * [D] + [F * D, F, D * F, D]
        return case["layers"] * layer + [D // 2, 33 * D, 20 * D, 20]
    rng = np.random.default_rng(case["count"])
    weight = np.exp(rng.uniform(0.0, math.log(1000.0), case["count"]))
    return [max(1, int(n)) for n in weight / weight.sum() * case["numel"]]


# ---------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rng = np.random.default_rng(seed)

    def randn(*shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype or TYPES[case["dtype"]])
    s = dict(case=case)
    if case["kind"] in ("qk", "qkv"):
        Z, H, N, d = case["Z"], case["H"], case["N"], case["d"]
        # queries and keys differ in size from head to head, as a trained projection's do
        size = torch.exp(torch.randn(3, H, 1, generator=g, device=DEV))
        s["qkv"] = (torch.randn(Z, N, 3, H, d, generator=g, device=DEV) * size).to(TYPES[case["dtype"]])
        shape = (H, d) if case["per_head"] else (d,)
        s["qw"], s["kw"] = 1.0 + randn(*shape, scale=0.2), 1.0 + randn(*shape, scale=0.2)
        s["mask"] = s["positions"] = None
        if case["min_len"] < N:
            lens = torch.from_numpy(_lengths(case)[rng.permutation(Z)])
            s["mask"] = (torch.arange(N)[None, :] >= lens[:, None]).to(DEV)
        if case["far"]:
            # residue numbers: chains of an assembly one behind the other, 1000 numbers left out between them, some assemblies starting far on
            start, chain = rng.integers(0, 100_000, (Z, 1)), max(1, int(rng.integers(100, 400)))
            s["positions"] = torch.from_numpy(start + np.arange(N)[None, :] + 1000 * (np.arange(N)[None, :] // chain)).to(DEV)
        if case["train"]:
            if case["kind"] == "qkv":
                s["leaves"] = [s["qkv"].requires_grad_(), s["qw"].requires_grad_(), s["kw"].requires_grad_()]
                s["d"] = [randn(Z, N, 3, H, d, dtype=TYPES[case["out"]])]
            else:
                s["q"], s["k"] = (s["qkv"][:, :, i].permute(0, 2, 1, 3).requires_grad_() for i in range(2))
                s["leaves"] = [s["q"], s["k"], s["qw"].requires_grad_(), s["kw"].requires_grad_()]
                s["d"] = [randn(Z, N, H, d, dtype=TYPES[case["out"]]).permute(0, 2, 1, 3) for _ in range(2)]
        elif case["kind"] == "qk":
            s["q"], s["k"] = (s["qkv"][:, :, i].permute(0, 2, 1, 3) for i in range(2))
        return s
    if case["kind"] == "ffn":
        M, D, F = case["M"], case["D"], case["F"]
        s["leaves"] = [randn(M, D), randn(2 * F, D, scale=D ** -0.5), randn(2 * F, scale=0.1) if case["bias"] else None,
                       randn(D, F, scale=F ** -0.5), randn(D, scale=0.1) if case["bias"] else None]
        if case["train"]:
            s["d"] = randn(M, D)
            for t in s["leaves"]:
                if t is not None:
                    t.requires_grad_()
        return s
    # gradients of trained layers: sizes of their elements differ by orders of magnitude from tensor to tensor
    sizes = _sizes(case)
    scale = np.exp(rng.normal(-7.0, 1.5, len(sizes)))
    s["grads"] = [randn(n, scale=float(c)) for n, c in zip(sizes, scale)]
    squares = sum(n * c * c for n, c in zip(sizes, scale))
    expected = {2.0: math.sqrt(squares), 1.0: 0.8 * sum(n * c for n, c in zip(sizes, scale)), math.inf: 4.0 * max(scale)}[case["p"]]
    s["max_norm"] = float(case["ratio"] * expected)
    # what is written lies in one buffer, tensor behind tensor, as a bucket's gradients and an optimizer's do
    if case["inplace"]:
        s["flat"] = torch.cat(s["grads"])
        s["grads"] = list(s["flat"].split(sizes))
        s["params"] = [torch.nn.Parameter(torch.empty_like(t)) for t in s["grads"]]
        for p, t in zip(s["params"], s["grads"]):
            p.grad = t
    else:
        s["flat"] = torch.empty(sum(sizes), dtype=TYPES[case["out"]], device=DEV)
        s["out"] = list(s["flat"].split(sizes))
    return s


# ---------------------------------------------------------------------------------------------------- one pass

def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["kind"] in ("qk", "qkv"):
        return _plain_qk(s, case)
    return _plain_ffn(s, case) if case["kind"] == "ffn" else _plain_clip(s, case)


def _run_own(s, case):
    import proteusai_amd as pa
    if case["kind"] in ("qk", "qkv"):
        how = dict(positions=s["positions"], base=BASE, eps=EPS, interleaved=case["interleaved"], mask=s["mask"], out_dtype=TYPES[case["out"]])
        if case["kind"] == "qkv":
            outs = [pa.qk_norm_rotate_qkv(s["qkv"], s["qw"], s["kw"], **how)]
        else:
            outs = list(pa.qk_norm_rotate(s["q"], s["k"], s["qw"], s["kw"], **how))
        return outs + list(torch.autograd.grad(outs, s["leaves"], s["d"])) if case["train"] else outs
    if case["kind"] == "ffn":
        y = pa.gated_mlp(*s["leaves"], act=case["act"])
        return [y, *torch.autograd.grad(y, [t for t in s["leaves"] if t is not None], s["d"])] if case["train"] else [y]
    if case["inplace"]:
        norm = pa.clip_grad_norm_(s["params"], s["max_norm"], norm_type=case["p"])
    else:
        norm, _ = pa.clip_grad_norm(s["grads"], s["max_norm"], norm_type=case["p"], out=s["out"])
    return [norm, s["flat"]]


def _angles(s, case):
    """cos and sin [Z or 1, 1, N, d/2] of position * base^(-2i/d), from angles in 64 bits."""
    i = torch.arange(case["d"] // 2, device=DEV, dtype=torch.float64)
    pos = torch.arange(case["N"], device=DEV)[None] if s["positions"] is None else s["positions"]
    angle = pos.double()[:, None, :, None] * BASE ** (-2.0 * i / case["d"])
    return torch.cos(angle).float(), torch.sin(angle).float()


def _pairs(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)


def _joined(a, b, interleaved):
    return torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)


def _plain_qk(s, case):
    c, sn = _angles(s, case)
    keep = None if s["mask"] is None else ~s["mask"][:, None, :, None]
    inter, out_type = case["interleaved"], TYPES[case["out"]]
    if case["kind"] == "qkv":
        parts = [s["qkv"].detach()[:, :, i].permute(0, 2, 1, 3) for i in range(3)]
        grads = [s["d"][0][:, :, i].permute(0, 2, 1, 3) for i in range(3)] if case["train"] else None
    else:
        parts, grads = [s["q"].detach(), s["k"].detach()], s["d"] if case["train"] else None
    outs, dx, dw = [], [], []
    for i, weight in enumerate((s["qw"], s["kw"])):
        x = parts[i].float()
        w = weight.detach().float()
        w = w[:, None, :] if case["per_head"] else w
        if keep is not None:
            x = torch.where(keep, x, 0.0)
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        n = x * r
        a, b = _pairs(n * w, inter)
        y = _joined(a * c - b * sn, b * c + a * sn, inter)
        outs.append(y if keep is None else torch.where(keep, y, 0.0))
        if case["train"]:
            d = grads[i].float()
            if keep is not None:
                d = torch.where(keep, d, 0.0)
            a, b = _pairs(d, inter)
            d = _joined(a * c + b * sn, b * c - a * sn, inter)
            dw.append((d * n).sum((0, 2) if case["per_head"] else (0, 1, 2)).to(weight.dtype))
            d = d * w
            dx.append(r * (d - n * (d * n).mean(-1, keepdim=True)))
    if case["kind"] == "qk":
        result = [y.to(out_type) for y in outs]
        return result + [g.to(p.dtype) for g, p in zip(dx, parts)] + dw if case["train"] else result
    v = parts[2].float()
    outs.append(v if keep is None else torch.where(keep, v, 0.0))
    result = [torch.stack([y.permute(0, 2, 1, 3) for y in outs], 2).to(out_type)]
    if case["train"]:
        dv = grads[2].float()
        dx.append(dv if keep is None else torch.where(keep, dv, 0.0))
        result += [torch.stack([g.permute(0, 2, 1, 3) for g in dx], 2).to(s["qkv"].dtype)] + dw
    return result


def _act(g, act):
    """act(g) and its derivative."""
    if act == "relu":
        return torch.clamp_min(g, 0.0), (g > 0).to(g.dtype)
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (0.5 / math.pi) ** 0.5
    sig = torch.sigmoid(g)
    return (g * sig, sig * (1.0 + g * (1.0 - sig))) if act == "silu" else (sig, sig * (1.0 - sig))


def _plain_ffn(s, case):
    x, w, b, wo, bo = (None if t is None else t.detach().float() for t in s["leaves"])
    F = case["F"]
    z = x @ w.t() if b is None else x @ w.t() + b
    a, slope = _act(z[:, :F], case["act"])
    u = z[:, F:]
    h = a * u
    y = h @ wo.t() if bo is None else h @ wo.t() + bo
    t = TYPES[case["dtype"]]
    if not case["train"]:
        return [y.to(t)]
    d = s["d"].float()
    dh = d @ wo
    dz = torch.cat((dh * u * slope, dh * a), 1)
    grads = [dz @ w, dz.t() @ x] + ([] if b is None else [dz.sum(0)]) + [d.t() @ h] + ([] if bo is None else [d.sum(0)])
    return [y.to(t)] + [g.to(t) for g in grads]


def _plain_clip(s, case):
    grads, p = s["grads"], case["p"]
    if p == 2.0:
        norm = torch.stack([t.double().square().sum() for t in grads]).sum().sqrt()
    elif p == 1.0:
        norm = torch.stack([t.double().abs().sum() for t in grads]).sum()
    else:
        norm = torch.stack([t.abs().amax().double() for t in grads]).amax()
    norm = norm.float()
    factor = torch.clamp_max(s["max_norm"] / (norm + 1e-6), 1.0)
    for t, o in zip(grads, grads if case["inplace"] else s["out"]):
        o.copy_(t.float() * factor)
    return [norm, s["flat"]]


# ---------------------------------------------------------------------------------------------------- the definition, in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("qk", "qkv"):
        return _exact_qk(s, case)
    if case["kind"] == "ffn":
        return _exact_ffn(s, case)
    return _exact_clip(s, case)


def _exact_qk(s, case):
    """Queries and keys as complex numbers turned by exp(i angle); gradients by the adjoint of each step."""
    Z, H, N, d = case["Z"], case["H"], case["N"], case["d"]
    x = s["qkv"].detach().double()                                              # [Z,N,3,H,d]
    valid = torch.ones(Z, N, dtype=torch.float64, device=DEV) if s["mask"] is None else (~s["mask"]).double()
    valid = valid.view(Z, N, 1, 1, 1)
    pos = torch.arange(N, device=DEV).expand(Z, N) if s["positions"] is None else s["positions"]
    freq = torch.tensor([BASE ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV).expand(Z, N, 1, 1, d // 2), pos.double().view(Z, N, 1, 1, 1) * freq)

    def as_complex(t):
        t = t.unflatten(-1, (d // 2, 2)) if case["interleaved"] else t.unflatten(-1, (2, d // 2)).transpose(-1, -2)
        return torch.view_as_complex(t.contiguous())

    def as_real(t):
        t = torch.view_as_real(t)
        return t.flatten(-2) if case["interleaved"] else t.transpose(-1, -2).flatten(-2)
    w = torch.stack([t.detach().double().expand(H, d) for t in (s["qw"], s["kw"])])
    x2 = x[:, :, :2] * valid
    scale = (x2.pow(2).sum(-1, keepdim=True) / d + EPS).pow(-0.5)
    y = as_real(as_complex(x2 * scale * w) * turn) * valid
    if case["kind"] == "qkv":
        outs = [torch.cat((y, x[:, :, 2:] * valid), 2)]
    else:
        outs = [y[:, :, i].permute(0, 2, 1, 3) for i in range(2)]
    if not case["train"]:
        return outs
    if case["kind"] == "qkv":
        dall = s["d"][0].double()
        dy, dv = dall[:, :, :2] * valid, dall[:, :, 2:] * valid
    else:
        dy, dv = torch.stack([t.permute(0, 2, 1, 3).double() for t in s["d"]], 2) * valid, None
    back = as_real(as_complex(dy) * turn.conj())
    dw = (back * x2 * scale).sum((0, 1))                                        # [2,H,d]
    m = back * w
    dx = scale * m - scale ** 3 * x2 * ((m * x2).sum(-1, keepdim=True) / d)
    dws = [dw[i] if case["per_head"] else dw[i].sum(0) for i in range(2)]
    if case["kind"] == "qkv":
        return outs + [torch.cat((dx, dv), 2)] + dws
    return outs + [dx[:, :, i].permute(0, 2, 1, 3) for i in range(2)] + dws


def _exact_ffn(s, case):
    """By autograd in float64 over the definition."""
    leaves = [None if t is None else t.detach().double().requires_grad_(case["train"]) for t in s["leaves"]]
    x, w, b, wo, bo = leaves
    nn = torch.nn.functional
    gate, up = nn.linear(x, w, b).chunk(2, -1)
    act = {"silu": nn.silu, "gelu": nn.gelu, "relu": nn.relu, "sigmoid": torch.sigmoid}[case["act"]]
    y = nn.linear(act(gate) * up, wo, bo)
    if not case["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, [t for t in leaves if t is not None], s["d"].double())]


def _exact_clip(s, case):
    """A running sum over pieces of the gradients, in float64."""
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for t in s["grads"]:
        for piece in t.split(1 << 25):
            size = piece.double().abs()
            total = torch.maximum(total, size.max()) if math.isinf(case["p"]) else total + (size ** case["p"]).sum()
    norm = total if math.isinf(case["p"]) else total ** (1.0 / case["p"])
    factor = min(1.0, s["max_norm"] / (float(norm) + 1e-6))
    return [norm, torch.cat([t.double() * factor for t in s["grads"]])]


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["kind"] in ("qk", "qkv"):
        tokens, parts = int(_lengths(case).sum()), 3 if case["kind"] == "qkv" else 2
        all_tokens = case["Z"] * case["N"]
        row = parts * case["H"] * case["d"]
        # padded rows: zeros to write, nothing to read
        bytes_ = row * (tokens * size[case["dtype"]] + all_tokens * size[case["out"]])
        flops = 2 * case["H"] * case["d"] * tokens * 7
        if case["train"]:
            bytes_ += row * (tokens * size[case["out"]] + all_tokens * size[case["dtype"]])
            flops *= 3
        return {"bytes": bytes_, "flops": flops}
    if case["kind"] == "ffn":
        M, D, F, b = case["M"], case["D"], case["F"], size[case["dtype"]]
        weights = 3 * D * F + (2 * F + D if case["bias"] else 0)
        return {"bytes": b * ((4 if case["train"] else 2) * M * D + (2 if case["train"] else 1) * weights), "flops": (3 if case["train"] else 1) * 6 * M * D * F}
    n = sum(_sizes(case))
    # within the bound in place there is nothing to write
    return {"bytes": n * (size[case["dtype"]] + (0 if case["inplace"] else size[case["out"]])), "flops": 3 * n}
