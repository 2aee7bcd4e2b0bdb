"""What the cross entropy from features refuses, before anything is launched (no GPU needed)."""
import ctypes

import pytest
import torch

import proteusai_amd as pa
from proteusai_amd import _lib

P = 0x10000                     # an aligned address that nothing reads


def tensors(M=6, D=16, V=10, dtype=torch.float32):
    return torch.zeros(M, D, dtype=dtype), torch.zeros(V, D, dtype=dtype), torch.zeros(M, dtype=torch.int64), torch.zeros(V, dtype=dtype)


def test_no_cpu_path():
    with pytest.raises(_lib.ProteusError, match="GPU"):
        pa.linear_cross_entropy(*tensors())


@pytest.mark.parametrize("kw", [dict(reduction="batchmean"), dict(label_smoothing=-0.1), dict(label_smoothing=1.5), dict(label_smoothing=float("nan"))])
def test_bad_arguments(kw):
    with pytest.raises(ValueError):
        pa.linear_cross_entropy(*tensors(), **kw)


def test_bad_shapes_and_types():
    x, w, t, b = tensors()
    for args in ((x, w[:, :8], t, b), (x, w[0], t, b), (x, w, t[:5], b), (x, w, t[None], b), (x, w, t, b[:5]), (x, w, t, w), (x[0, 0], w, t, b)):
        with pytest.raises(AssertionError):
            pa.linear_cross_entropy(*args)
    with pytest.raises(NotImplementedError, match="int64"):
        pa.linear_cross_entropy(x, w, t.int(), b)
    with pytest.raises(NotImplementedError, match="int64"):
        pa.linear_cross_entropy(x, w, t.float(), b)


def args(**kw):
    a = _lib.CeArgs(x=P, weight=P, bias=P, target=P, ignore_index=-100, rows=100, d=64, vocab=300, dtype=_lib.DTYPE_BF16, reduction=_lib.CE_MEAN, label_smoothing=0.0)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,code", [
    ({}, 0), (dict(rows=0), -2), (dict(rows=-1), -2), (dict(rows=(1 << 24) + 1), -2), (dict(vocab=0), -2), (dict(vocab=(1 << 24) + 1), -2), (dict(d=0), -2), (dict(d=60), -2), (dict(d=60, dtype=_lib.DTYPE_F32), 0),
    (dict(d=62, dtype=_lib.DTYPE_F32), -2), (dict(d=(1 << 16) + 8), -2), (dict(dtype=3), -9), (dict(dtype=-1), -9), (dict(reduction=3), -7), (dict(label_smoothing=-0.5), -2), (dict(label_smoothing=2.0), -2),
    (dict(label_smoothing=float("nan")), -2), (dict(bias=None), 0), (dict(dtype=_lib.DTYPE_F16), 0)])
def test_sizes(kw, code):
    lib = _lib.load()
    assert lib.proteus_linear_ce_check(args(**kw)) == code
    sizes = lib.proteus_linear_ce_fwd_bytes(args(**kw)), lib.proteus_linear_ce_bwd_bytes(args(**kw))
    assert all(n > 0 for n in sizes) if code == 0 else sizes == (0, 0)
    if code:
        assert lib.proteus_linear_ce_fwd(args(**kw), P, P, 1 << 40, P, 1 << 40, None) == code
        assert lib.proteus_linear_ce_bwd(args(**kw), P, P, 1 << 40, P, P, P, P, 1 << 40, None) == code


def test_pointers_and_workspaces():
    lib = _lib.load()
    f, b, k = lib.proteus_linear_ce_fwd_bytes(args()), lib.proteus_linear_ce_bwd_bytes(args()), lib.proteus_linear_ce_kept_bytes(args())
    assert k == 1600 and lib.proteus_linear_ce_kept_bytes(args(rows=0)) == lib.proteus_linear_ce_kept_bytes(args(d=60)) == 0 and lib.proteus_linear_ce_check(None) == -1
    assert lib.proteus_linear_ce_kept_bytes(args(vocab=20)) == 256 + 100 * 20 * 4

    def fwd(loss=P, kept=P, kept_bytes=k, ws=P, ws_bytes=f, **kw):
        return lib.proteus_linear_ce_fwd(args(**kw), loss, kept, kept_bytes, ws, ws_bytes, None)

    def bwd(dloss=P, kept=P, kept_bytes=k, dx=P, dw=P, db=P, ws=P, ws_bytes=b, **kw):
        return lib.proteus_linear_ce_bwd(args(**kw), dloss, kept, kept_bytes, dx, dw, db, ws, ws_bytes, None)
    for call in (fwd, bwd):
        for name in ("x", "weight", "target"):
            assert call(**{name: None}) == -1
        for name, by in (("x", 8), ("weight", 8), ("bias", 2), ("target", 4)):
            assert call(**{name: P + by}) == -5
        assert call(ws=None) == -1 and call(ws=P + 16) == -5 and call(kept=P + 8) == -5 and call(kept_bytes=k - 1) == -8
    assert fwd(loss=None) == -1 and fwd(loss=P + 2) == -5 and fwd(ws_bytes=f - 1) == -8
    assert bwd(dloss=None) == -1 and bwd(kept=None) == -1 and bwd(dx=P + 8) == -5 and bwd(dw=P + 4) == -5 and bwd(db=P + 2) == -5 and bwd(ws_bytes=b - 1) == -8
    assert bwd(bias=None) == -1                                            # a bias's gradient without a bias
    assert bwd(dx=None, dw=None, db=None) == 0                              # nothing asked for: nothing launched


def test_workspaces_keep_to_what_they_document():
    """The backward's grows with the tokens, and with the vocabulary only by sums and copies, past 1 GB of gradients of logits."""
    lib = _lib.load()

    def ws(rows, vocab, d=64, **kw):
        return lib.proteus_linear_ce_bwd_bytes(args(rows=rows, vocab=vocab, d=d, bias=None, **kw))
    for rows, vocab in ((16384, 65536), (16384, 1 << 20), (1 << 20, 1 << 20), (1 << 20, 20), (1, 1 << 24)):
        most = max(1 << 30, rows * 2112 * 2) + rows * (2 * 64 + 4 + 16 + 4) + vocab * 4                # gradients of logits (rows of whole 128 bytes), features and numbers of tokens, a bias
        sums = 32 * 4 * 64 * max(rows if rows < 65536 else 0, vocab if vocab < 65536 else 0) + 4 * 64 * rows
        assert ws(rows, vocab) < most + sums + (1 << 20), (rows, vocab)
    assert lib.proteus_linear_ce_fwd_bytes(args(rows=16384, vocab=65536)) < 16384 * 65536 // 8 + (16384 * 64 * 2 + 16384 * 16 + 65536 * 4 + (1 << 20))


@pytest.mark.parametrize("ignore", [-100, 0, 2 ** 40])
@pytest.mark.parametrize("V", [10, 1])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_the_torch_expression_keeps_to_the_vocabulary_and_the_tokens_that_count(ignore, V, smoothing):
    """It stands in for the kernels under autocast and the like: NaN for a target that is no word (on a GPU torch would read outside of the logits), nothing of a token that is left out."""
    from proteusai_amd.linear_ce import _expression
    g = torch.Generator().manual_seed(1)
    x, w, b = torch.randn(6, 16, generator=g), torch.randn(V, 16, generator=g), torch.randn(V, generator=g)
    target = torch.tensor([V - 1, ignore, V - 1, ignore, V - 1, V - 1])
    plain = torch.nn.functional.cross_entropy(torch.nn.functional.linear(x, w, b), target, ignore_index=ignore, label_smoothing=smoothing, reduction="none")
    dirty = x.clone()
    dirty[1], dirty[3] = float("nan"), float("inf")
    leaves = [t.clone().requires_grad_() for t in (dirty, w, b)]
    clean = [t.clone().requires_grad_() for t in (x, w, b)]
    got = _expression(leaves[0], leaves[1], leaves[2], target, ignore, smoothing, "none")
    assert torch.equal(got.detach(), plain)
    want = torch.autograd.grad(_expression(clean[0], clean[1], clean[2], target, ignore, smoothing, "none").sum(), clean)
    for p, q in zip(torch.autograd.grad(got.sum(), leaves), want):
        assert torch.equal(p, q) and bool(torch.isfinite(p).all())
    for bad in (V, -1, 2 ** 50, -2 ** 62):
        t = target.clone()
        t[2] = bad
        leaf = x.clone().requires_grad_()
        loss = _expression(leaf, w, b, t, ignore, smoothing, "none")
        dx, = torch.autograd.grad(loss.sum(), leaf)
        rest = torch.arange(6) != 2
        assert loss[2].isnan() and torch.equal(loss[rest].detach(), plain[rest]) and bool(dx[2].isnan().all()) and bool(torch.isfinite(dx[rest]).all())
        for reduction in ("mean", "sum"):
            assert _expression(x, w, b, t, ignore, smoothing, reduction).isnan()


@pytest.mark.parametrize("rows,vocab,d", [(1 << 20, 1 << 17, 8), (1 << 20, 1 << 17, 64), (1 << 22, 1 << 17, 64), (1 << 24, 1 << 14, 16)])
def test_the_largest_launches_keep_to_what_a_grid_may_have(rows, vocab, d):
    """2^32 - 1 threads.  Beyond that only tiles of 256 x 256, whose workgroups take several, will do: they leave 8 bytes for each 128 logits (others for each 64)."""
    n = _lib.load().proteus_linear_ce_fwd_bytes(args(rows=rows, vocab=vocab, d=d, bias=None))
    assert n <= rows * vocab // 128 * 8 + rows * (2 * d + 16) + vocab * 4 + (1 << 20)
