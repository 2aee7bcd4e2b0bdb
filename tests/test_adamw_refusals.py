"""What AdamW's step and the optimizer refuse, before anything is launched (no GPU needed)."""
import copy
import ctypes
import pickle

import pytest
import torch

import proteusai_amd as pa
from proteusai_amd import _lib


def lists(n=8, count=2, dtype=torch.float32, grad=torch.float32):
    return [torch.zeros(n, dtype=dtype) for _ in range(count)], [torch.zeros(n, dtype=grad) for _ in range(count)], [torch.zeros(n) for _ in range(count)], [torch.zeros(n) for _ in range(count)]


def test_no_cpu_path():
    with pytest.raises(_lib.ProteusError, match="GPU"):
        pa.adamw_(*lists(), 1)
    p, g, _, _ = lists()
    with pytest.raises(_lib.ProteusError, match="GPU"):
        pa.adamw8_(p, g, [pa.adamw8_state(x) for x in p], 1)
    x = torch.nn.Parameter(torch.zeros(3))
    x.grad = torch.zeros(3)
    with pytest.raises(_lib.ProteusError, match="GPU"):
        pa.AdamW([x]).step()


@pytest.mark.parametrize("kw,error", [(dict(lr=-1e-3), ValueError), (dict(lr=float("nan")), ValueError), (dict(betas=(1.0, 0.9)), ValueError), (dict(betas=(0.9, -0.1)), ValueError), (dict(eps=-1.0), ValueError),
                                      (dict(weight_decay=-0.1), ValueError), (dict(max_norm=1.0), ValueError), (dict(norm=torch.zeros(())), ValueError), (dict(norm=torch.zeros(()), max_norm=-1.0), ValueError),
                                      (dict(masters=[None]), AssertionError)])
def test_bad_arguments(kw, error):
    with pytest.raises(error):
        pa.adamw_(*lists(), 1, **kw)
    p, g, _, _ = lists()
    with pytest.raises(error):
        pa.adamw8_(p, g, [pa.adamw8_state(x) for x in p], 1, **kw)


def test_bad_steps_and_lists():
    for step in (0, -3, 2 ** 63):
        with pytest.raises(ValueError, match="step"):
            pa.adamw_(*lists(), step)
    p, g, m, v = lists()
    with pytest.raises(AssertionError):
        pa.adamw_(p, g[:1], m, v, 1)
    with pytest.raises(AssertionError):
        pa.adamw_(p, g, m, v[:1], 1)
    with pytest.raises(NotImplementedError):
        pa.adamw_([x.to_sparse() for x in p], g, m, v, 1)
    pa.adamw_([], [], [], [], 1)                                            # nothing to do


@pytest.mark.parametrize("kw", [dict(bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(max_norm=-1.0)])
def test_optimizer_arguments(kw):
    with pytest.raises(ValueError):
        pa.AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_no_captured_step_whose_number_replays_would_not_count(monkeypatch):
    """Refused before anything happens, also where the parameters have stepped before; with capturable=True only their first step is."""
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    x = torch.nn.Parameter(torch.ones(3))
    x.grad = torch.ones(3)
    for bits in (32, 8):
        opt = pa.AdamW([x], bits=bits)
        opt.state[x].update(step=4, exp_avg=torch.zeros(3), exp_avg_sq=torch.zeros(3), moments=pa.adamw8_state(x))
        with pytest.raises(RuntimeError, match="capturable=True"):
            opt.step(lambda: pytest.fail("the closure was called"))
        assert opt.state[x]["step"] == 4 and bool((x == 1).all()) and not opt.state[x]["exp_avg"].any() and not opt.state[x]["moments"].any()


@pytest.mark.parametrize("code", [1, 98, 719])
def test_a_launch_that_fails_raises_and_is_not_repeated(monkeypatch, code):
    """What went out before it has been applied: the step must not be taken again by the other path."""
    calls = []

    class Ops:
        def adamw(self, *args):
            calls.append(args)
            return code
    monkeypatch.setattr(_lib, "ops", Ops)
    monkeypatch.setattr(pa.adamw, "_general", lambda *args: pytest.fail("the step was taken again"))
    with pytest.raises(_lib.ProteusError):
        pa.adamw_(*lists(), 1)
    p, g, _, _ = lists()
    with pytest.raises(_lib.ProteusError):
        pa.adamw8_(p, g, [pa.adamw8_state(x) for x in p], 1)
    assert len(calls) == 2


def test_copies_keep_what_the_optimizer_is():
    x = torch.nn.Parameter(torch.zeros(3))
    kw = dict(bits=8, master_weights=True, max_norm=2.0, capturable=True, seed=4)
    opt = pa.AdamW([x], lr=3e-4, **kw)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert type(other) is pa.AdamW and {k: getattr(other, k) for k in kw} == kw and other.norm is None and other.param_groups[0]["lr"] == 3e-4


def test_a_loaded_state_goes_into_the_tensors_there_are():
    """Those that a captured step writes, and the rate that a schedule fills; shared by groups only where they are to have the same."""
    def optimizer(rate, **kw):
        x = [torch.nn.Parameter(torch.ones(2, 3).t()), torch.nn.Parameter(torch.ones(5, dtype=torch.bfloat16))]
        return pa.AdamW([{"params": x[:1]}, {"params": x[1:], **kw}], lr=rate, capturable=True, master_weights=True)

    def begun(opt, seed):
        g = torch.Generator().manual_seed(seed)
        for group in opt.param_groups:
            group["steps"] = torch.tensor(seed)
            for p in group["params"]:
                opt.state[p].update({k: torch.zeros_like(p, dtype=torch.float32).copy_(torch.randn(p.shape, generator=g)) for k in ("exp_avg", "exp_avg_sq")})
                if p.dtype != torch.float32:
                    opt.state[p]["master"] = torch.randn(p.shape, generator=g)
        return opt

    def tensors(opt):
        return [v for p in opt.state for v in opt.state[p].values()] + [g["steps"] for g in opt.param_groups]
    for saved_rate in (torch.tensor(0.25), torch.tensor(0.25, dtype=torch.float64), 0.25):
        rate = torch.tensor(0.5)
        saved, opt, fresh = begun(optimizer(saved_rate), 7), begun(optimizer(rate), 3), optimizer(rate.clone())
        were, state = tensors(opt), copy.deepcopy(saved.state_dict())
        opt.load_state_dict(state)
        assert len(were) == 7 and all(a is b for a, b in zip(tensors(opt), were)) and opt.param_groups[0]["lr"] is rate and float(rate) == 0.25
        fresh.load_state_dict(state)
        assert all(g["lr"].dtype == torch.float32 and float(g["lr"]) == 0.25 for g in fresh.param_groups)
        for a, b, c in zip(tensors(opt), tensors(fresh), tensors(saved)):
            assert torch.equal(a, b) and torch.equal(a, c.to(a.dtype)) and a.dtype == b.dtype and a.stride() == b.stride() == c.stride()
            assert all(x.data_ptr() != c.data_ptr() for x in (a, b))
        opt.load_state_dict(opt.state_dict())                                 # its own
        assert all(a is b for a, b in zip(tensors(opt), were)) and all(torch.equal(a, c.to(a.dtype)) for a, c in zip(were, tensors(saved)))
    rate = torch.tensor(0.5)
    opt = begun(optimizer(rate), 3)
    opt.load_state_dict(begun(optimizer(0.25, lr=0.125), 7).state_dict())
    assert [float(g["lr"]) for g in opt.param_groups] == [0.25, 0.125] and float(rate) == 0.5
    number = begun(optimizer(0.5), 3)
    number.load_state_dict(begun(optimizer(0.25), 7).state_dict())
    assert [g["lr"] for g in number.param_groups] == [0.25, 0.25]
    number.load_state_dict(begun(optimizer(torch.tensor(0.125)), 7).state_dict())
    assert all(isinstance(g["lr"], torch.Tensor) and float(g["lr"]) == 0.125 for g in number.param_groups)


def test_state_of_8_bits():
    for n, rows in ((0, 0), (1, 1), (512, 1), (513, 2)):
        s = pa.adamw8_state(torch.zeros(n))
        assert s.shape == (rows, 1056) and s.dtype == torch.uint8 and _lib.load().proteus_adamw_state_bytes(n) == s.numel()
    assert _lib.load().proteus_adamw_state_bytes(-1) == 0
    p = torch.zeros(3, 5)
    s = pa.adamw8_state(p)
    s[0, :3] = torch.tensor([0x38, 0xB9, 0x01], dtype=torch.uint8)          # 1, -1.125, the least
    s[0, 512:515] = torch.tensor([0x40, 0x7E, 0x00], dtype=torch.uint8)     # 2, 448, 0
    s[0, 1024], s[0, 1040] = 127 + 3, 127 - 8
    m, v = pa.adamw8_moments(p, s)
    assert m.shape == v.shape == p.shape
    assert m.view(-1)[:3].tolist() == [8.0, -9.0, 2.0 ** -6] and v.view(-1)[:3].tolist() == [2.0 ** -14, 1.75 ** 2, 0.0]
    with pytest.raises(AssertionError):
        pa.adamw8_moments(torch.zeros(513), s)


def test_c_entry():
    lib = _lib.load()
    p = 0x1000

    def args(n=1, **kw):
        a = _lib.AdamwArgs(count=n, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, step=1)
        ptr = ctypes.c_void_p * 1
        a.params, a.grads, a.exp_avgs, a.exp_avg_sqs = ptr(p), ptr(p), ptr(p), ptr(p)
        a.numel, a.param_types, a.grad_types = (ctypes.c_int64 * 1)(8), (ctypes.c_int * 1)(0), (ctypes.c_int * 1)(0)
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.byref(a)

    def one(t, v):
        return (t * 1)(v)
    vp, ci, i64 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64
    check = lib.proteus_adamw_check
    assert check(args()) == 0 and check(args(0)) == 0
    assert check(None) == -1 and check(args(-1)) == -2
    for name in ("params", "grads", "numel", "param_types", "grad_types", "exp_avgs", "exp_avg_sqs"):
        assert check(args(**{name: None})) == -1
    for name in ("params", "grads", "exp_avgs", "exp_avg_sqs"):
        assert check(args(**{name: one(vp, None)})) == -1
        assert check(args(**{name: one(vp, p + 2)})) == -5
    assert check(args(states=one(vp, p))) == -1                              # both kinds of moments
    assert check(args(states=one(vp, p), exp_avgs=None, exp_avg_sqs=None)) == 0
    assert check(args(states=one(vp, p + 8), exp_avgs=None, exp_avg_sqs=None)) == -5
    for kw in (dict(lr=-1.0), dict(beta1=1.0), dict(beta2=-0.5), dict(eps=-1.0), dict(weight_decay=float("nan")), dict(step=0), dict(norm=p, max_norm=-1.0), dict(numel=one(i64, -1)), dict(numel=one(i64, 1 << 40))):
        assert check(args(**kw)) == -2, kw
    assert check(args(step=0, step_gpu=p)) == 0 and check(args(lr=-1.0, lr_gpu=p)) == 0
    for pt, gt, rc in ((0, 1, 0), (0, 2, 0), (1, 1, 0), (1, 0, 0), (1, 2, -9), (2, 1, -9), (3, 0, -9), (0, 7, -9)):
        assert check(args(param_types=one(ci, pt), grad_types=one(ci, gt))) == rc
    assert check(args(masters=one(vp, p))) == -9                              # of an fp32 parameter
    assert check(args(masters=one(vp, p), param_types=one(ci, 1))) == 0 and check(args(masters=one(vp, p + 2), param_types=one(ci, 1))) == -5
    assert lib.proteus_adamw(args(beta1=2.0), None) == -2                     # (the launching entry point looks first)
