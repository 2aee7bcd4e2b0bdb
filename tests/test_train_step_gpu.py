"""GPU tests of the two ends of a training step together and with what lies between: the encoder's loss from its features, clipping and AdamW in one pass, eager and captured."""
import copy

import pytest
import torch
import torch.nn.functional as F

import proteusai_amd as pa
from proteusai_amd import synth

pytestmark = pytest.mark.gpu


def batch(gpu, Z, N, seed=0):
    g = torch.Generator().manual_seed(seed)
    coords = torch.stack([synth.random_walk_chain(N, g) for _ in range(Z)]).to(gpu)
    mask = torch.zeros(Z, N, dtype=torch.bool, device=gpu)
    for i in range(Z):
        mask[i, N - i * (N // (2 * Z)):] = True
    return coords, mask, torch.randint(0, 33, (Z, N), generator=g).to(gpu), torch.randint(0, 20, (Z, N), generator=g).to(gpu)


def network(gpu, dtype=torch.float32, seed=4, **kw):
    torch.manual_seed(seed)
    m = pa.ProteusEncoder(d_model=128, heads=2, layers=2, d_hidden=256, rotary_base=10000.0, gated="silu", **kw).to(gpu)
    for layer in m.layers:
        layer.attn.spread_weights.requires_grad_(False)         # (their gradients are added up by atomics, whose order is not the same on every call)
    for part in (m.layers, m.aa_embedding, m.head):
        part.to(dtype)
    return m, [p for n, p in m.named_parameters() if "beta" not in n and p.requires_grad]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
@pytest.mark.parametrize("smoothing", [0.0, 0.1])
def test_loss_of_the_encoder(gpu, dtype, smoothing):
    """As torch's on the features: the loss to 1e-5 (sums of 128 products in fp32 on either side), the head's gradients to twice half a step of their type and as much for the rounded gradients of the logits."""
    model, params = network(gpu, dtype)
    coords, mask, tokens, target = batch(gpu, 3, 90)
    target[0, :5] = -100
    for reduction in ("mean", "sum", "none"):
        loss = model.loss(coords, tokens, target, mask, label_smoothing=smoothing, reduction=reduction)
        x = model.features(coords, tokens, mask)
        w, b = model.head.weight.detach().float().requires_grad_(), model.head.bias.detach().float().requires_grad_()
        logits = F.linear(x.detach().float(), w, b)
        want = F.cross_entropy(logits.flatten(0, 1), target.masked_fill(mask, -100).flatten(), label_smoothing=smoothing, reduction=reduction)
        assert loss.dtype == torch.float32 and ((loss.detach() - want.view(loss.shape)).abs() <= 1e-5 * (1 + want.detach().abs().max())).all()
        if reduction == "none":
            assert loss.shape == target.shape and bool((loss[mask] == 0).all())
        got = torch.autograd.grad(loss.sum(), [model.head.weight, model.head.bias], retain_graph=True)
        for g, q in zip(got, torch.autograd.grad(want.sum(), [w, b])):
            assert float((g.float() - q).norm()) <= (4 * torch.finfo(dtype).eps + 1e-5) * float(q.norm())
    grads = torch.autograd.grad(model.loss(coords, tokens, target, mask), params, allow_unused=True)
    assert all(g is None or bool(torch.isfinite(g).all()) for g in grads) and sum(g is not None for g in grads) > 20
    handle = model.head.register_forward_hook(lambda m, i, o: None)             # a hook on the head sees its call
    hooked = model.loss(coords, tokens, target, mask, label_smoothing=smoothing)
    handle.remove()
    assert abs(float(hooked.detach()) - float(model.loss(coords, tokens, target, mask, label_smoothing=smoothing).detach())) <= 2 * torch.finfo(dtype).eps * 10


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["float32", "bfloat16"])
def test_captured_training_step(gpu, dtype, bits):
    """Loss, backward, norm, clipping and AdamW, captured and replayed on new tokens, beside the same steps taken eagerly: the same bits."""
    coords, mask, tokens, target = batch(gpu, 2, 100)
    eager, eager_params = network(gpu, dtype)
    model, params = network(gpu, dtype)

    def optimizer(params):
        return pa.AdamW(params, lr=3e-3, bits=bits, master_weights=True, max_norm=0.5, capturable=True)

    def step(model, params, opt, tokens, target):
        loss = model.loss(coords, tokens, target, mask, label_smoothing=0.1)
        for p, g in zip(params, torch.autograd.grad(loss, params, allow_unused=True)):
            p.grad = g
        opt.step()
        return loss.detach()
    oe, oc = optimizer(eager_params), optimizer(params)
    static = tokens.clone(), target.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = float(step(model, params, oc, *static))
    torch.cuda.current_stream().wait_stream(stream)
    assert first == float(step(eager, eager_params, oe, tokens, target))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step(model, params, oc, *static)
    for i in range(4):
        new = torch.randint(0, 33, tokens.shape, device=gpu), torch.randint(0, 20, target.shape, device=gpu)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager, eager_params, oe, *new)
        assert torch.equal(loss, want) and torch.equal(oc.norm, oe.norm), i
        for p, q in zip(params, eager_params):
            assert torch.equal(p, q), i
    assert int(oc.param_groups[0]["steps"]) == 5


@pytest.mark.parametrize("bits", [32, 8])
def test_training_runs_and_resumes(gpu, bits):
    """A dozen steps with a schedule of torch's, saved and resumed in between, give the bits of the steps without."""
    coords, mask, tokens, target = batch(gpu, 2, 80)

    def begin():
        model, params = network(gpu)
        opt = pa.AdamW([{"params": [p for p in params if p.dim() > 1]}, {"params": [p for p in params if p.dim() <= 1], "weight_decay": 0.0}], lr=1e-3, bits=bits, max_norm=1.0)
        return model, opt, torch.optim.lr_scheduler.LambdaLR(opt, lambda t: min(1.0, (t + 1) / 8))

    def go(model, opt, schedule, steps):
        for _ in range(steps):
            opt.zero_grad()
            model.loss(coords, tokens, target, mask).backward()
            opt.step()
            schedule.step()
    a = begin()
    go(*a, 12)
    b = begin()
    go(*b, 5)
    saved = copy.deepcopy([x.state_dict() for x in b])
    c = begin()
    for x, s in zip(c, saved):
        x.load_state_dict(s)
    go(*c, 7)
    for p, q in zip(a[0].parameters(), c[0].parameters()):
        assert torch.equal(p, q)


def test_streams_and_graphs_side_by_side(gpu):
    """Losses and steps of several models on streams of their own, and two captured losses replayed in turn, give the bits of one after the other."""
    def job(i):
        g = torch.Generator(device=gpu).manual_seed(i)
        M, D, V = ((900, 64, 700), (33, 512, 20), (4000, 128, 3000))[i]
        dtype = (torch.bfloat16, torch.float32, torch.float16)[i]
        x, w = torch.randn(M, D, generator=g, device=gpu).to(dtype), (torch.randn(V, D, generator=g, device=gpu) * 0.1).to(dtype)
        t = torch.randint(0, V, (M,), generator=g, device=gpu)
        t[::3] = -100
        state = pa.adamw8_state(w)

        def run():
            weight = w.clone()
            leaves = [x.detach().requires_grad_(), weight.detach().requires_grad_()]
            loss = pa.linear_cross_entropy(leaves[0], leaves[1], t, label_smoothing=0.1)
            dx, dw = torch.autograd.grad(loss, leaves)
            mine = state.clone()
            pa.adamw8_([weight], [dw], [mine], 3, norm=pa.grad_norm([dw]), max_norm=0.1)
            return [loss.detach(), dx, dw, weight, mine]
        return run
    jobs = [job(i) for i in range(3)]
    want = [run() for run in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(3):
        got = []
        for run, stream in zip(jobs, streams):
            with torch.cuda.stream(stream):
                got.append(run())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    graphs = []
    for run in jobs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        graphs.append((graph, held))
    for i in range(4):
        for graph, _ in graphs if i % 2 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for (_, x), y in zip(graphs, want) for a, b in zip(x, y)), i
        jobs[i % 3]()


def test_loss_behind_a_head_that_is_looked_at(gpu):
    """A hook on the head has its call: targets that are no words give NaN, as they do without it."""
    model, _ = network(gpu)
    coords, mask, tokens, target = batch(gpu, 2, 40)
    mask[:] = False
    target[0, 3], target[1, 5], target[1, 7] = 20, -1, -100
    plain = model.loss(coords, tokens, target, mask, reduction="none").detach()
    handle = model.head.register_forward_hook(lambda m, i, o: None)
    hooked = model.loss(coords, tokens, target, mask, reduction="none").detach()
    assert model.loss(coords, tokens, target, mask).isnan()
    handle.remove()
    assert torch.equal(hooked.isnan(), plain.isnan()) and int(plain.isnan().sum()) == 2 and float(hooked[1, 7]) == 0.0
    assert ((hooked - plain).nan_to_num(0.0).abs() <= 1e-5 * (1 + plain.nan_to_num(0.0).abs().max())).all()
