"""GPU tests of the norm and rotation, the gated block and the clipping used at once: captured graphs replayed in turn, streams side by side, backwards of one graph twice.
Each result is compared with the same calls one after the other, to the bit."""
import pytest
import torch

import proteusai_amd as pa

pytestmark = pytest.mark.gpu


class Step:
    """A step through all three: rotated queries and keys into a gated block, gradients of its leaves, clipped into tensors of fp32."""

    def __init__(self, gpu, N, H, d, hidden, dtype, seed):
        g = torch.Generator().manual_seed(seed)
        D = H * d
        self.shape, self.gen = (2, N, 3, H, d), g

        def t(*s, scale=1.0):
            return (torch.randn(*s, generator=g) * scale).to(dtype).to(gpu)
        self.qkv, self.w, self.wo = t(*self.shape), t(2 * hidden, D, scale=D ** -0.5), t(D, hidden, scale=hidden ** -0.5)
        self.b, self.bo, self.qw, self.kw, self.d = t(2 * hidden), t(D), t(d), t(H, d)[0].clone(), t(2, N, D)
        self.mask = torch.zeros(2, N, dtype=torch.bool, device=gpu)
        self.mask[1, N // 2:] = True
        self.positions = torch.randint(-5000, 5000, (2, N), generator=g).to(gpu)
        self.leaves = [v.requires_grad_() for v in (self.qkv, self.qw, self.kw, self.w, self.b, self.wo, self.bo)]

    def fill(self):
        with torch.no_grad():
            self.qkv.copy_(torch.randn(self.shape, generator=self.gen))
            self.d.copy_(torch.randn(self.d.shape, generator=self.gen))

    def forward(self):
        r = pa.qk_norm_rotate_qkv(self.qkv, self.qw, self.kw, self.positions, mask=self.mask)
        x = (r[:, :, 0] + r[:, :, 1] * r[:, :, 2]).flatten(-2)
        return pa.gated_mlp(x, self.w, self.b, self.wo, self.bo)

    def run(self):
        y = self.forward()
        grads = torch.autograd.grad(y, self.leaves, self.d)
        norm, out = pa.clip_grad_norm(grads, 0.5, out=[torch.empty(v.shape, device=v.device) for v in grads])
        return [y.detach(), norm, *grads, *out]


def steps(gpu):
    return [Step(gpu, 700, 8, 64, 1000, torch.bfloat16, 1), Step(gpu, 33, 4, 32, 72, torch.bfloat16, 2), Step(gpu, 520, 8, 64, 1032, torch.float32, 3)]


def same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_graphs_replayed_in_turn(gpu):
    all_ = steps(gpu)
    graphs = []
    for s in all_:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            s.run()
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = s.run()
        graphs.append((graph, held))
    for i in range(4):
        for s in all_:
            s.fill()
        for graph, _ in graphs if i % 2 else graphs[::-1]:
            graph.replay()
        torch.cuda.synchronize()
        for s, (_, held) in zip(all_, graphs):
            assert same(held, s.run()), i


def test_streams_side_by_side(gpu):
    all_ = steps(gpu)
    want = [s.run() for s in all_]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in all_]
    for _ in range(3):
        got = []
        for s, stream in zip(all_, streams):
            with torch.cuda.stream(stream):
                got.append(s.run())
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want))


def test_backward_twice_and_in_parts(gpu):
    for s in steps(gpu):
        y = s.forward()
        whole = torch.autograd.grad(y, s.leaves, s.d, retain_graph=True)
        assert same(whole, torch.autograd.grad(y, s.leaves, s.d, retain_graph=True))
        for i, leaf in enumerate(s.leaves):
            part, = torch.autograd.grad(y, leaf, s.d, retain_graph=True)
            assert torch.equal(part, whole[i]), i


def test_checkpointed_forward(gpu):
    from torch.utils.checkpoint import checkpoint
    for s in steps(gpu):
        want = torch.autograd.grad(s.forward(), s.leaves, s.d)
        got = torch.autograd.grad(checkpoint(s.forward, use_reentrant=False), s.leaves, s.d)
        assert same(got, want)


def test_clipped_parameters_shared_by_two_modules(gpu):
    """A parameter that two modules share is listed once or refused: scaling its gradient twice is no clipping."""
    p = torch.nn.Parameter(torch.randn(1000, device=gpu))
    p.grad = torch.randn(1000, device=gpu)
    before = p.grad.clone()
    with pytest.raises(ValueError, match="share memory"):
        pa.clip_grad_norm_([p, p], 0.1)
    assert torch.equal(p.grad, before)
    norm = pa.clip_grad_norm_([p], 0.1)
    assert abs(float(norm) - float(before.double().norm())) <= 2.0 ** -23 * float(norm)
    assert float(pa.grad_norm([before, before])) == pytest.approx(float(before.double().norm()) * 2 ** 0.5, rel=2.0 ** -22)
