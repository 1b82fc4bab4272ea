"""Newton-Schulz orthogonalisation and the Muon optimiser against the iteration in 64 bits.

The bound of an error, in Frobenius norms: a product of factors P, Q that are held to 22 bits and summed in 32 over K is
off by (2^-21 + 2^-23 (3 K / 16 + 16)) | |P| |Q| | (three matrix instructions for 16 of K, and the sum inside one). It
passes into X by |X|_2 and the coefficients, and grows a step by at most the largest derivative of
s -> a s + b s^3 + c s^5. The low half of a number is subnormal below 2^-14, where its steps are 2^-24: with scales of 2^13
or more (entries near 1 and below) each entry held is off by another 2^-38 at most. An output of fewer bits adds half a
step of its type.
"""
import copy
import math

import pytest
import torch

from ding.torch_utils import orthogonalize, Muon, Adam

DEFAULT = (3.4445, -4.7750, 2.0315)
gpu = pytest.mark.gpu


def oracle(matrix, steps=5, coefficients=DEFAULT, eps=1e-7):
    """The iteration on one matrix in 64 bits, and how far (Frobenius) 22-bit factors may be from it."""
    a, b, c = coefficients
    x = matrix.detach().cpu().double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + eps)
    side, entries = float(x.shape[0]), math.sqrt(x.numel())
    err = 2.0 ** -22 * x.norm() + 2.0 ** -38 * entries

    def local(p, q):
        return (2.0 ** -21 + 2.0 ** -23 * (3 * p.shape[1] / 16 + 16)) * (p.abs() @ q.abs()).norm()

    for _ in range(steps):
        g = x @ x.t()
        bg = b * g + c * (g @ g)
        top = torch.linalg.matrix_norm(x, 2)
        s = torch.linspace(0, 1, 1001).double() * top * 1.001
        slope = (a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max()
        off_g = local(x, x.t()) + 2.0 ** -22 * g.norm() + 2.0 ** -38 * side
        off_b = abs(b) * off_g + abs(c) * (2 * top ** 2 * off_g + local(g, g)) + 2.0 ** -22 * bg.norm() + 2.0 ** -38 * side
        err = slope * err + off_b * top + local(bg, x) + 2.0 ** -21 * (a * x.norm())
        x = a * x + bg @ x
        err = err + 2.0 ** -22 * x.norm() + 2.0 ** -38 * entries
    return (x.t() if tall else x), err


def check(matrix, steps=5, coefficients=DEFAULT, eps=1e-7):
    got = orthogonalize(matrix, steps, coefficients, eps)
    assert got.shape == matrix.shape and got.dtype == matrix.dtype and got.is_contiguous()
    half = torch.finfo(got.dtype).eps / 2
    floor = 2.0 ** -25 if got.dtype == torch.float16 else 0.0
    many = matrix.reshape(-1, *matrix.shape[-2:])
    for one, other in zip(many, got.reshape(many.shape)):
        want, err = oracle(one, steps, coefficients, eps)
        off = (other.cpu().double() - want).norm()
        allowed = err + half * (want.norm() + err) + floor * math.sqrt(want.numel())
        assert off <= allowed, f"off by {off:.3g} of {want.norm():.3g}, allowed {allowed:.3g}"
    return got


def case(*shape, dtype=torch.float32, device='cpu', scale=1e-3, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rank = max(1, min(shape[-2:]) // 4)
    strong = torch.randn(*shape[:-1], rank, generator=gen) @ torch.randn(*shape[:-2], rank, shape[-1], generator=gen)
    return ((strong / math.sqrt(rank) + 0.1 * torch.randn(*shape, generator=gen)) * scale).to(dtype).to(device)


# --------------------------------------------------------------------------------------------------------------- CPU


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize('shape', [(1, 1), (1, 9), (9, 1), (12, 12), (10, 33), (33, 10), (2, 3, 8, 5)])
def test_cpu_lane(shape, dtype):
    check(case(*shape, dtype=dtype))


def test_cpu_singular_values():
    x = torch.randn(40, 60, generator=torch.Generator().manual_seed(0))
    s = torch.linalg.svdvals(orthogonalize(x))
    assert s.min() > 0.6 and s.max() < 1.3
    s = torch.linalg.svdvals(orthogonalize(x, steps=12, coefficients=(1.875, -1.25, 0.375)))
    assert torch.allclose(s, torch.ones_like(s), atol=1e-5)
    assert torch.equal(orthogonalize(torch.zeros(3, 4)), torch.zeros(3, 4))
    assert orthogonalize(torch.zeros(0, 4)).shape == (0, 4)


def test_refusals():
    x = case(4, 5)
    for args in (dict(matrix=x[0]), dict(matrix=x.long()), dict(steps=0), dict(eps=0.0), dict(eps=float('nan')),
                 dict(coefficients=(1., 2.)), dict(coefficients=(float('inf'), 0., 0.)),
                 dict(coefficients=(3., 3., 3.))):
        with pytest.raises(ValueError):
            orthogonalize(**{'matrix': x, **args})


def _net(device='cpu', dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    net = torch.nn.Sequential(
        torch.nn.Embedding(11, 12), torch.nn.Flatten(), torch.nn.Linear(36, 24), torch.nn.LayerNorm(24),
        torch.nn.Linear(24, 24), torch.nn.ReLU(), torch.nn.Linear(24, 24), torch.nn.ReLU(), torch.nn.Linear(24, 5)
    )
    return net.to(device=device, dtype=dtype)


def _grads(net, seed):
    gen = torch.Generator().manual_seed(seed)
    for p in net.parameters():
        p.grad = torch.randn(p.shape, generator=gen).to(device=p.device, dtype=p.dtype)


def _want_step(p, grads, group):
    """The optimiser's definition for one parameter and its gradients so far, in 64 bits."""
    w = p.double().cpu()
    buf = m = v = torch.zeros_like(w)
    for n, g in enumerate(grads, 1):
        g = g.double().cpu()
        w = w * (1 - group['lr'] * group['weight_decay'])
        if w.dim() >= 2 and not group['use_adam']:
            buf = group['momentum'] * buf + g
            u = g + group['momentum'] * buf if group['nesterov'] else buf
            flat = u.reshape(u.shape[0], -1)
            w = w - group['lr'] * 0.2 * math.sqrt(max(flat.shape)) * oracle(flat)[0].reshape(w.shape)
        else:
            b1, b2 = group['betas']
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
            w = w - group['lr'] * (m / (1 - b1 ** n)) / ((v / (1 - b2 ** n)).sqrt() + group['eps'])
    return w


def _check_optimizer(device, dtype, tol):
    net = _net(device, dtype)
    start = [p.detach().clone() for p in net.parameters()]
    groups = [
        dict(params=list(net[0].parameters()) + list(net[-1].parameters()), use_adam=True),
        dict(params=[p for layer in net[1:-1] for p in layer.parameters()], nesterov=True),
    ]
    opt = Muon(groups, lr=0.01, weight_decay=0.1)
    seen = [[] for _ in start]
    for step in range(4):
        _grads(net, step)
        for s, p in zip(seen, net.parameters()):
            s.append(p.grad.clone())
        opt.step()
        if step == 1:  # states go through a checkpoint as they are
            state = copy.deepcopy(opt.state_dict())
            opt = Muon(groups, lr=0.01, weight_decay=0.1)
            opt.load_state_dict(state)
            assert all(v.dtype == torch.float32 for s in opt.state.values() for v in s.values())
    at = {p: g for g in opt.param_groups for p in g['params']}
    for p, s, grads in zip(net.parameters(), start, seen):
        want = _want_step(s, grads, at[p])
        assert (p.detach().cpu().double() - want).abs().max() <= tol * max(1.0, want.abs().max())


def test_optimizer_cpu():
    # four steps of 0.01 * 0.2 sqrt(36) times updates that are right to 1e-5, and 32-bit roundings of the weights
    _check_optimizer('cpu', torch.float32, 4 * 0.012 * 1e-4 + 8 * 2.0 ** -24)


def _check_half_weights(device):
    """Weights of half precision whose gradients are near either end of its range: their momentum passes it."""
    for size in (60000.0, 2.0 ** -22):
        torch.manual_seed(3)
        net = torch.nn.Conv2d(6, 20, 3, bias=False).to(device=device, dtype=torch.float16)
        net = net.to(memory_format=torch.channels_last)
        p, opt, grads = net.weight, Muon(net.parameters(), lr=0.01), []
        start = p.detach().clone()
        for step in range(4):
            sign = torch.randint(0, 2, p.shape, generator=torch.Generator().manual_seed(step // 3)) * 2 - 1
            p.grad = (sign * size).to(device=device, dtype=torch.float16)
            grads.append(p.grad.clone())
            opt.step()
        want = _want_step(start, grads, opt.param_groups[0])
        # a rounding of the weight a step, and steps of 0.01 * 0.2 sqrt(54) times updates that are right to 1e-4
        assert (p.detach().cpu().double() - want).abs().max() <= 4 * 2.0 ** -11 * want.abs().max() + 4 * 0.015 * 1e-4


def test_optimizer_half_weights_cpu():
    _check_half_weights('cpu')


def test_optimizer_options():
    net = _net()
    for clip in (dict(grad_clip_type='clip_norm', clip_value=0.5), dict(grad_clip_type='clip_value', clip_value=0.1),
                 dict(grad_clip_type='ignore_norm', ignore_value=1e-3), dict(nesterov=False)):
        opt = Muon(net.parameters(), lr=0.01, **clip)
        before = [p.detach().clone() for p in net.parameters()]
        _grads(net, 0)
        opt.step()
        moved = any(not torch.equal(a, b) for a, b in zip(before, net.parameters()))
        assert moved == (clip.get('grad_clip_type') != 'ignore_norm')
        assert opt.get_grad() >= 0
    for bad in (dict(momentum=1.0), dict(lr=-1.0), dict(weight_decay=-1.0)):
        with pytest.raises(ValueError):
            Muon(net.parameters(), **bad)
    with pytest.raises(KeyError):
        Muon(net.parameters(), grad_clip_type='clip')
    net[0].weight.grad = None  # a parameter that took no part
    before = net[0].weight.detach().clone()
    Muon(net.parameters(), lr=0.01, weight_decay=0.1).step()
    assert torch.equal(before, net[0].weight)


# --------------------------------------------------------------------------------------------------------------- GPU


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('shape', [
    (1, 1), (1, 9), (9, 1), (5, 5), (31, 33), (64, 64), (65, 130), (128, 128), (129, 127), (200, 1000), (1000, 200),
    (1, 5000), (257, 640), (513, 514), (3, 40, 70), (2, 2, 150, 90), (7, 128, 256), (40, 16, 16)
])
def test_gpu_shapes(shape, dtype):
    check(case(*shape, dtype=dtype, device='cuda', seed=sum(shape)))


@gpu
@pytest.mark.parametrize('steps,coefficients', [(1, DEFAULT), (2, DEFAULT), (7, DEFAULT), (10, (1.875, -1.25, 0.375)),
                                                (8, (1.5, -0.5, 0.0))])
@pytest.mark.parametrize('shape', [(60, 100), (300, 200)])
def test_gpu_steps(shape, steps, coefficients):
    check(case(*shape, device='cuda'), steps, coefficients)
    check(case(*shape, dtype=torch.bfloat16, device='cuda'), steps, coefficients)


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(40, 3000), (130, 8000), (7000, 33), (2, 190, 2500), (1100, 1500)])
def test_gpu_depth_in_parts(shape, dtype):
    check(case(*shape, dtype=dtype, device='cuda'))


@gpu
@pytest.mark.parametrize('shape', [(3, 70, 150), (2, 300, 140)])
def test_gpu_strides(shape):
    b, m, n = shape
    x = case(b, m, n + 6, device='cuda')
    check(x[..., 3:n + 3])
    check(x.transpose(1, 2))
    check(x[:, ::2, ::3])
    check(x.permute(1, 2, 0).contiguous().permute(2, 0, 1))
    check(x[:1].expand(3, m, n + 6))
    check(x[0, :1].expand(m, n + 6))  # rank one


@gpu
@pytest.mark.parametrize('shape', [(40, 60), (200, 300)])
def test_gpu_extreme_values(shape):
    for scale in (1e-30, 1e25, 1e30):
        check(case(*shape, device='cuda', scale=scale), eps=1e-7)
    check(case(*shape, device='cuda', scale=1e-30), eps=1e-38)
    x = torch.stack([case(*shape, device='cuda', seed=s) for s in range(4)])
    x[1] = 0
    x[2, 3, 4] = float('nan')
    got = orthogonalize(x)
    assert torch.equal(got[1], torch.zeros_like(got[1])) and torch.isnan(got[2]).any()
    assert torch.equal(got[0], orthogonalize(x[0])) and torch.equal(got[3], orthogonalize(x[3]))
    x[2, 3, 4] = float('inf')
    assert not torch.isfinite(orthogonalize(x)[2]).all()


@gpu
def test_gpu_refusals():
    with pytest.raises(TypeError):
        orthogonalize(torch.zeros(3, 4, dtype=torch.double, device='cuda'))
    assert orthogonalize(torch.zeros(0, 3, 4, device='cuda')).shape == (0, 3, 4)
    assert orthogonalize(torch.zeros(2, 0, 4, device='cuda')).shape == (2, 0, 4)
    assert not orthogonalize(torch.ones(2, 3, device='cuda', requires_grad=True)).requires_grad


@gpu
def test_gpu_stream_and_graph():
    for shape, dtype in (((2, 60, 100), torch.float32), ((300, 500), torch.bfloat16)):
        x = case(*shape, dtype=dtype, device='cuda')
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = [orthogonalize(x) for _ in range(3)][-1]
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, orthogonalize(x))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = orthogonalize(x)
        for seed in range(3):
            x.copy_(case(*shape, dtype=dtype, device='cuda', seed=seed + 4))
            graph.replay()
            got = kept.clone()
            torch.cuda.synchronize()
            assert torch.equal(got, orthogonalize(x))


@gpu
def test_gpu_optimizer():
    _check_optimizer('cuda', torch.float32, 4 * 0.012 * 1e-4 + 8 * 2.0 ** -24)


@gpu
def test_gpu_optimizer_half_weights():
    _check_half_weights('cuda')


@gpu
def test_gpu_optimizer_graph():
    nets = [_net('cuda') for _ in range(2)]
    opts = [Muon(net.parameters(), lr=0.01, grad_clip_type='clip_norm', clip_value=1.0) for net in nets]
    for net, opt in zip(nets, opts):
        _grads(net, 0)
        opt.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        opts[1].step()
    for seed in range(1, 5):
        gen = torch.Generator().manual_seed(seed)
        for p, q in zip(nets[0].parameters(), nets[1].parameters()):
            g = torch.randn(p.shape, generator=gen).cuda()
            p.grad.copy_(g)
            q.grad.copy_(g)
        opts[0].step()
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(nets[0].parameters(), nets[1].parameters()):
            assert torch.allclose(p, q, atol=1e-6)


@gpu
def test_gpu_optimizer_trains():
    for cls in (Muon, Adam):
        net = _net('cuda')
        opt = cls(net.parameters(), lr=3e-3)
        for step in range(5):
            tokens = torch.randint(0, 11, (64, 3), device='cuda')
            loss = torch.nn.functional.cross_entropy(net(tokens), tokens.sum(-1) % 5)
            opt.zero_grad()
            loss.backward()
            opt.step()
        assert all(torch.isfinite(p).all() for p in net.parameters())
