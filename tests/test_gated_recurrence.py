"""The gated linear recurrence: the CPU lane and the HIP kernels against the formulas in 64 bits.

Tolerances count roundings of 2^-24. The gates a = 1 / (1 + e), b = e a with e = exp(-f) are off by (2 |f| + 2) of them
through the exponential, weighted by the other gate, and 4 more. Every step adds at most 4 roundings of each of its
terms, in whatever order a scan joins them; the bound of a state is the same recurrence over these errors, taken over
absolute values. An output of fewer bits adds half a step of its type.
"""
import pytest
import torch

from ding.torch_utils import gated_linear_recurrence, get_lstm, GatedLinearRNN

R = 2.0 ** -24
gpu = pytest.mark.gpu


def oracle(x, f, h0, reset, g=None, g_last=None):
    """name -> (value, how far 32-bit arithmetic may be off), in 64 bits on the CPU."""
    # the kernels multiply G (h - x); autograd on the CPU adds G h a b and -G x a b, each with its own roundings, which
    # are as large as if nothing cancelled
    apart = not x.is_cuda
    x, f = x.detach().cpu().double(), f.detach().cpu().double()
    T = x.shape[0]
    a, b = torch.sigmoid(f), torch.sigmoid(-f)
    near = (2 * f.abs() + 2) * R
    ea, eb = b * near + 4 * R, a * near + 4 * R
    on = torch.ones(T, x.shape[1], 1, dtype=torch.double)
    if reset is not None:
        on = (~reset.cpu()).double().unsqueeze(-1)
    h = torch.zeros_like(x[0]) if h0 is None else h0.detach().cpu().double()
    size, err = h.abs(), torch.zeros_like(h)
    hs, before, sizes, errs, err_before = [], [], [], [], []
    for t in range(T):
        h, size, err = on[t] * h, on[t] * size, on[t] * err
        before.append(h)
        err_before.append(err)
        err = a[t] * err + a[t] * size * (ea[t] + 4 * R) + b[t] * x[t].abs() * (eb[t] + 4 * R)
        h, size = a[t] * h + b[t] * x[t], a[t] * size + b[t] * x[t].abs()
        err = err + 4 * R * size
        hs.append(h)
        errs.append(err)
    out = {'h': (torch.stack(hs), torch.stack(errs)), 'last': (hs[-1], errs[-1])}
    if g is not None or g_last is not None:
        g = torch.zeros_like(x) if g is None else g.cpu().double()
        G = torch.zeros_like(x[0]) if g_last is None else g_last.cpu().double()
        size, err = G.abs(), torch.zeros_like(G)
        dx, df, edx, edf = [], [], [], []
        for t in range(T - 1, -1, -1):
            G, size = G + g[t], size + g[t].abs()
            err = err + 4 * R * size
            diff = before[t] - x[t]
            dx.append(b[t] * G)
            edx.append(b[t] * err + b[t] * size * (eb[t] + 2 * R))
            df.append(G * diff * a[t] * b[t])
            both = before[t].abs() + x[t].abs()
            wide = both if apart else diff.abs()
            edf.append(a[t] * b[t] * (err * wide + size * (err_before[t] + R * both) +
                                      size * wide * (ea[t] + eb[t] + 4 * R)))
            err = on[t] * (a[t] * err + a[t] * size * (ea[t] + 4 * R))
            G, size = on[t] * a[t] * G, on[t] * a[t] * size
        out['dx'] = (torch.stack(dx[::-1]), torch.stack(edx[::-1]))
        out['dgate'] = (torch.stack(df[::-1]), torch.stack(edf[::-1]))
        out['dh0'] = (G, err)
    return out


def close(got, want, tol, name):
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2 if got.dtype in (torch.float16, torch.bfloat16) else 0.0
    floor = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -120
    bad = ~((got.double() - want).abs() <= tol + half * (want.abs() + tol) + floor)
    assert not bad.any(), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, at {bad.nonzero()[:4].tolist()}: got {got[bad][:4].tolist()}, "
        f"want {want[bad][:4].tolist()}, within {tol[bad][:4].tolist()}"
    )


def check(x, f, h0=None, reset=None, use=('h', 'last'), seed=0):
    gen = torch.Generator().manual_seed(seed)
    leaves = [x.detach().requires_grad_(), f.detach().requires_grad_()]
    start = None
    if h0 is not None:
        start = h0.detach().requires_grad_()
        leaves.append(start)
    h, last = gated_linear_recurrence(leaves[0], leaves[1], start, reset)
    assert h.dtype == x.dtype and h.shape == x.shape and last.shape == x.shape[1:]
    g = torch.randn(x.shape, generator=gen).to(x.dtype).to(x.device) if 'h' in use else None
    g_last = torch.randn(last.shape, generator=gen).to(last.dtype).to(x.device) if 'last' in use else None
    pairs = [(o, v) for o, v in ((h, g), (last, g_last)) if v is not None]
    grads = torch.autograd.grad([o for o, _ in pairs], leaves, [v for _, v in pairs])
    want = oracle(x, f, h0, reset, g, g_last)
    got = dict(zip(('h', 'last', 'dx', 'dgate', 'dh0'), (h, last) + grads))
    for name, v in got.items():
        close(v, *want[name], name)
    return got


def case(T, B, D, dtype=torch.float32, device='cpu', start=True, reset=0.1, seed=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(T, B, D, generator=gen).to(dtype)
    f = (torch.randn(T, B, D, generator=gen) * 2 + 2).to(dtype)
    h0 = torch.randn(B, D, generator=gen) if start else None
    mask = torch.rand(T, B, generator=gen) < reset if reset else None
    return tuple(None if v is None else v.to(device) for v in (x, f, h0, mask))


# --------------------------------------------------------------------------------------------------------------- CPU


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize('T,start,reset', [(1, True, 0.5), (1, False, 0), (9, True, 0.2), (40, False, 0.1)])
def test_cpu_lane(T, start, reset, dtype):
    check(*case(T, 3, 5, dtype, start=start, reset=reset))


def test_cpu_differences():
    x, f, h0, reset = case(6, 2, 3, torch.float64)
    leaves = [v.double().requires_grad_() for v in (x, f, h0)]
    assert torch.autograd.gradcheck(lambda *v: gated_linear_recurrence(*v, reset), leaves)


def test_refusals():
    x, f, h0, reset = case(4, 2, 3)
    for bad in (dict(x=x[0]), dict(x=x[:0], gate=f[:0]), dict(gate=f[:2]), dict(gate=f.double()), dict(h0=h0[:1]),
                dict(h0=h0.long()), dict(reset=reset[:2]), dict(reset=reset.float()), dict(x=x.long(), gate=f.long())):
        args = dict(x=x, gate=f, h0=h0, reset=reset)
        args.update(bad)
        with pytest.raises((ValueError, TypeError)):
            gated_linear_recurrence(**args)


def test_module_steps_equal_the_sequence():
    torch.manual_seed(0)
    rnn = get_lstm('glr', 6, 8, num_layers=2)
    assert isinstance(rnn, GatedLinearRNN)
    x = torch.randn(7, 3, 6)
    whole, state = rnn(x)
    parts, prev = [], None
    for t in range(7):
        out, prev = rnn(x[t:t + 1], prev)
        parts.append(out)
    assert torch.allclose(whole, torch.cat(parts), atol=1e-6)
    assert len(state) == 3 and state[0]['h'].shape == (2, 1, 8)
    assert torch.allclose(state[1]['h'], prev[1]['h'], atol=1e-6)
    reset = torch.zeros(7, 3, dtype=torch.bool)
    reset[4, 1] = True
    cut, _ = rnn(x, reset=reset)
    again, _ = rnn(x[4:, 1:2])
    assert torch.allclose(cut[4:, 1:2], again, atol=1e-6)
    assert torch.allclose(cut[:, 0], whole[:, 0], atol=1e-6)


def test_recurrent_q_network():
    from ding.model import DRQN
    torch.manual_seed(0)
    model = DRQN(5, 3, [16, 16], lstm_type='glr')
    data = torch.randn(6, 2, 5)
    out = model({'obs': data, 'prev_state': [None, None]}, saved_state_timesteps=[2, 4])
    plain = model({'obs': data, 'prev_state': [None, None]})
    assert torch.allclose(out['logit'], plain['logit'], atol=1e-6) and out['logit'].shape == (6, 2, 3)
    step = model({'obs': data[0], 'prev_state': [None, None]}, inference=True)
    assert torch.allclose(step['logit'], plain['logit'][0], atol=1e-6)
    plain['logit'].sum().backward()
    assert all(p.grad is not None for p in model.rnn.parameters())


# --------------------------------------------------------------------------------------------------------------- GPU


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('T', [1, 2, 7, 8, 9, 16, 17, 31, 33, 64, 127, 129, 256, 257, 513, 1300])
def test_gpu_lengths(T, dtype):
    check(*case(T, 3, 37, dtype, 'cuda', seed=T))


@gpu
@pytest.mark.parametrize('B,D', [(1, 1), (1, 2), (5, 1), (2, 63), (1, 64), (1, 129), (3, 128), (7, 200), (260, 3)])
@pytest.mark.parametrize('start,reset', [(True, 0.1), (False, 0)])
@pytest.mark.parametrize('T', [5, 300])
def test_gpu_widths(T, B, D, start, reset):
    check(*case(T, B, D, torch.bfloat16, 'cuda', start, reset, seed=D))
    check(*case(T, B, D, torch.float32, 'cuda', start, reset, seed=D))


@gpu
@pytest.mark.parametrize('use', [('h', ), ('last', )])
def test_gpu_only_one_gradient_is_given(use):
    check(*case(70, 2, 50, torch.float32, 'cuda'), use=use)
    check(*case(700, 2, 50, torch.bfloat16, 'cuda'), use=use)


@gpu
@pytest.mark.parametrize('T', [3, 150, 900])
def test_gpu_strides(T):
    B, D = 3, 46
    gen = torch.Generator().manual_seed(T)
    packed = torch.randn(T, B, 2 * D + 1, generator=gen).cuda().to(torch.bfloat16)
    check(packed[..., :D], packed[..., D:2 * D])
    check(packed[..., 1:D + 1], packed[..., D + 1:])
    other = torch.randn(B, T, 2 * D, generator=gen).cuda().transpose(0, 1)  # batch first in memory
    check(other[..., :D], other[..., D:])
    check(other[:, :1, :D].expand(T, B, D), other[..., D:])  # one input for the whole batch
    dense = torch.randn(D, T, B, generator=gen).cuda().permute(1, 2, 0)  # channels are not dense
    check(dense, dense.flip(0))
    check(*case(T, B, D, torch.float32, 'cuda', start=False)[:2], h0=torch.randn(D, B, generator=gen).cuda().t(),
          reset=(torch.rand(B, T, generator=gen) < 0.1).cuda().t())
    check(*case(T, B, D, torch.float32, 'cuda', start=False)[:2], h0=torch.randn(B, D, generator=gen).cuda().bfloat16())


@gpu
@pytest.mark.parametrize('T', [4, 400])
def test_gpu_extreme_gates(T):
    x, f, h0, reset = case(T, 2, 40, torch.float32, 'cuda')
    f[..., :10] = 30.0  # keeps its state
    f[..., 10:20] = -30.0  # follows its input
    f[..., 20:24] = 1e4
    f[..., 24:28] = -1e4
    f[..., 28] = float('inf')
    f[..., 29] = float('-inf')
    h, last = gated_linear_recurrence(x, f, h0, reset)
    assert torch.isfinite(h).all() and torch.equal(h[-1], last)
    keep = [i for i in range(40) if i not in (28, 29)]
    check(x[..., keep].contiguous(), f[..., keep].contiguous(), h0[:, keep].contiguous(), reset)
    reset[:] = True
    check(x, f.clamp(-50, 50), h0, reset)
    f[1, 0, 5] = float('nan')
    bad = torch.isnan(gated_linear_recurrence(x, f, h0)[0])
    assert bad[1:, 0, 5].all() and bad.sum() == T - 1


@gpu
def test_gpu_reset_hides_what_was_before():
    x, f, h0, _ = case(600, 2, 70, torch.float32, 'cuda')
    reset = torch.zeros(600, 2, dtype=torch.bool, device='cuda')
    reset[350, 0] = True
    x[100, 0] = float('inf')
    h, last = gated_linear_recurrence(x, f, h0, reset)
    assert torch.isfinite(h[350:]).all() and torch.isfinite(last).all() and torch.isfinite(h[:, 1]).all()
    again, _ = gated_linear_recurrence(x[350:, :1], f[350:, :1])
    want = oracle(x[350:, :1], f[350:, :1], None, None)
    close(h[350:, :1], *want['h'], 'h')
    close(again, *want['h'], 'h')


@gpu
@pytest.mark.parametrize('T', [1, 200])
def test_gpu_without_gradient(T):
    x, f, h0, reset = case(T, 2, 30, device='cuda')
    want = gated_linear_recurrence(x, f, h0, reset)
    with torch.inference_mode():
        again = gated_linear_recurrence(x, f, h0, reset)
    with torch.no_grad():
        out = gated_linear_recurrence(x.requires_grad_(), f, h0, reset)
    assert not out[0].requires_grad
    for a, b, c in zip(want, out, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    h, last = gated_linear_recurrence(x, f, h0.requires_grad_(), reset)
    assert h.requires_grad and last.requires_grad
    dx, dh0 = torch.autograd.grad(h.sum(), [x, h0])  # the gates take none
    assert torch.isfinite(dx).all() and torch.isfinite(dh0).all()


@gpu
def test_gpu_refusals():
    x, f, h0, reset = case(4, 2, 3, device='cuda')
    with pytest.raises(TypeError):
        gated_linear_recurrence(x.double(), f.double())
    with pytest.raises(ValueError):
        gated_linear_recurrence(x, f, h0.cpu())
    empty = gated_linear_recurrence(x[:, :0], f[:, :0])
    assert empty[0].shape == (4, 0, 3) and empty[1].shape == (0, 3)
    h, _ = gated_linear_recurrence(x.requires_grad_(), f)
    grad, = torch.autograd.grad(h.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@gpu
def test_gpu_offsets_pass_32_bits():
    T, D = 16500, 131072
    x = torch.empty(T, 1, D, dtype=torch.bfloat16, device='cuda').normal_()
    f = torch.empty_like(x).normal_(2.0)
    assert x.numel() > 2 ** 31
    x.requires_grad_()
    f.requires_grad_()
    h, last = gated_linear_recurrence(x, f)
    g = torch.zeros_like(h)
    g[-40:] = 1.0
    dx, df = torch.autograd.grad(h, [x, f], g)
    tail = slice(T - 600, T)  # a state forgets what lies 600 steps back: 0.998^600 at most, and far less here
    cols = torch.tensor([0, 1, D // 2, D - 2, D - 1], device='cuda')
    want = oracle(x[tail][..., cols], f[tail][..., cols], None, None, g[tail][..., cols])
    close(last[..., cols], want['last'][0], want['last'][1] + 1e-6, 'last')
    close(dx[tail][..., cols], *want['dx'], 'dx')
    close(h[-100:][..., cols], want['h'][0][-100:], want['h'][1][-100:] + 1e-6, 'h')


@gpu
def test_gpu_stream_and_graph():
    x, f, h0, reset = case(900, 2, 300, torch.bfloat16, 'cuda')
    g = torch.randn(900, 2, 300, device='cuda').bfloat16()

    def step():
        leaves = [v.detach().requires_grad_() for v in (x, f, h0)]
        h, last = gated_linear_recurrence(*leaves, reset)
        return (h, last) + torch.autograd.grad([h, last], leaves, [g, torch.ones_like(last)])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for seed in range(3):
        for to, new in zip((x, f, h0, reset), case(900, 2, 300, torch.bfloat16, 'cuda', seed=seed + 3)):
            to.copy_(new)
        graph.replay()
        got = [t.clone() for t in kept]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@gpu
def test_gpu_two_streams_at_once():
    cases = [case(2000, 2, 256, torch.bfloat16, 'cuda', seed=s) for s in (1, 2)]
    alone = [gated_linear_recurrence(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for c, s in zip(cases, streams):
        with torch.cuda.stream(s):
            for _ in range(4):
                out = gated_linear_recurrence(*c)
            got.append(out)
    torch.cuda.synchronize()
    for a, b in zip(alone, got):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@gpu
def test_gpu_module():
    torch.manual_seed(0)
    rnn = get_lstm('glr', 20, 48, num_layers=2)
    x = torch.randn(30, 4, 20)
    want, _ = rnn(x)
    got, state = rnn.cuda()(x.cuda())
    assert torch.allclose(want, got.cpu(), atol=1e-4) and state[0]['h'].is_cuda
    got.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in rnn.parameters())


def _r2d2(cuda):
    from ding.policy import create_policy
    from ding.policy.base_policy import get_policy_cls
    from ding.utils import EasyDict, deep_merge_dicts
    cfg = dict(
        type='r2d2', cuda=cuda, on_policy=False,
        model=dict(obs_shape=8, action_shape=3, encoder_hidden_size_list=[32, 32], lstm_type='glr'),
        learn=dict(batch_size=4), collect=dict(unroll_len=8, env_num=2), unroll_len=8, nstep=2, burnin_step=2,
    )
    cfg = EasyDict(deep_merge_dicts(get_policy_cls(EasyDict(dict(type='r2d2'))).default_config(), cfg))
    policy = create_policy(cfg, enable_field=['learn', 'collect'])
    gen = torch.Generator().manual_seed(0)
    samples = [{
        'obs': [torch.randn(8, generator=gen) for _ in range(8)],
        'action': [torch.randint(0, 3, (), generator=gen) for _ in range(8)],
        'reward': [torch.randn(2, generator=gen) for _ in range(8)],
        'done': [False] * 8,
        'prev_state': [None] * 8,
    } for _ in range(4)]
    info = policy._forward_learn(samples)
    assert torch.isfinite(torch.as_tensor(float(info['total_loss'])))
    for _ in range(2):  # a collector's steps, with the states that the first left
        out = policy._forward_collect({i: torch.randn(8, generator=gen) for i in range(2)}, eps=0.1)
        assert set(out) == {0, 1}


def test_recurrent_policy_cpu():
    _r2d2(False)


@gpu
def test_recurrent_policy_gpu():
    _r2d2(True)
