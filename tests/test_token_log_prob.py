"""Token log probabilities: the CPU lane and the HIP kernels against the formulas in 64 bits.

Tolerances count roundings of 2^-24 (32-bit steps). With d = (x - max) log2(e) / T, s = sum 2^d:
a term's exponent is off by 2 roundings of |d|, the exponential and the logarithm by 2 each, and a sum over a row passes
at most 32 + 6 + 4 + 6 additions, held here as 50. An output of fewer bits adds half a step of its type.
"""
import math

import pytest
import torch

from ding.rl_utils import (
    token_log_prob, naive_method, efficient_method, fused_method, grpo_policy_error, grpo_policy_data,
    rloo_policy_error, rloo_policy_data
)

R = 2.0 ** -24
LOG2E = 1.4426950408889634
LN2 = math.log(2.0)
gpu = pytest.mark.gpu


def oracle(logits, index, temperature=1.0, ignore_index=None, top_k=0, g_lp=None, g_h=None, g_top=None):
    """The formulas in 64 bits on the CPU, and how far 32-bit arithmetic may be from them."""
    x = logits.detach().cpu().double()
    V = x.shape[-1]
    index = index.cpu().long()
    live = torch.ones_like(index, dtype=torch.bool) if ignore_index is None else index != ignore_index
    on = live.unsqueeze(-1)
    d = (x - x.amax(-1, keepdim=True)) * (LOG2E / temperature)
    log2s = d.exp2().sum(-1, keepdim=True).log2()
    lp2 = d - log2s
    p = lp2.exp2()
    finite = torch.where(p > 0, d, torch.zeros_like(d))
    mean_d, mean_d2 = (p * finite.abs()).sum(-1), (p * finite ** 2).sum(-1)
    token = torch.where(live, index, torch.zeros_like(index)).clamp(0, V - 1).unsqueeze(-1)
    out, tol = {}, {}
    hit = d.gather(-1, token).squeeze(-1)
    near = (50 + 2 * mean_d + 4 * log2s.squeeze(-1) + 4) * R
    out['log_prob'] = torch.where(live, lp2.gather(-1, token).squeeze(-1) * LN2, 0.0)
    tol['log_prob'] = 3 * R * hit.abs() + near
    h = (log2s.squeeze(-1) - (p * finite).sum(-1)) * LN2
    out['entropy'] = torch.where(live, h, 0.0)
    tol['entropy'] = (3 * mean_d2 + 110 * mean_d) * R + near
    if top_k:
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top_k]
        out['top_index'] = torch.where(on, order, -1)
        out['top_log_prob'] = torch.where(on, lp2.gather(-1, order) * LN2, 0.0)
        tol['top_log_prob'] = 3 * R * d.gather(-1, order).abs() + near.unsqueeze(-1)
    if g_lp is not None or g_h is not None or g_top is not None:
        zero = torch.zeros(index.shape, dtype=torch.double)
        g_lp = zero if g_lp is None else g_lp.cpu().double()
        g_h = zero if g_h is None else g_h.cpu().double()
        share = torch.zeros_like(x)
        share.scatter_add_(-1, token, g_lp.unsqueeze(-1))
        total = g_lp
        size = g_lp.abs()
        if g_top is not None:
            g_top = g_top.cpu().double()
            share.scatter_add_(-1, order, g_top)
            total = total + g_top.sum(-1)
            size = size + g_top.abs().sum(-1)
        gh, h1 = g_h.unsqueeze(-1), h.unsqueeze(-1)
        lp = torch.where(p > 0, lp2 * LN2, torch.zeros_like(p))
        grad = share - p * total.unsqueeze(-1) - gh * p * (lp + h1)
        out['grad'] = torch.where(on, grad / temperature, 0.0)
        factor = size.unsqueeze(-1) + gh.abs() * (lp.abs() + h1)
        part = p * factor
        # the sum of a row's top + 1 upstream gradients rounds top times. A probability below the smallest normal
        # number 2^-126 comes out of the exponential as 0: off by at most 2^-126, times what it is multiplied by.
        tol['grad'] = (part * (3 * finite.abs() * R + near.unsqueeze(-1) + (8 + top_k) * R) + 2.0 ** -126 * factor +
                       p * gh.abs() * (tol['entropy'].unsqueeze(-1) + 3 * R * finite.abs() + near.unsqueeze(-1)) +
                       8 * R * share.abs()) / temperature
    return out, tol


def close(got, want, tol, name=''):
    got = got.detach().cpu()
    half = 0.0 if got.dtype in (torch.float32, torch.float64) else torch.finfo(got.dtype).eps / 2
    floor = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -126
    # a value beyond the type's largest number rounds to infinity
    want = torch.where(want.abs() > torch.finfo(got.dtype).max, want.sign() * float('inf'), want)
    got = got.double()
    bad = ~((got - want).abs() <= tol + half * (want.abs() + tol) + floor)
    both = (torch.isnan(got) & torch.isnan(want)) | (torch.isinf(want) & (got == want))
    bad &= ~both
    assert not bad.any(), (
        f"{name}: {int(bad.sum())} of {bad.numel()} off, at {bad.nonzero()[:4].tolist()}: got {got[bad][:4].tolist()}, "
        f"want {want[bad][:4].tolist()}, within {tol[bad][:4].tolist()}"
    )


def check(logits, index, temperature=1.0, ignore_index=None, top_k=0, entropy=True, seed=0):
    """Forward and gradient of one call against the oracle."""
    gen = torch.Generator().manual_seed(seed)
    leaf = logits.detach().requires_grad_()
    got = token_log_prob(leaf, index, temperature, ignore_index, entropy, top_k)
    heads, grads = [got.log_prob], [torch.randn(index.shape, generator=gen)]
    if entropy:
        heads.append(got.entropy)
        grads.append(torch.randn(index.shape, generator=gen))
    if top_k:
        heads.append(got.top_log_prob)
        grads.append(torch.randn(*index.shape, top_k, generator=gen))
    grad, = torch.autograd.grad(heads, [leaf], [g.to(h.device, h.dtype) for g, h in zip(grads, heads)])
    want, tol = oracle(logits, index, temperature, ignore_index, top_k, grads[0], grads[1] if entropy else None,
                       grads[-1] if top_k else None)
    close(got.log_prob, want['log_prob'], tol['log_prob'], 'log_prob')
    if entropy:
        close(got.entropy, want['entropy'], tol['entropy'], 'entropy')
    if top_k:
        assert torch.equal(got.top_index.cpu(), want['top_index'])
        close(got.top_log_prob, want['top_log_prob'], tol['top_log_prob'], 'top_log_prob')
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    close(grad, want['grad'], tol['grad'], 'grad')
    return got, grad


def case(shape, V, dtype=torch.float32, device='cpu', scale=3.0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    logits = (torch.randn(*shape, V, generator=gen) * scale).to(dtype)
    index = torch.randint(0, V, shape, generator=gen)
    return logits.to(device), index.to(device)


# --------------------------------------------------------------------------------------------------------------- CPU


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize('top_k', [0, 3])
def test_cpu_lane(dtype, top_k):
    logits, index = case((3, 5), 37, dtype)
    index[0, :2] = -100
    check(logits, index, 0.7, -100, top_k)


def test_cpu_masks():
    logits, index = case((4, ), 11)
    logits[:, 3:7] = float('-inf')
    index = index.remainder(3)
    check(logits, index, 1.3, None, 2)
    logits[1] = float('-inf')
    got = token_log_prob(logits, index, entropy=True)
    assert torch.isnan(got.log_prob[1]) and torch.isfinite(got.log_prob[[0, 2, 3]]).all()
    low = torch.full((2, 9), torch.finfo(torch.float32).min)
    got = token_log_prob(low, torch.zeros(2, dtype=torch.long), temperature=0.5, entropy=True)
    assert torch.allclose(got.log_prob, torch.full((2, ), -math.log(9.0)))


def test_cpu_differences():
    logits, index = case((2, 3), 7, torch.float64)
    index[1, 2] = -1
    leaf = logits.requires_grad_()

    def f(x):
        out = token_log_prob(x, index, 0.8, -1, True, 2)
        return out.log_prob, out.entropy, out.top_log_prob

    assert torch.autograd.gradcheck(f, (leaf, ))


def test_refusals():
    logits, index = case((2, 3), 7)
    with pytest.raises(ValueError):
        token_log_prob(logits, index[:, :2])
    with pytest.raises(ValueError):
        token_log_prob(logits, index, temperature=0.0)
    with pytest.raises(ValueError):
        token_log_prob(logits, index, temperature=float('nan'))
    with pytest.raises(ValueError):
        token_log_prob(logits, index, temperature=1e-40)
    with pytest.raises(ValueError):
        token_log_prob(logits, index, top_k=8)
    with pytest.raises(ValueError):
        token_log_prob(logits, index, top_k=-1)
    with pytest.raises(TypeError):
        token_log_prob(logits, index.float())
    with pytest.raises(TypeError):
        token_log_prob(logits.long(), index)
    with pytest.raises(ValueError):
        token_log_prob(logits[..., :0], index)
    with pytest.raises(Exception):
        token_log_prob(logits, index + 7)


def test_methods_and_losses_agree():
    new, action = case((4, 6), 19, seed=1)
    old, ref = case((4, 6), 19, seed=2)[0], case((4, 6), 19, seed=3)[0]
    assert torch.allclose(fused_method(new, action), naive_method(new, action), atol=1e-6)
    assert torch.allclose(fused_method(new, action), efficient_method(new, action), atol=1e-5)
    adv, weight = torch.randn(4), (torch.rand(4, 6) > 0.3).float()
    a = grpo_policy_error(grpo_policy_data(new, old, ref, action, adv, weight))
    b = grpo_policy_error(grpo_policy_data(new, old, ref, action, adv, weight), log_prob_fn=fused_method)
    assert torch.allclose(a[0].policy_loss, b[0].policy_loss, atol=1e-5)
    a = rloo_policy_error(rloo_policy_data(new, old, action, torch.randn(4, 1), weight))
    assert torch.isfinite(a[0].policy_loss)


# --------------------------------------------------------------------------------------------------------------- GPU


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('V', [1, 2, 18, 64, 65, 512, 513, 2000, 8191, 8192, 8193, 50001])
def test_gpu_sizes(V, dtype):
    logits, index = case((3, 5), V, dtype, 'cuda', seed=V)
    check(logits, index, 0.9, None, min(V, 4))
    check(logits, index, entropy=False)


@gpu
@pytest.mark.parametrize('V,top_k', [(40, 32), (512, 32), (700, 32), (8192, 1), (20000, 32), (131072, 20)])
def test_gpu_top(V, top_k):
    logits, index = case((4, ), V, torch.bfloat16, 'cuda', seed=V + 1)
    logits = (logits * 0.3).round() * 0.5  # many ties
    logits[1] = 0.25  # nothing but ties
    logits[2] = torch.arange(V, device='cuda').remainder(251).to(torch.bfloat16) - 300
    logits[3, ::2] = -0.0
    logits[3, 1::2] = 0.0
    index[0] = logits[0].float().argmax()
    check(logits, index, 1.1, None, top_k)


@gpu
@pytest.mark.parametrize('rows', [256, 257])
@pytest.mark.parametrize('V,top_k', [(8200, 1), (20000, 7), (40000, 32)])
def test_gpu_top_of_many_rows(rows, V, top_k):
    gen = torch.Generator(device='cuda').manual_seed(V)
    logits = torch.empty(rows, V, device='cuda').normal_(0, 2, generator=gen).bfloat16()
    logits[0] = 1.0
    logits[1] = torch.arange(V, device='cuda').float().div(V).bfloat16()  # long runs of equal logits
    logits[2] = -torch.arange(V, device='cuda').float().bfloat16()
    logits[3, 5:] = float('-inf')
    index = torch.randint(0, V, (rows, ), device='cuda', generator=gen)
    index[3] = 2
    got = token_log_prob(logits, index, entropy=True, top_k=top_k)
    want = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[:, :top_k]
    assert torch.equal(got.top_index, want)
    keep = list(range(6)) + [100, rows - 1]
    want, tol = oracle(logits[keep], index[keep], 1.0, None, top_k)
    close(got.top_log_prob[keep], want['top_log_prob'], tol['top_log_prob'], 'top_log_prob')
    close(got.entropy[keep], want['entropy'], tol['entropy'], 'entropy')


@gpu
@pytest.mark.parametrize('V', [30, 300, 1025, 9001])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gpu_masks(V, dtype):
    logits, index = case((6, ), V, dtype, 'cuda')
    logits[:, 1::3] = float('-inf')
    logits[2, 1:] = float('-inf')  # a single token left
    logits[3, 1::3] = torch.finfo(dtype).min
    logits[4, :] = torch.finfo(dtype).min  # all of them the type's lowest: uniform
    index = torch.zeros_like(index)
    check(logits, index, 0.5, None, 3)
    index[5] = 1  # a masked token that was taken
    got = token_log_prob(logits, index, entropy=True)
    assert got.log_prob[5].item() == float('-inf') and torch.isfinite(got.entropy).all()
    logits[0] = float('-inf')
    logits[1, 2] = float('nan')
    logits[2, 0] = float('inf')
    got = token_log_prob(logits, index, entropy=True)
    assert torch.isnan(got.log_prob[:3]).all() and torch.isnan(got.entropy[:3]).all()
    assert torch.isfinite(got.log_prob[3:5]).all()


@gpu
@pytest.mark.parametrize('V', [21, 400, 3001, 17000])
def test_gpu_ignored_rows(V):
    logits, index = case((4, 6), V, torch.bfloat16, 'cuda')
    index[0, 1:4] = -100
    index[3] = -100
    logits[3] = float('nan')  # rows that are not read
    got, grad = check(logits.nan_to_num(), index, 1.0, -100, 2)
    assert torch.equal(token_log_prob(logits, index, ignore_index=-100).log_prob[3], torch.zeros(6, device='cuda'))
    index[:] = 0
    check(logits.nan_to_num(), index, 1.0, 0, 2)


@gpu
@pytest.mark.parametrize('V', [8193, 16384, 17003])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gpu_many_rows(V, dtype):
    rows = 1030  # enough for a workgroup to walk a row of its own
    logits = torch.empty(rows, V, dtype=dtype, device='cuda').normal_(0, 3)
    logits[:, 8190::7] = float('-inf')
    logits[1, :8192] = float('-inf')  # nothing but masked tokens at first
    logits[2] = torch.finfo(dtype).min
    logits[3, :8192] = torch.finfo(dtype).min
    logits[4] = torch.linspace(-40, 40, V, device='cuda').to(dtype)  # the maximum moves all the time
    logits[5, 5] = float('nan')
    logits[6] = float('-inf')
    index = torch.randint(0, V // 8, (rows, ), device='cuda') * 7
    index[7::5] = -100
    index[1] = 8193 - 1 if V == 8193 else 8193
    index[2:5] = 3
    got = token_log_prob(logits, index, 0.8, -100, True)
    assert torch.isnan(got.log_prob[5:7]).all() and torch.isnan(got.entropy[5:7]).all()
    keep = [0, 1, 2, 3, 4, 7, 8, 9, 500, rows - 2, rows - 1]
    want, tol = oracle(logits[keep], index[keep], 0.8, -100)
    close(got.log_prob[keep], want['log_prob'], tol['log_prob'], 'log_prob')
    close(got.entropy[keep], want['entropy'], tol['entropy'], 'entropy')
    alone = token_log_prob(logits, index, 0.8, -100).log_prob  # without the entropy
    assert torch.equal(alone.nan_to_num(), got.log_prob.nan_to_num())


@gpu
@pytest.mark.parametrize('V', [18, 333, 5001])
def test_gpu_strides(V):
    full, _ = case((3, 6), V + 3, torch.bfloat16, 'cuda')
    index = torch.randint(0, V, (3, 5), device='cuda')
    check(full[:, :-1, 1:V + 1], index, 1.0, None, 2)  # shifted, a part of the vocabulary
    check(full[:, 1:, :V], index)
    check(full.transpose(0, 1)[:5, :, :V], index.t())
    check(full[:1, :1, :V].expand(3, 5, V), index)  # the same row for every token
    check(full[:, :5, :V].permute(2, 0, 1).contiguous().permute(1, 2, 0), index)  # V is not the dense dimension
    check(full[:2, :4, :V].reshape(2, 2, 2, V), index[:2, :4].reshape(2, 2, 2))
    check(full[0, 0, :V], index[0, 0])
    check(full[0, :5, :V], index[0].int())


@gpu
@pytest.mark.parametrize('V', [18, 300, 1000, 20000])
def test_gpu_token_out_of_range(V):
    logits, index = case((5, ), V, torch.float32, 'cuda')
    index[1], index[3] = V, -1
    leaf = logits.requires_grad_()
    out = token_log_prob(leaf, index, entropy=True).log_prob
    assert torch.isnan(out[[1, 3]]).all() and torch.isfinite(out[[0, 2, 4]]).all()
    grad, = torch.autograd.grad(out.sum(), leaf)
    assert torch.isnan(grad[[1, 3]]).all() and torch.isfinite(grad[[0, 2, 4]]).all()


@gpu
def test_gpu_nothing_to_do():
    out = token_log_prob(torch.empty(0, 4, 9, device='cuda'), torch.empty(0, 4, dtype=torch.long, device='cuda'),
                         entropy=True, top_k=2)
    assert out.log_prob.shape == (0, 4) and out.top_index.shape == (0, 4, 2)


@gpu
def test_gpu_refusals():
    logits, index = case((2, 3), 50, torch.float32, 'cuda')
    with pytest.raises(TypeError):
        token_log_prob(logits.double(), index)
    with pytest.raises(ValueError):
        token_log_prob(logits, index, top_k=33)
    with pytest.raises(ValueError):
        token_log_prob(logits, index.cpu())
    leaf = logits.requires_grad_()
    grad, = torch.autograd.grad(token_log_prob(leaf, index).log_prob.sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@gpu
def test_gpu_only_one_gradient_is_given():
    logits, index = case((4, ), 900, torch.float32, 'cuda')
    leaf = logits.requires_grad_()
    for pick in ('log_prob', 'entropy', 'top_log_prob'):
        out = token_log_prob(leaf, index, 1.0, None, True, 3)
        head = getattr(out, pick)
        grad, = torch.autograd.grad(head.sum(), leaf)
        g = torch.ones(4)
        want, tol = oracle(logits, index, 1.0, None, 3, g if pick == 'log_prob' else None,
                           g if pick == 'entropy' else None, torch.ones(4, 3) if pick == 'top_log_prob' else None)
        close(grad, want['grad'], tol['grad'], pick)


@gpu
@pytest.mark.parametrize('rows', [8, 1100])
@pytest.mark.parametrize('V', [1, 2, 18, 500, 5000, 40000])
def test_gpu_signs(rows, V):
    """Rows of one likely token: no rounding makes a probability larger than 1 or an entropy negative."""
    gen = torch.Generator().manual_seed(V)
    logits = torch.randn(rows, V, generator=gen).cuda()
    index = torch.randint(0, V, (rows,), generator=gen).cuda()
    logits[torch.arange(rows).cuda(), index] = torch.logspace(0, 4, rows).cuda()
    for top in (0, min(V, 2)):
        out = token_log_prob(logits, index, temperature=0.7, entropy=True, top_k=top)
        assert (out.log_prob <= 0).all() and (out.entropy >= 0).all()
        assert top == 0 or (out.top_log_prob <= 0).all()
        # One entry: with r the rounding of max k, d = r, s = 2^r and t = r 2^r, so both results are r - log2 s. The
        # power and the logarithm are off by a step (2^-23) of numbers near 1, t / s by less: 2^-22 and some.
        assert V > 1 or max(-out.log_prob.min(), out.entropy.max()) <= 2.0 ** -21


@gpu
@pytest.mark.parametrize('V', [18, 300, 9001])
def test_gpu_temperatures(V):
    logits, index = case((4, ), V, torch.float32, 'cuda')
    for temperature in (1e-30, 1e-3, 1e3, 1e30):
        got = token_log_prob(logits, index, temperature, entropy=True)
        want, tol = oracle(logits, index, temperature)
        close(got.log_prob, want['log_prob'], tol['log_prob'], 'log_prob')
        close(got.entropy, want['entropy'], tol['entropy'], 'entropy')


@gpu
def test_gpu_without_gradient():
    logits, index = case((3, 5), 700, torch.bfloat16, 'cuda')
    want = token_log_prob(logits, index, entropy=True, top_k=2)
    leaf = logits.detach().requires_grad_()
    with torch.no_grad():
        out = token_log_prob(leaf, index, entropy=True, top_k=2)
    assert not out.log_prob.requires_grad
    with torch.inference_mode():
        again = token_log_prob(logits, index, entropy=True, top_k=2)
    for a, b, c in zip(want, out, again):
        assert torch.equal(a, b) and torch.equal(a, c)
    out = token_log_prob(leaf, index, entropy=True, top_k=2)
    assert out.log_prob.requires_grad and out.entropy.requires_grad and not out.top_index.requires_grad
    leaf.data.add_(0)
    kept = token_log_prob(leaf, index)
    with torch.no_grad():
        leaf.add_(1.0)  # what the backward pass reads was changed
    with pytest.raises(RuntimeError):
        kept.log_prob.sum().backward()


@gpu
def test_gpu_offsets_pass_32_bits():
    V, rows = 70000, 31000
    logits = torch.empty(rows, V, dtype=torch.bfloat16, device='cuda').normal_()
    assert logits.numel() > 2 ** 31
    index = torch.randint(0, V, (rows, ), device='cuda')
    leaf = logits.requires_grad_()
    out = token_log_prob(leaf, index, entropy=True)
    g = torch.ones(rows, device='cuda')
    grad, = torch.autograd.grad([out.log_prob, out.entropy], [leaf], [g, g])
    last = slice(rows - 3, rows)
    want, tol = oracle(logits[last], index[last], g_lp=g[last], g_h=g[last])
    close(out.log_prob[last], want['log_prob'], tol['log_prob'])
    close(out.entropy[last], want['entropy'], tol['entropy'])
    close(grad[last], want['grad'], tol['grad'])


@gpu
def test_gpu_stream_and_graph():
    logits, index = case((8, 16), 10001, torch.bfloat16, 'cuda')
    g = torch.randn(8, 16, device='cuda')

    def step():
        leaf = logits.detach().requires_grad_()
        out = token_log_prob(leaf, index, 0.9, None, True, 4)
        grad, = torch.autograd.grad([out.log_prob, out.entropy], [leaf], [g, g])
        return out.log_prob, out.entropy, out.top_log_prob, out.top_index, grad

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
        logits.copy_(case((8, 16), 10001, torch.bfloat16, 'cuda', seed=seed + 5)[0])
        graph.replay()
        got = [t.clone() for t in kept]
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@gpu
def test_gpu_losses():
    new, action = case((4, 33), 3000, torch.float32, 'cuda', seed=1)
    old, ref = (case((4, 33), 3000, torch.float32, 'cuda', seed=s)[0] * 0.1 + new * 0.9 for s in (2, 3))
    adv, weight = torch.randn(4, device='cuda'), (torch.rand(4, 33, device='cuda') > 0.3).float()
    leaf = new.requires_grad_()
    losses = []
    for fn in (naive_method, fused_method):
        loss = grpo_policy_error(grpo_policy_data(leaf, old, ref, action, adv, weight), log_prob_fn=fn)[0].policy_loss
        losses.append((loss.detach(), torch.autograd.grad(loss, leaf)[0]))
    # both are 32-bit evaluations of the same expression: ratios exp(a - b) of log probabilities near 10 are off by a
    # few 2^-24 * 100
    assert torch.allclose(losses[0][0], losses[1][0], rtol=1e-4, atol=1e-5)
    assert (losses[0][1] - losses[1][1]).norm() <= 1e-4 * losses[0][1].norm()
