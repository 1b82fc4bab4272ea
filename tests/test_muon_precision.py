"""Muon's steps against its definition in 64 bits: weights of few bits, momentum that one direction dominates, and
matrices too large for one workgroup."""
import math

import pytest
import torch

from ding.torch_utils import Muon

gpu = pytest.mark.gpu


def exact_steps(grads, momentum, nesterov, lr):
    """What the steps add up to in 64 bits."""
    a, b, c = 3.4445, -4.7750, 2.0315
    total = buf = torch.zeros_like(grads[0], dtype=torch.float64)
    for g in grads:
        buf = momentum * buf + g.double()
        x = g.double() + momentum * buf if nesterov else buf
        x = x.reshape(x.shape[0], -1)
        scale = 0.2 * math.sqrt(max(x.shape))
        tall = x.shape[0] > x.shape[1]
        x = x.t().contiguous() if tall else x
        x = x / (x.norm() + 1e-7)
        for _ in range(5):
            gram = x @ x.t().contiguous()
            x = a * x + (b * gram + c * (gram @ gram)) @ x
        total = total - lr * scale * (x.t() if tall else x).reshape(g.shape)
    return total


def check(device, dtype, shape, noise, nesterov=True, steps=3):
    """Weights that start at zero take a few steps.

    Each step rounds the weights, by half a step of their type at most. The updates are off by what factors of 22 bits
    cost, 2^-22 * 485 = 1.2e-4, and by the momentum's roundings, 2^-24 of the mean or 6e-6 of 1% of noise: 2e-4."""
    gen = torch.Generator().manual_seed(sum(shape))
    p = torch.zeros(shape, dtype=dtype, device=device).requires_grad_()
    opt, grads = Muon([p], lr=0.5, nesterov=nesterov), []
    for _ in range(steps):
        g = (noise < 1) + noise * torch.randn(shape, generator=gen)
        p.grad = g.to(device=device, dtype=dtype)
        grads.append(p.grad.clone())
        opt.step()
    want = exact_steps(grads, 0.95, nesterov, 0.5)
    size = want.norm()
    off = (p.detach().double() - want).norm() / size
    allowed = steps * torch.finfo(dtype).eps / 2 + 2e-4
    assert off <= allowed, f"off by {off:.3g}, allowed {allowed:.3g}"


@pytest.mark.parametrize('nesterov', [True, False])
@pytest.mark.parametrize('noise', [1.0, 1e-2])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
def test_steps_cpu(dtype, noise, nesterov):
    check('cpu', dtype, (48, 96), noise, nesterov)
    check('cpu', dtype, (40, 3, 3, 3), noise, nesterov)


@gpu
@pytest.mark.parametrize('noise', [1.0, 1e-2])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('shape', [(48, 96), (130, 700), (1025, 515), (64, 33, 3, 3)])
def test_steps_gpu(shape, dtype, noise):
    check('cuda', dtype, shape, noise)


@gpu
def test_steps_gpu_float64():
    """Weights of 64 bits are refused by the kernels as any such matrix is."""
    p = torch.zeros(8, 8, dtype=torch.float64, device='cuda').requires_grad_()
    p.grad = torch.ones_like(p)
    with pytest.raises(TypeError):
        Muon([p]).step()
