"""Orthogonalised matrices where precision is lost first: one direction far above the others.

A matrix of a mean component and small noise has all its other singular values below 1/100 of the largest. Five steps
multiply those by a^5 = 485 and with them whatever error came to lie among them.
"""
import pytest
import torch

from ding.torch_utils import orthogonalize
from ding.torch_utils.optimizer_helper import _newton_schulz_plan

DEFAULT = (3.4445, -4.7750, 2.0315)
gpu = pytest.mark.gpu


def dominated(kind, m, n, noise, seed=0):
    gen = torch.Generator().manual_seed(seed)
    rows, columns = torch.randn(m, 1, generator=gen), torch.randn(1, n, generator=gen)
    mean = {'all': torch.ones(1, 1), 'rows': rows, 'columns': columns, 'outer': rows @ columns}[kind]
    return mean + noise * torch.randn(m, n, generator=gen)


def exact(matrix, steps=5, coefficients=DEFAULT, eps=1e-7):
    """The iteration in 64 bits, on the matrix's device."""
    a, b, c = coefficients
    tall = matrix.shape[-2] > matrix.shape[-1]
    x = matrix.detach().double()
    x = x.transpose(-2, -1).contiguous() if tall else x
    x = x / (x.norm(dim=(-2, -1), keepdim=True) + eps)
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1).contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if tall else x


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('m,n', [(64, 64), (1001, 2731), (4096, 16384)])
def test_span_keeps_digits(m, n, dtype):
    """A step on the Gram matrix after the first of a span costs max(q) in precision, q(u) = a + b u + c u^2."""
    for coefficients, steps, q in ((DEFAULT, 5, 3.4445), ((1.875, -1.25, 0.375), 10, 1.875), ((1.5, -0.5, 0.0), 8, 1.5)):
        span = _newton_schulz_plan(coefficients, steps, dtype, m, n)[1]
        assert q ** (max(span, 1) - 1) <= (1 if dtype == torch.float32 else 4)


@gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('kind,noise', [('all', 1e-2), ('all', 3e-3), ('rows', 3e-3), ('columns', 3e-3), ('outer', 3e-3)])
@pytest.mark.parametrize('m,n', [(200, 260), (768, 2900), (2731, 1001), (1500, 6100)])
def test_gpu_dominant_direction(m, n, kind, noise, dtype):
    """The result is off by its rounding and by what 22-bit factors cost.

    Rounding: as far as the rounded 64-bit result; over 52000 entries and more the sums of the squared roundings of two
    such results differ by 2% at most (five deviations of 0.9 / sqrt(52000)). Factors: 2^-22 of X, which five steps
    multiply by 485 at most and a span of two steps by 3.4445 once more: 4e-4."""
    x = dominated(kind, m, n, noise).to(dtype).cuda()
    want = exact(x)
    rounding = (want.to(dtype).double() - want).norm()
    off = (orthogonalize(x).double() - want).norm()
    assert off <= 1.02 * rounding + 4e-4 * want.norm(), f"off by {off / want.norm():.3g}"


def check_range(device):
    """Numbers at the ends of their types' ranges, and an eps that is nothing beside any of them."""
    for dtype, small in ((torch.float32, 1e-37), (torch.float32, 1e-43), (torch.bfloat16, 1e-37), (torch.float16, 1e-6)):
        for shape in ((20, 30), (200, 300), (3, 90, 140), (300, 200)):
            zero = torch.zeros(shape, dtype=dtype, device=device)
            for eps in (1e-7, 1e-38, 1e-100, 5e-324):
                assert torch.equal(orthogonalize(zero, eps=eps), zero)
            gen = torch.Generator().manual_seed(0)
            noise = torch.randn(shape, generator=gen)
            for scale in (small, torch.finfo(dtype).max / 8):
                x = (noise * scale).to(dtype).to(device)
                # a rounding, and 2^-22 * 485 for factors of 22 bits (the lane on the CPU is nearer)
                want = exact(x, eps=1e-100)
                allowed = torch.finfo(dtype).eps / 2 + 1.2e-4
                for eps in (1e-100, 5e-324):
                    off = (orthogonalize(x, eps=eps).double() - want).norm() / want.norm()
                    assert off <= allowed, f"{dtype} {shape} {scale} {eps}: off by {off:.3g}"


def test_range_cpu():
    check_range('cpu')


@gpu
def test_gpu_range():
    check_range('cuda')


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_gpu_largest_norm(dtype):
    """A norm whose inverse is subnormal in 32 bits."""
    gen = torch.Generator(device='cuda').manual_seed(0)
    x = torch.empty(2200, 2100, device='cuda').uniform_(-1, 1, generator=gen).mul_(3e38).to(dtype)
    want = exact(x)
    off = (orthogonalize(x).double() - want).norm() / want.norm()
    assert off <= torch.finfo(dtype).eps / 2 + 1.2e-4, f"off by {off:.3g}"
