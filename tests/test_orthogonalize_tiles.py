"""Every way in which the products of an orthogonalisation are cut, on matrices of odd sizes.

Products go by tiles of 64 to 256 a side (128 in two forms: eight waves where each compute unit has one at most), and
those of symmetric results may also be cut along their depth. The sizes that reach each of them follow from a table of
costs, so the tests ask for the plan and hold it to what a case is listed for.
"""
import pytest
import torch

from ding.ops import dispatch
from ding.torch_utils import orthogonalize
from ding.torch_utils.optimizer_helper import _newton_schulz_plan

DEFAULT = (3.4445, -4.7750, 2.0315)
SLOW = (1.875, -1.25, 0.375)  # spans of three steps on the Gram matrix, which pairs two products in one launch
gpu = pytest.mark.gpu

# batch, rows, cols
CASES = [
    (17, 101, 203), (1, 129, 1163), (33, 587, 65), (130, 65, 587), (130, 129, 143), (64, 513, 530), (33, 193, 329),
    (64, 101, 911), (33, 1163, 129), (33, 193, 1739), (2, 1702, 1001), (3, 1001, 1020), (2, 1001, 8003),
    (3, 1500, 1514), (5, 1500, 1520), (33, 1001, 1015), (1, 1500, 8003), (1, 3015, 3001), (1, 3001, 8003),
    (3, 3001, 3015), (1, 4097, 4111), (17, 65, 8003),
]


def plan(batch, rows, cols, single):
    cuts = dispatch.newton_schulz_plan(batch, rows, cols, single)
    return {
        name: (side, 'eight waves' if side == 128 and groups <= 256 else '', parts > 1)
        for name, (side, parts, groups) in zip(('first', 'gram', 'one', 'two', 'update'), cuts)
    }


@pytest.mark.skipif(not dispatch.is_available(), reason='the kernels are not built')
def test_cases_reach_every_cut():
    sides = {(64, ''), (96, ''), (128, ''), (128, 'eight waves'), (192, ''), (256, '')}
    seen = {}
    for case in CASES:
        for single in (False, True):
            for name, (side, form, parts) in plan(*case, single).items():
                seen.setdefault(name if single or name != 'first' else 'gram', set()).add((side, form, parts))
    assert plan(17, 101, 203, False) == {}  # a workgroup takes 128 x 256 whole
    for name in ('gram', 'one', 'two', 'update'):
        reached = {(side, form) for side, form, _ in seen[name]}
        assert reached >= sides, (name, sides - reached)
    assert {(side, form) for side, form, parts in seen['first'] if not parts} >= sides
    assert {(side, form) for side, form, parts in seen['gram'] if parts} >= sides
    assert {side for side, _, parts in seen['first'] if parts} >= {96, 128, 256}


def make(batch, rows, cols, dtype):
    gen = torch.Generator(device='cuda').manual_seed(rows + cols)
    rank = max(1, min(rows, cols) // 8)

    def normal(*shape):
        return torch.randn(*shape, device='cuda', generator=gen)

    return (torch.bmm(normal(batch, rows, rank), normal(batch, rank, cols)) / rank ** 0.5 +
            0.3 * normal(batch, rows, cols)).to(dtype)


def exact(x, steps, coefficients):
    a, b, c = coefficients
    x = x.double()
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        gram = x @ x.t().contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


def check(x, steps=5, coefficients=DEFAULT):
    """Factors of 22 bits: 2^-22 of X, times a^steps = 485 (1.875^8 = 153): 1.2e-4 in all. An entry takes its part of
    that, spread as noise is: within eight deviations; a rounding of the result is half a step of the entry."""
    got = orthogonalize(x, steps, coefficients)
    half = torch.finfo(x.dtype).eps / 2
    for one, other in zip(x, got):
        tall = one.shape[0] > one.shape[1]
        want = exact(one.t().contiguous() if tall else one, steps, coefficients)
        want = want.t() if tall else want
        off = (other.double() - want).abs()
        size = want.square().mean().sqrt()
        assert (off <= half * (want.abs() + 1e-3 * size) + 1e-3 * size).all(), off.max() / size
        assert off.norm() <= (half + 1.2e-4) * want.norm(), off.norm() / want.norm()


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('batch,rows,cols', CASES)
def test_gpu_cuts(batch, rows, cols, dtype):
    check(make(batch, rows, cols, dtype))


@gpu
@pytest.mark.parametrize('batch,rows,cols', CASES)
def test_gpu_cuts_in_pairs(batch, rows, cols):
    assert _newton_schulz_plan(SLOW, 8, torch.bfloat16, *sorted((rows, cols)))[1] == 3
    check(make(batch, rows, cols, torch.bfloat16), 8, SLOW)
