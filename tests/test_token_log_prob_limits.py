"""Token log probabilities at the ends of what a call may hold."""
import pytest
import torch

from ding.rl_utils import token_log_prob

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize('rows,V,threads', [(2 ** 28 + 70, 2, 16), (2 ** 26 + 37, 66, 64), (2 ** 24 + 5, 513, 256)])
def test_gpu_more_rows_than_a_launch_holds(rows, V, threads):
    """A launch takes fewer than 2^32 threads, `threads` of them a row."""
    assert rows * threads >= 2 ** 32
    gen = torch.Generator(device='cuda').manual_seed(rows % 1000)
    logits = torch.empty(rows, V, dtype=torch.bfloat16, device='cuda').normal_(generator=gen).requires_grad_()
    index = torch.randint(0, V, (rows, ), device='cuda', generator=gen)
    out = token_log_prob(logits, index, entropy=True)
    grad, = torch.autograd.grad([out.log_prob.sum() + out.entropy.sum()], [logits])
    edge = 2 ** 32 // threads
    parts = [slice(at, at + 100) for at in (0, edge - 150, edge - 50, rows - 100)]
    parts += [slice(at, at + 4096) for at in range(4096, rows - 4096, rows // 64)]
    for part in parts:
        x = logits[part].detach().double()
        lp = torch.log_softmax(x, -1)
        p = lp.exp()
        h = -(p * lp).sum(-1, keepdim=True)
        want = torch.zeros_like(x).scatter_(-1, index[part].unsqueeze(-1), 1.0) - p - p * (lp + h)
        # some hundred roundings of 2^-24 of numbers below 16, and the gradient's to 8 bits
        assert (out.log_prob[part] - lp.gather(-1, index[part].unsqueeze(-1)).squeeze(-1)).abs().max() <= 1e-4
        assert (out.entropy[part] - h.squeeze(-1)).abs().max() <= 1e-4
        assert ((grad[part] - want).abs() <= 2.0 ** -8 * want.abs() + 1e-4).all()


@gpu
@pytest.mark.parametrize('rows', [3, 256, 257])
@pytest.mark.parametrize('V,top_k', [(1048577, 32), (1200000, 29)])
def test_gpu_top_of_long_rows(rows, V, top_k):
    """How many largest entries a call may ask for goes by the row's length alone, not by the number of rows."""
    gen = torch.Generator(device='cuda').manual_seed(rows)
    logits = torch.empty(rows, V, dtype=torch.bfloat16, device='cuda').normal_(generator=gen)
    index = torch.randint(0, V, (rows, ), device='cuda', generator=gen)
    out = token_log_prob(logits, index, entropy=True, top_k=top_k)
    for r in (0, rows // 2, rows - 1):
        x = logits[r].cpu()
        order = torch.sort(x.float(), descending=True, stable=True).indices[:top_k]
        lp = torch.log_softmax(x.double(), -1)
        assert torch.equal(out.top_index[r].cpu(), order)
        # a sum of 2^20 terms over 2^10 threads and some hundred roundings of 2^-24 of numbers below 16
        assert (out.top_log_prob[r].cpu() - lp[order]).abs().max() <= 1e-4
        assert abs(out.log_prob[r].item() - lp[index[r].item()].item()) <= 1e-4
        assert abs(out.entropy[r].item() + (lp.exp() * lp).sum().item()) <= 1e-4


@gpu
@pytest.mark.parametrize('rows', [1, 300])
def test_gpu_too_many_top(rows):
    logits = torch.zeros(1, 4194305, dtype=torch.bfloat16, device='cuda').expand(rows, -1)
    index = torch.zeros(rows, dtype=torch.long, device='cuda')
    with pytest.raises(ValueError, match='31'):
        token_log_prob(logits, index, top_k=32)
    assert token_log_prob(logits[:, :4194304], index, top_k=32).top_index[-1].tolist() == list(range(32))


@gpu
@pytest.mark.parametrize('V', [300, 9001])
def test_gpu_one_copy_for_both_directions(V):
    """Logits that need a copy are copied once: the backward pass makes room for the gradient alone."""
    gen = torch.Generator(device='cuda').manual_seed(V)
    index = torch.randint(0, V, (6, 5, 8), device='cuda', generator=gen)
    apart = torch.randn(6, 5, 8, V, 2, device='cuda', generator=gen)[..., 0]
    unfolded = torch.randn(12, 10, 16, V, device='cuda', generator=gen)[::2, ::2, ::2]
    for logits in (apart, unfolded):
        grads = []
        for x in (logits.detach(), logits.contiguous()):
            x.requires_grad_()
            out = token_log_prob(x, index, entropy=True)
            total = out.log_prob.sum() + out.entropy.sum()
            before = torch.cuda.memory_allocated()
            torch.cuda.reset_peak_memory_stats()
            grads.append(torch.autograd.grad(total, x)[0])
            assert torch.cuda.max_memory_allocated() - before < 1.5 * x.numel() * 4
        assert torch.equal(*grads)
