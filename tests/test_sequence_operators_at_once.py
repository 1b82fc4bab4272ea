"""The sequence operators side by side: on two streams at once, in two graphs whose replays take turns, under autocast."""
import pytest
import torch

from ding.rl_utils import token_log_prob
from ding.torch_utils import GatedLinearRNN, Muon, gated_linear_recurrence, orthogonalize

gpu = pytest.mark.gpu


def calls(seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, to=torch.float32):
        return torch.randn(*shape, device='cuda', generator=gen).to(to)

    packed = normal(3000, 3, 2 * 333, to=torch.float16)
    matrices = [normal(700, 900), normal(900, 700, to=torch.bfloat16), normal(17, 100, 200)]
    logits = normal(300, 40001, to=torch.bfloat16)
    index = torch.randint(0, 40001, (300, ), device='cuda', generator=gen)

    def run():
        x, f = packed[..., :333].detach().requires_grad_(), packed[..., 333:].detach().requires_grad_()
        h, last = gated_linear_recurrence(x, f)
        out = [h, last, *torch.autograd.grad([h, last], [x, f], [torch.ones_like(h), torch.ones_like(last)])]
        out += [orthogonalize(m) for m in matrices]
        leaf = logits.detach().requires_grad_()
        got = token_log_prob(leaf, index, entropy=True, top_k=5)
        grads = [torch.ones_like(got.log_prob), torch.ones_like(got.entropy)]
        return out + list(got) + list(torch.autograd.grad([got.log_prob, got.entropy], [leaf], grads))

    return run


@gpu
def test_two_streams_at_once():
    runs = [calls(seed) for seed in range(2)]
    alone = [run() for run in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for run, stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                got.append(run())
        torch.cuda.synchronize()
        for one, other in zip(alone, got):
            for a, b in zip(one, other):
                assert torch.equal(a.detach(), b.detach())


@gpu
def test_two_graphs_in_turns():
    runs = [calls(seed) for seed in range(2)]
    alone = [[v.detach().clone() for v in run()] for run in runs]
    graphs, kept = [], []
    for run in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept.append([v.detach() for v in run()])
        graphs.append(graph)
    for turn in range(4):
        for at in ((0, 1), (1, 0))[turn % 2]:
            graphs[at].replay()
            torch.cuda.synchronize()
            for a, b in zip(alone[at], kept[at]):
                assert torch.equal(a, b)
        runs[0]()


def train(device, low):
    torch.manual_seed(0)
    core, head = GatedLinearRNN(12, 24, 2).to(device), torch.nn.Linear(24, 70).to(device)
    params = list(core.parameters()) + list(head.parameters())
    x, index = torch.randn(9, 4, 12).to(device), torch.randint(0, 70, (9, 4)).to(device)
    state = None
    for _ in range(2):  # the second unroll starts from the first one's states
        with torch.autocast(device, dtype=torch.bfloat16, enabled=low):
            out, state = core(x, state)
            got = token_log_prob(head(out), index, entropy=True)
    grads = torch.autograd.grad(-(got.log_prob + 0.1 * got.entropy).mean(), params)
    assert state[0]['h'].dtype == torch.float32
    for p, g in zip(params, grads):
        assert g.dtype == p.dtype
        p.grad = g
    Muon(params).step()
    assert all(torch.isfinite(p).all() for p in params)
    return [g.cpu().double() for g in grads]


def check_autocast(device):
    """Some ten roundings to 8 bits lie between an input and a gradient: 10 * 2^-8 of its norm."""
    for low, whole in zip(train(device, True), train('cpu', False)):
        assert (low - whole).norm() <= 0.04 * whole.norm()


def test_autocast_cpu():
    check_autocast('cpu')


@gpu
def test_autocast_gpu():
    check_autocast('cuda')
