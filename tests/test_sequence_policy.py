"""A learner's step of a token policy with the recurrence, the token log probabilities and the orthogonalised update
together, against the same step from elementary operations in 64 bits."""
import math

import pytest
import torch
import torch.nn as nn

from ding.rl_utils import token_log_prob, grpo_policy_data, grpo_policy_error, fused_method
from ding.torch_utils import get_lstm, Muon

gpu = pytest.mark.gpu


class Policy(nn.Module):

    def __init__(self, vocab: int, width: int, layers: int = 2):
        super().__init__()
        self.embed = nn.Embedding(vocab, width)
        self.core = get_lstm('glr', width, width, num_layers=layers)
        self.head = nn.Linear(width, vocab)

    def forward(self, tokens, prev_state=None, reset=None):
        """tokens [B, T] -> logits [B, T, V], next_state"""
        h, state = self.core(self.embed(tokens.t()), prev_state, reset=None if reset is None else reset.t())
        return self.head(h).transpose(0, 1), state


def batch(B, T, vocab, device, seed=0):
    gen = torch.Generator().manual_seed(seed)
    tokens = torch.randint(0, vocab, (B, T + 1), generator=gen)
    labels = tokens[:, 1:].clone()
    lengths = torch.randint(1, T + 1, (B, ), generator=gen)
    lengths[0] = T
    labels[torch.arange(T)[None] >= lengths[:, None]] = -100  # padding
    reset = torch.rand(B, T, generator=gen) < 0.05
    return [v.to(device) for v in (tokens, labels, reset, torch.randn(B, generator=gen))]


def plain_loss(policy, tokens, labels, reset, adv):
    """The same loss from elementary operations on 64-bit copies of the parameters."""
    P = {k: v.detach().double().cpu().requires_grad_() for k, v in policy.named_parameters()}
    tokens, labels, reset, adv = (v.cpu() for v in (tokens, labels, reset, adv.double()))
    x = P['embed.weight'][tokens[:, :-1]]
    for i in range(policy.core.num_layers):
        value, gate = (x @ P[f'core.project.{i}.weight'].t() + P[f'core.project.{i}.bias']).chunk(2, dim=-1)
        a, h, out = torch.sigmoid(gate), torch.zeros_like(value[:, 0]), []
        for t in range(x.shape[1]):
            h = torch.where(reset[:, t, None], torch.zeros_like(h), h)
            h = a[:, t] * h + (1 - a[:, t]) * value[:, t]
            out.append(h)
        x = torch.stack(out, 1) if i == 0 else x + torch.stack(out, 1)
    logp = torch.log_softmax(x @ P['head.weight'].t() + P['head.bias'], -1)
    live = labels != -100
    taken = logp.gather(-1, labels.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    entropy = -(logp.exp() * logp).sum(-1)
    loss = -((adv[:, None] * taken + 0.01 * entropy) * live).sum() / live.sum()
    return loss, torch.autograd.grad(loss, list(P.values()))


def fused_loss(policy, tokens, labels, reset, adv):
    logits, _ = policy(tokens[:, :-1], reset=reset)
    out = token_log_prob(logits, labels, ignore_index=-100, entropy=True)
    return -(adv[:, None] * out.log_prob + 0.01 * out.entropy).sum() / (labels != -100).sum()


def run(device, B, T, vocab, width):
    torch.manual_seed(0)
    policy = Policy(vocab, width).to(device)
    matrices = [p for n, p in policy.named_parameters() if n.startswith('core') and p.dim() == 2]
    others = [p for n, p in policy.named_parameters() if not (n.startswith('core') and p.dim() == 2)]
    opt = Muon([dict(params=matrices), dict(params=others, use_adam=True)], lr=1e-2, grad_clip_type='clip_norm',
               clip_value=1.0)
    for step in range(3):
        data = batch(B, T, vocab, device, seed=step)
        loss = fused_loss(policy, *data)
        opt.zero_grad()
        loss.backward()
        want, grads = plain_loss(policy, *data)
        # 32-bit products of up to `width` terms, a recurrence and a softmax: some hundred roundings of 2^-24
        assert abs(loss.item() - want.item()) <= 1e-4 * max(1.0, abs(want.item()))
        for (name, p), g in zip(policy.named_parameters(), grads):
            assert (p.grad.cpu().double() - g).norm() <= 1e-4 * g.norm() + 1e-7, name
        before = [p.detach().clone() for p in matrices]
        opt.step()
        for p, b in zip(matrices, before):
            # the step has singular values of 0.2 sqrt(max(m, n)) lr times 0.68 to 1.2, but for small ones
            s = torch.linalg.svdvals((p.detach() - b).cpu().double()) / (1e-2 * 0.2 * math.sqrt(max(p.shape)))
            assert s.max() < 1.3 and s[0] > 0.5
    # one token at a time, as a collector decodes, is the same policy
    tokens = batch(B, 6, vocab, device)[0][:, :6]
    with torch.no_grad():
        whole, _ = policy(tokens)
        state, parts = None, []
        for t in range(6):
            logits, state = policy(tokens[:, t:t + 1], state)
            parts.append(logits)
            top = token_log_prob(logits[:, -1], tokens[:, t], top_k=3)
            assert top.top_index.shape == (B, 3) and (top.top_log_prob[:, 0] >= top.log_prob - 1e-6).all()
    assert torch.allclose(whole, torch.cat(parts, 1), atol=1e-4)


def test_learner_step_cpu():
    run('cpu', 3, 12, 31, 16)


@gpu
@pytest.mark.parametrize('B,T,vocab,width', [(3, 12, 31, 16), (4, 150, 700, 64), (2, 300, 9000, 40)])
def test_learner_step_gpu(B, T, vocab, width):
    run('cuda', B, T, vocab, width)


@gpu
def test_group_loss_gpu():
    torch.manual_seed(0)
    policy, reference = Policy(900, 32).cuda(), Policy(900, 32).cuda()
    tokens, labels, reset, adv = batch(4, 40, 900, 'cuda')
    labels, weight = labels.clamp(min=0), (labels != -100).float()
    opt = Muon(policy.parameters(), lr=1e-3)
    for _ in range(2):
        logits, _ = policy(tokens[:, :-1], reset=reset)
        with torch.no_grad():
            ref, _ = reference(tokens[:, :-1], reset=reset)
        loss, info = grpo_policy_error(
            grpo_policy_data(logits, logits.detach(), ref, labels, adv, weight), log_prob_fn=fused_method
        )
        opt.zero_grad()
        loss.policy_loss.backward()
        opt.step()
        assert math.isfinite(info.approx_kl)
    assert all(torch.isfinite(p).all() for p in policy.parameters())


@gpu
def test_learner_step_in_a_graph():
    torch.manual_seed(0)
    policies = [Policy(300, 32).cuda() for _ in range(2)]
    policies[1].load_state_dict(policies[0].state_dict())
    opts = [Muon(p.parameters(), lr=1e-3) for p in policies]
    data = batch(3, 140, 300, 'cuda')

    def step(policy, opt):
        loss = fused_loss(policy, *data)
        grads = torch.autograd.grad(loss, list(policy.parameters()))
        for p, g in zip(policy.parameters(), grads):
            p.grad = g
        opt.step()
        return loss

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for policy, opt in zip(policies, opts):
            step(policy, opt)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step(policies[1], opts[1])
    for seed in range(3):
        for to, new in zip(data, batch(3, 140, 300, 'cuda', seed=seed + 7)):
            to.copy_(new)
        loss = step(policies[0], opts[0])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(loss, kept, atol=1e-5)
        for p, q in zip(policies[0].parameters(), policies[1].parameters()):
            assert torch.allclose(p, q, atol=1e-5)
