"""Memory-efficient token log-prob extraction for LLM policies.

Parity: reference ding/rl_utils/log_prob_utils.py. ``efficient_method`` avoids
materializing the [B,S,V] log-softmax: logp(a) = logit(a) - logsumexp(logits).
``token_log_prob`` and ``fused_method`` read the logits once on a GPU (HIP
kernels, ding/ops/csrc/token_ops.hip) and keep two numbers per token for the
backward pass instead of [B,S,V] intermediates.
"""
from collections import namedtuple
from typing import Optional

import torch
from torch import Tensor

token_log_prob_output = namedtuple('token_log_prob_output', ['log_prob', 'entropy', 'top_log_prob', 'top_index'])


def naive_method(logits: Tensor, index: Tensor) -> Tensor:
    return torch.log_softmax(logits, dim=-1).gather(-1, index.unsqueeze(-1)).squeeze(-1)


def efficient_method(logits: Tensor, index: Tensor) -> Tensor:
    taken = logits.gather(-1, index.unsqueeze(-1)).squeeze(-1)
    lse = torch.logsumexp(logits, dim=-1)
    return taken - lse


def less_efficient_method(logits: Tensor, index: Tensor) -> Tensor:
    dist = torch.distributions.Categorical(logits=logits)
    return dist.log_prob(index)


def _token_log_prob_torch(logits: Tensor, index: Tensor, temperature: float, ignore_index: Optional[int],
                          entropy: bool, top_k: int):
    live = torch.ones_like(index, dtype=torch.bool) if ignore_index is None else index != ignore_index
    z = logits if logits.dtype == torch.float64 else logits.float()
    z = torch.where(live.unsqueeze(-1), z, torch.zeros((), dtype=z.dtype, device=z.device))
    # the maximum leaves before the temperature divides: a row of the type's lowest value stays finite
    log_p = torch.log_softmax((z - z.detach().amax(-1, keepdim=True)) / temperature, dim=-1)
    token = torch.where(live, index, torch.zeros_like(index)).long().unsqueeze(-1)
    zero = torch.zeros((), dtype=z.dtype, device=z.device)
    log_prob = torch.where(live, log_p.gather(-1, token).squeeze(-1), zero)
    h = top = top_index = None
    if entropy:
        p = log_p.exp()
        h = torch.where(live, -(p * log_p.masked_fill(p == 0, 0.)).sum(-1), zero)
    if top_k:
        top_index = torch.sort(z, dim=-1, descending=True, stable=True).indices[..., :top_k]
        top = torch.where(live.unsqueeze(-1), log_p.gather(-1, top_index), zero)
        top_index = top_index.masked_fill(~live.unsqueeze(-1), -1)
    return log_prob, h, top, top_index


def token_log_prob(
        logits: Tensor,
        index: Tensor,
        temperature: float = 1.0,
        ignore_index: Optional[int] = None,
        entropy: bool = False,
        top_k: int = 0,
) -> token_log_prob_output:
    """
    Overview:
        Log probabilities of given tokens, with the distribution's entropy and its most likely tokens if wanted.
        Differentiable with respect to ``logits`` through ``log_prob``, ``entropy`` and ``top_log_prob`` (once).
    Arguments:
        - logits (:obj:`torch.Tensor`): [..., V] of float32, bfloat16 or float16, of any strides; a copy is \
            made only where the last dimension is not dense, or the leading ones do not fold into two. Entries of \
            ``-inf`` are masked tokens.
        - index (:obj:`torch.Tensor`): [...] of integers, the tokens that were taken.
        - temperature (:obj:`float`): The logits are divided by it; in [1e-30, 1e30].
        - ignore_index (:obj:`Optional[int]`): Rows whose token is this (prompts, padding) are not read: their \
            outputs are 0, their top indexes -1, their gradient 0.
        - entropy (:obj:`bool`): Whether to return the entropy.
        - top_k (:obj:`int`): The number of most likely tokens to return, on a GPU at most 32, and at most 4096 for \
            all of a row's parts of 32768 entries (32 of up to 4194304 entries). Among equal logits the lower index \
            comes first.
    Returns:
        - output (:obj:`namedtuple`): ``log_prob`` [...], ``entropy`` [...], ``top_log_prob`` [..., top_k] in \
            float32 (float64 for float64 logits, which are taken on the CPU only), ``top_index`` [..., top_k] in \
            int64; None for what was not asked for.
    .. note::
        A row that leaves no token (all ``-inf``), or that holds NaN or ``+inf``, gives NaN as ``naive_method`` does.
        A token outside [0, V) raises on the CPU and gives NaN on a GPU.
    """
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., V] with V >= 1, got {tuple(logits.shape)}")
    if index.shape != logits.shape[:-1]:
        raise ValueError(f"index must be {tuple(logits.shape[:-1])} for these logits, got {tuple(index.shape)}")
    if not logits.is_floating_point() or index.is_floating_point() or index.dtype == torch.bool:
        raise TypeError(f"logits must be floating point and index integers, got {logits.dtype} and {index.dtype}")
    if index.device != logits.device:
        raise ValueError(f"index is on {index.device}, logits on {logits.device}")
    if not 1e-30 <= temperature <= 1e30:  # beyond, its inverse leaves the range of 32 bits
        raise ValueError(f"temperature must be in [1e-30, 1e30], got {temperature}")
    if not 0 <= top_k <= logits.shape[-1]:
        raise ValueError(f"top_k must be in [0, {logits.shape[-1]}], got {top_k}")
    from ding.ops import dispatch
    if dispatch.use_hip_autograd(logits):
        if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise TypeError(f"logits on a GPU must be float32, bfloat16 or float16, got {logits.dtype}")
        if top_k > 32:
            raise ValueError(f"top_k must be at most 32 on a GPU, got {top_k}")
        parts = -(-logits.shape[-1] // 32768)
        if parts > 1 and top_k * parts > 4096:
            raise ValueError(f"top_k must be at most {4096 // parts} of {logits.shape[-1]} entries on a GPU, got {top_k}")
        return token_log_prob_output(
            *dispatch.token_log_prob(logits, index, temperature, ignore_index, entropy, top_k)
        )
    return token_log_prob_output(
        *_token_log_prob_torch(logits, index, temperature, ignore_index, entropy, top_k)
    )


def fused_method(logits: Tensor, index: Tensor) -> Tensor:
    """The other methods' signature over ``token_log_prob``; returns float32."""
    return token_log_prob(logits, index).log_prob
