"""Optimizers with integrated gradient clip/ignore, PCGrad, and the
orthogonalised update of weight matrices (orthogonalize, Muon).

Parity: reference ding/torch_utils/optimizer_helper.py (Adam:107,
RMSprop:395, PCGrad:650, grad monitoring helpers).

Clip semantics (matching the reference's option set):
  grad_clip_type in {None, 'clip_value', 'clip_norm', 'clip_momentum_norm',
  'ignore_value', 'ignore_norm'} — clip_* rescales gradients, ignore_*
  zeroes the whole step when the threshold trips.
"""
import math
from functools import lru_cache
from typing import Iterable, List, Optional, Tuple, Union

import torch
import torch.nn as nn

inf = math.inf


def calculate_grad_norm(model: torch.nn.Module, norm_type: int = 2) -> float:
    grads = [p.grad for p in model.parameters() if p.grad is not None]
    if not grads:
        return 0.0
    return torch.norm(torch.stack([torch.norm(g.detach(), norm_type) for g in grads]), norm_type).item()


def calculate_grad_norm_without_bias_two_norm(model: torch.nn.Module) -> float:
    grads = [p.grad for n, p in model.named_parameters() if p.grad is not None and "bias" not in n]
    if not grads:
        return 0.0
    return torch.norm(torch.stack([torch.norm(g.detach(), 2) for g in grads]), 2).item()


def grad_ignore_norm(parameters, max_norm: float, norm_type: float = 2.0) -> float:
    """Zero all grads when total norm exceeds max_norm."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    parameters = [p for p in parameters if p.grad is not None]
    if not parameters:
        return 0.0
    total = torch.norm(torch.stack([torch.norm(p.grad.detach(), norm_type) for p in parameters]), norm_type)
    if total > max_norm:
        for p in parameters:
            p.grad.zero_()
    return float(total)


def grad_ignore_value(parameters, clip_value: float) -> None:
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    parameters = [p for p in parameters if p.grad is not None]
    flag = any(p.grad.detach().abs().max() > clip_value for p in parameters)
    if flag:
        for p in parameters:
            p.grad.zero_()


class Adam(torch.optim.Adam):
    """torch Adam + built-in gradient clip/ignore executed in step()."""

    def __init__(
        self,
        params: Iterable,
        lr: float = 1e-3,
        betas=(0.9, 0.999),
        eps: float = 1e-8,
        weight_decay: float = 0,
        amsgrad: bool = False,
        optim_type: str = 'adam',
        grad_clip_type: Optional[str] = None,
        clip_value: Optional[float] = None,
        clip_coef: float = 5,
        clip_norm_type: float = 2.0,
        clip_momentum_timestep: int = 100,
        ignore_value: Optional[float] = None,
        ignore_coef: float = 5,
        ignore_norm_type: float = 2.0,
        ignore_momentum_timestep: int = 100,
        capturable: bool = False,
        flatten_grads: bool = False,
    ):
        self._grad_clip_type = grad_clip_type
        self._clip_value = clip_value
        self._clip_norm_type = clip_norm_type
        self._clip_coef = clip_coef
        self._ignore_value = ignore_value
        self._ignore_norm_type = ignore_norm_type
        self._ignore_coef = ignore_coef
        self._clip_momentum_timestep = clip_momentum_timestep
        self._ignore_momentum_timestep = ignore_momentum_timestep
        # capturable=True keeps Adam's step counters on-device so the whole
        # optimizer update can live inside a hipGraph capture (MI355X:
        # removes ~30 launches + host work per replayed minibatch)
        params = list(params)
        leaves = [p for p in params if isinstance(p, torch.Tensor)]
        # fused Adam: ONE multi-tensor kernel per step instead of the foreach
        # chain — rocprof on the PPO bench showed the eager optimizer
        # (multi_tensor_apply + fills + adds) at ~27 ms/step of the 180 ms
        # step. GPU-resident float params only; DING_FUSED_ADAM=0 disables.
        import os as _os
        use_fused = (
            _os.environ.get('DING_FUSED_ADAM', '1') not in ('0', 'false') and not capturable
            and len(leaves) == len(params) and len(leaves) > 0
            and all(p.is_cuda and p.dtype in (torch.float32, torch.float16, torch.bfloat16) for p in leaves)
        )
        super().__init__(
            params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, amsgrad=amsgrad,
            capturable=capturable, foreach=(True if capturable else None) if not use_fused else None,
            fused=use_fused or None,
        )
        if grad_clip_type in ('clip_momentum_norm', 'ignore_momentum_norm'):
            for group in self.param_groups:
                group.setdefault('step_count', 0)
                group['grad_norm_ema'] = None
        # flat gradient buffer: every param.grad becomes a view into ONE
        # contiguous tensor, so grad-clip is 1 norm + 1 scale kernel and
        # zero_grad is 1 fill — rocprof showed the per-param reduce/fill
        # storm at ~25 ms/step on the PPO bench. Views have stable addresses,
        # which also makes backward hipGraph-capture friendly.
        self._flat_grad_buf = None
        if flatten_grads and leaves and all(p.is_cuda for p in leaves):
            total = sum(p.numel() for p in leaves)
            buf = torch.zeros(total, device=leaves[0].device, dtype=leaves[0].dtype)
            off = 0
            for p in leaves:
                p.grad = buf[off:off + p.numel()].view_as(p)
                off += p.numel()
            self._flat_grad_buf = buf

    def _params(self) -> List[torch.Tensor]:
        return [p for group in self.param_groups for p in group['params']]

    def _apply_clip(self):
        t = self._grad_clip_type
        if t is None:
            return
        params = self._params()
        if t == 'clip_norm' and self._flat_grad_buf is not None:
            buf = self._flat_grad_buf
            total_norm = torch.linalg.vector_norm(buf, self._clip_norm_type)
            scale = (self._clip_value / (total_norm + 1e-6)).clamp(max=1.0)
            buf.mul_(scale)
            return
        if t == 'clip_value':
            nn.utils.clip_grad_value_(params, self._clip_value)
        elif t == 'clip_norm':
            # foreach=True: one fused norm + scale instead of a reduce per param
            _fe = True if (params and all(p.is_cuda for p in params)) else None
            nn.utils.clip_grad_norm_(params, self._clip_value, self._clip_norm_type, foreach=_fe)
        elif t == 'ignore_value':
            grad_ignore_value(params, self._ignore_value)
        elif t == 'ignore_norm':
            grad_ignore_norm(params, self._ignore_value, self._ignore_norm_type)
        elif t in ('clip_momentum_norm', 'ignore_momentum_norm'):
            # threshold = coef * EMA of historical grad norms
            for group in self.param_groups:
                ps = [p for p in group['params'] if p.grad is not None]
                if not ps:
                    continue
                norm = torch.norm(
                    torch.stack([torch.norm(p.grad.detach(), self._clip_norm_type) for p in ps]),
                    self._clip_norm_type
                ).item()
                ema = group.get('grad_norm_ema')
                ema = norm if ema is None else 0.99 * ema + 0.01 * norm
                group['grad_norm_ema'] = ema
                group['step_count'] = group.get('step_count', 0) + 1
                if group['step_count'] >= self._clip_momentum_timestep:
                    coef = self._clip_coef if t == 'clip_momentum_norm' else self._ignore_coef
                    threshold = coef * ema
                    if norm > threshold:
                        if t == 'clip_momentum_norm':
                            scale = threshold / (norm + 1e-6)
                            for p in ps:
                                p.grad.mul_(scale)
                        else:
                            for p in ps:
                                p.grad.zero_()
        else:
            raise KeyError(f"unknown grad_clip_type {t}")

    def step(self, closure=None):
        self._apply_clip()
        return super().step(closure)

    def zero_grad(self, set_to_none: bool = True):
        if self._flat_grad_buf is not None:
            # keep the grad views alive: one fill over the flat buffer
            self._flat_grad_buf.zero_()
            return
        return super().zero_grad(set_to_none)

    def get_grad(self) -> float:
        return calculate_grad_norm_without_bias_two_norm(_FakeModel(self._params()))


class _FakeModel:

    def __init__(self, params):
        self._p = params

    def named_parameters(self):
        return [(f"p{i}", p) for i, p in enumerate(self._p)]

    def parameters(self):
        return self._p


class RMSprop(torch.optim.RMSprop):
    """torch RMSprop + built-in gradient clip/ignore."""

    def __init__(
        self,
        params: Iterable,
        lr: float = 1e-2,
        alpha: float = 0.99,
        eps: float = 1e-8,
        weight_decay: float = 0,
        momentum: float = 0,
        centered: bool = False,
        grad_clip_type: Optional[str] = None,
        clip_value: Optional[float] = None,
        clip_norm_type: float = 2.0,
        ignore_value: Optional[float] = None,
        ignore_norm_type: float = 2.0,
    ):
        self._grad_clip_type = grad_clip_type
        self._clip_value = clip_value
        self._clip_norm_type = clip_norm_type
        self._ignore_value = ignore_value
        self._ignore_norm_type = ignore_norm_type
        super().__init__(
            params, lr=lr, alpha=alpha, eps=eps, weight_decay=weight_decay, momentum=momentum, centered=centered
        )

    def _params(self):
        return [p for group in self.param_groups for p in group['params']]

    def step(self, closure=None):
        t = self._grad_clip_type
        params = self._params()
        if t == 'clip_value':
            nn.utils.clip_grad_value_(params, self._clip_value)
        elif t == 'clip_norm':
            # foreach=True: one fused norm + scale instead of a reduce per param
            _fe = True if (params and all(p.is_cuda for p in params)) else None
            nn.utils.clip_grad_norm_(params, self._clip_value, self._clip_norm_type, foreach=_fe)
        elif t == 'ignore_value':
            grad_ignore_value(params, self._ignore_value)
        elif t == 'ignore_norm':
            grad_ignore_norm(params, self._ignore_value, self._ignore_norm_type)
        return super().step(closure)


@lru_cache(maxsize=256)
def _newton_schulz_plan(coefficients: Tuple[float, float, float], steps: int, dtype: torch.dtype, m: int, n: int):
    """How the kernels run the iteration on an m x n matrix (m <= n): the scales and the span of ``newton_schulz``.

    The scales are powers of two that bring X, G = X X^T, b G + c G G, Q = a + b G + c G G and a product of Qs near the
    top of half precision without passing it: no entry of a matrix is larger than its largest singular value, and those
    follow s -> s q(s^2), q(u) = a + b u + c u^2 from [0, 1]. The largest value over the range so far lies at an end or
    where the derivative vanishes.

    The span: running on G needs 3 m^2 n + (4 span - 3) m^3 flops a span, running on X 3 m^2 n + m^3 a step. But an error of
    G, 2^-22 of its largest entry, grows by max(q)^2 a step where one of X grows by max(q), and where one direction
    dominates, the others are as small as errors of G soon become. Each step on G after the first of a span so costs a
    factor of max(q) in precision, and a span may cost 4 for results of 16 bits: two steps with the usual coefficients.
    Matrices of a mean component plus 1e-3 to 1e-2 of noise (200 x 260 to 4096 x 8192) are then 1e-5 to 6e-4 off before
    the result's rounding, no more than with library products in 32 bits, but for few; spans of three steps were up to
    1.5e-3 off, of five 0.3% to 100%. float32 has no room for it.
    """
    a, b, c = coefficients
    top, most_x, most_b, qs = 1.001, 1.001, 0.0, []
    for _ in range(steps):
        ends = [top ** 2]
        inner = ends + ([-b / (2 * c)] if c != 0 and 0 < -b / (2 * c) < top ** 2 else [])
        most_b = max([most_b] + [abs(b * u + c * u * u) for u in inner])
        qs.append(max([abs(a)] + [abs(a + b * u + c * u * u) for u in inner]))
        root = 9 * b * b - 20 * a * c
        for sign in (-1, 1):
            u = (-3 * b + sign * math.sqrt(max(root, 0.0))) / (10 * c) if c != 0 else (-a / (3 * b) if b else 0.0)
            if root >= 0 and 0 < u < top ** 2:
                ends.append(u)
        top = 1.001 * max(abs(math.sqrt(u) * (a + b * u + c * u * u)) for u in ends)
        if not top < 64:
            raise ValueError(f"coefficients {coefficients} let singular values grow without bound in {steps} steps")
        most_x = max(most_x, top)
    span, room = 0, 4.0 if dtype in (torch.bfloat16, torch.float16) else 0.0
    least = steps * (3 * n + m)
    for count in range(2, steps + 1):
        counts = [min(count, steps - at) for at in range(0, steps, count)]
        flops = sum(3 * n + (4 * k - 3) * m for k in counts)
        if max(qs) ** (count - 1) <= room and flops < least:
            least, span = flops, count
    most_p = max(math.prod(qs[at:at + span]) for at in range(0, steps, span)) if span else 1.0
    bounds = (most_x, most_x ** 2, most_b, max(qs), most_p)
    return tuple(2.0 ** math.floor(math.log2(32768 / max(v, 2.0 ** -10))) for v in bounds), span


def _orthogonalize_torch(x: torch.Tensor, steps: int, coefficients: Tuple[float, float, float], eps: float):
    a, b, c = coefficients
    dtype, tall = x.dtype, x.shape[-2] > x.shape[-1]
    x = x.transpose(-2, -1) if tall else x
    x = x.to(torch.float64 if dtype == torch.float64 else torch.float32).contiguous()
    # the norm in 64 bits: squares of 32-bit numbers overflow and vanish
    x = (x / (x.double().square().sum((-2, -1), keepdim=True).sqrt() + eps)).to(x.dtype)
    for _ in range(steps):
        gram = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return (x.transpose(-2, -1) if tall else x).to(dtype).contiguous()


@torch.no_grad()
def orthogonalize(
        matrix: torch.Tensor,
        steps: int = 5,
        coefficients: Tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
        eps: float = 1e-7,
) -> torch.Tensor:
    """
    Overview:
        Moves the singular values of a matrix towards 1 and leaves its singular vectors: Newton-Schulz steps
        ``X <- a X + (b X X^T + c (X X^T)^2) X`` from ``X = matrix / (|matrix|_F + eps)``. The default coefficients
        bring singular values of more than about 1/300 of the norm into [0.7, 1.2] in five steps. On a GPU the
        products run on the matrix units to 22 bits (HIP kernels, ding/ops/csrc/ortho_ops.hip). Not differentiable.
    Arguments:
        - matrix (:obj:`torch.Tensor`): [..., m, n] of float32, bfloat16 or float16, any strides; a batch is \
            orthogonalised together, which is faster than one matrix after the other. On a GPU sides are at most \
            2^20 and matrices fewer than 32768.
        - steps (:obj:`int`): Number of steps, at least 1.
        - coefficients (:obj:`Tuple[float, float, float]`): a, b and c.
        - eps (:obj:`float`): Is added to the norm: a zero matrix gives zeros. On a GPU entries are held to about \
            1e-11 of the normalised matrix, so one whose norm is far below ``eps`` loses its digits.
    Returns:
        - update (:obj:`torch.Tensor`): [..., m, n], a new dense tensor of the same type.
    """
    if matrix.dim() < 2 or not matrix.is_floating_point():
        raise ValueError(f"matrix must be floating point [..., m, n], got {tuple(matrix.shape)} of {matrix.dtype}")
    if steps < 1:
        raise ValueError(f"steps must be at least 1, got {steps}")
    if not eps > 0:
        raise ValueError(f"eps must be positive, got {eps}")
    coefficients = tuple(float(v) for v in coefficients)
    if len(coefficients) != 3 or not all(math.isfinite(v) for v in coefficients):
        raise ValueError(f"coefficients must be three finite numbers, got {coefficients}")
    plan = _newton_schulz_plan(coefficients, int(steps), matrix.dtype, *sorted(matrix.shape[-2:]))
    from ding.ops import dispatch
    if not dispatch.use_hip_autograd(matrix):
        return _orthogonalize_torch(matrix, steps, coefficients, eps)
    if matrix.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"matrix on a GPU must be float32, bfloat16 or float16, got {matrix.dtype}")
    flat = matrix.reshape(-1, *matrix.shape[-2:]) if matrix.numel() else matrix.new_empty(0, 1, 1)
    return dispatch.newton_schulz(flat, int(steps), coefficients, float(eps), *plan).view(matrix.shape)


class Muon(torch.optim.Optimizer):
    """Momentum whose update of a weight matrix is orthogonalised, with the same gradient clip/ignore as ``RMSprop``.

    A parameter of two or more dimensions is taken as the matrix [shape[0], rest]. Its update is
    ``orthogonalize(g + momentum * buf)`` times 0.2 sqrt(max(rows, cols)), which has the root mean square of a usual
    Adam step, so a learning rate tuned for Adam fits. Other parameters, and groups with ``use_adam=True`` (embeddings,
    output heads), take Adam steps with the same learning rate. Matrices of one shape are orthogonalised together.
    Weight decay is decoupled. Momentum and Adam states are 32 bit whatever the parameter's type; nothing is read back
    to the host, so a step can be captured into a graph unless an ``ignore_*`` clip is chosen.
    """

    def __init__(
        self,
        params: Iterable,
        lr: float = 1e-3,
        momentum: float = 0.95,
        nesterov: bool = True,
        weight_decay: float = 0,
        ns_steps: int = 5,
        ns_coefficients: Tuple[float, float, float] = (3.4445, -4.7750, 2.0315),
        ns_eps: float = 1e-7,
        betas: Tuple[float, float] = (0.9, 0.999),
        eps: float = 1e-8,
        use_adam: bool = False,
        grad_clip_type: Optional[str] = None,
        clip_value: Optional[float] = None,
        clip_norm_type: float = 2.0,
        ignore_value: Optional[float] = None,
        ignore_norm_type: float = 2.0,
    ):
        if not 0 <= momentum < 1:
            raise ValueError(f"momentum must be in [0, 1), got {momentum}")
        if lr < 0 or weight_decay < 0:
            raise ValueError(f"lr and weight_decay must not be negative, got {lr} and {weight_decay}")
        if grad_clip_type not in (None, 'clip_value', 'clip_norm', 'ignore_value', 'ignore_norm'):
            raise KeyError(f"unknown grad_clip_type {grad_clip_type}")
        self._grad_clip_type = grad_clip_type
        self._clip_value = clip_value
        self._clip_norm_type = clip_norm_type
        self._ignore_value = ignore_value
        self._ignore_norm_type = ignore_norm_type
        super().__init__(
            params,
            dict(
                lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, ns_steps=ns_steps,
                ns_coefficients=ns_coefficients, ns_eps=ns_eps, betas=betas, eps=eps, use_adam=use_adam
            )
        )

    def _params(self):
        return [p for group in self.param_groups for p in group['params']]

    def _apply_clip(self):
        t = self._grad_clip_type
        params = self._params()
        if t == 'clip_value':
            nn.utils.clip_grad_value_(params, self._clip_value)
        elif t == 'clip_norm':
            _fe = True if (params and all(p.is_cuda for p in params)) else None
            nn.utils.clip_grad_norm_(params, self._clip_value, self._clip_norm_type, foreach=_fe)
        elif t == 'ignore_value':
            grad_ignore_value(params, self._ignore_value)
        elif t == 'ignore_norm':
            grad_ignore_norm(params, self._ignore_value, self._ignore_norm_type)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._apply_clip()
        for group in self.param_groups:
            params = [p for p in group['params'] if p.grad is not None]
            if not params:
                continue
            if group['weight_decay'] != 0:
                torch._foreach_mul_(params, 1 - group['lr'] * group['weight_decay'])
            alike = {}
            for p in params:
                matrix = p.dim() >= 2 and not group['use_adam']
                shape = (p.shape[0], p.numel() // p.shape[0]) if matrix and p.numel() else None
                alike.setdefault((shape, p.dtype, p.device), []).append(p)
            for (shape, _, _), same in alike.items():
                if shape is None:
                    self._adam(group, same)
                else:
                    self._orthogonal(group, same, shape)
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        super().load_state_dict(state_dict)
        # torch casts states to their parameter's type; they are taken again in the 32 bits they were kept in
        ids = [i for group in state_dict['param_groups'] for i in group['params']]
        for i, p in zip(ids, self._params()):
            for key, value in state_dict['state'].get(i, {}).items():
                self.state[p][key] = value.detach().to(device=p.device, dtype=torch.float32, copy=True)

    def _orthogonal(self, group: dict, params: List[torch.Tensor], shape: Tuple[int, int]) -> None:
        for p in params:
            if 'momentum_buffer' not in self.state[p]:
                self.state[p]['momentum_buffer'] = torch.zeros_like(p, dtype=torch.float32)
        bufs = [self.state[p]['momentum_buffer'] for p in params]
        grads = [p.grad.float() for p in params]
        torch._foreach_mul_(bufs, group['momentum'])
        torch._foreach_add_(bufs, grads)
        updates = torch._foreach_add(grads, bufs, alpha=group['momentum']) if group['nesterov'] else bufs
        # In 32 bits also for weights of 16: a step multiplies the small singular values by up to 485, and with them what a
        # rounding of the momentum would put among them (momentum of a mean and 1% of noise: the step 46% off in bfloat16).
        stacked = torch.stack([u.reshape(shape) for u in updates])
        stacked = stacked.double() if params[0].dtype == torch.float64 else stacked
        update = orthogonalize(stacked, group['ns_steps'], group['ns_coefficients'], group['ns_eps'])
        step = group['lr'] * 0.2 * math.sqrt(max(shape))
        torch._foreach_add_(params, [u.view(p.shape) for u, p in zip(update.unbind(0), params)], alpha=-step)

    def _adam(self, group: dict, params: List[torch.Tensor]) -> None:
        beta1, beta2 = group['betas']
        for p in params:
            state = self.state[p]
            if 'step' not in state:
                state['step'] = torch.zeros((), dtype=torch.float32, device=p.device)
                state['exp_avg'] = torch.zeros_like(p, dtype=torch.float32)
                state['exp_avg_sq'] = torch.zeros_like(p, dtype=torch.float32)
        steps, first, second = ([self.state[p][k] for p in params] for k in ('step', 'exp_avg', 'exp_avg_sq'))
        grads = [p.grad.float() for p in params]
        torch._foreach_add_(steps, 1)
        torch._foreach_lerp_(first, grads, 1 - beta1)
        torch._foreach_mul_(second, beta2)
        torch._foreach_addcmul_(second, grads, grads, 1 - beta2)
        for p, n, m, v in zip(params, steps, first, second):
            scale = group['lr'] / (1 - beta1 ** n)
            p.sub_((scale * m / ((v / (1 - beta2 ** n)).sqrt() + group['eps'])).to(p.dtype))

    def get_grad(self) -> float:
        return calculate_grad_norm_without_bias_two_norm(_FakeModel(self._params()))


class PCGrad:
    """Projecting Conflicting Gradients (NeurIPS 2020) wrapper for multi-task
    losses. Parity: reference optimizer_helper.py:650."""

    def __init__(self, optimizer: torch.optim.Optimizer, reduction: str = 'mean'):
        self._optim = optimizer
        assert reduction in ('mean', 'sum')
        self._reduction = reduction

    @property
    def optimizer(self):
        return self._optim

    def zero_grad(self):
        self._optim.zero_grad(set_to_none=False)

    def step(self):
        self._optim.step()

    def pc_backward(self, objectives: List[torch.Tensor]):
        grads, shapes, has_grads = [], [], []
        for obj in objectives:
            self._optim.zero_grad(set_to_none=False)
            obj.backward(retain_graph=True)
            grad, shape, has_grad = self._retrieve_grad()
            grads.append(self._flatten(grad))
            has_grads.append(self._flatten(has_grad))
            shapes.append(shape)
        pc_grad = self._project_conflicting(grads, has_grads)
        pc_grad = self._unflatten(pc_grad, shapes[0])
        self._set_grad(pc_grad)

    def _project_conflicting(self, grads, has_grads):
        import copy
        import random
        shared = torch.stack(has_grads).prod(0).bool()
        pc_grad = [g.clone() for g in grads]
        for g_i in pc_grad:
            others = list(grads)
            random.shuffle(others)
            for g_j in others:
                dot = torch.dot(g_i, g_j)
                if dot < 0:
                    g_i -= dot * g_j / (g_j.norm() ** 2 + 1e-12)
        merged = torch.zeros_like(grads[0])
        stacked = torch.stack(pc_grad)
        if self._reduction == 'mean':
            merged[shared] = stacked[:, shared].mean(dim=0)
        else:
            merged[shared] = stacked[:, shared].sum(dim=0)
        merged[~shared] = stacked[:, ~shared].sum(dim=0)
        return merged

    def _retrieve_grad(self):
        grad, shape, has_grad = [], [], []
        for group in self._optim.param_groups:
            for p in group['params']:
                shape.append(p.shape)
                if p.grad is None:
                    grad.append(torch.zeros_like(p))
                    has_grad.append(torch.zeros_like(p))
                else:
                    grad.append(p.grad.clone())
                    has_grad.append(torch.ones_like(p))
        return grad, shape, has_grad

    @staticmethod
    def _flatten(grads):
        return torch.cat([g.reshape(-1) for g in grads])

    @staticmethod
    def _unflatten(flat, shapes):
        out, idx = [], 0
        for s in shapes:
            n = int(torch.tensor(s).prod().item()) if len(s) else 1
            out.append(flat[idx:idx + n].reshape(s))
            idx += n
        return out

    def _set_grad(self, grads):
        i = 0
        for group in self._optim.param_groups:
            for p in group['params']:
                p.grad = grads[i]
                i += 1


def configure_weight_decay(model: nn.Module, weight_decay: float) -> List[dict]:
    """Split params into decay (matmul weights) / no-decay (bias, norm, emb)."""
    decay, no_decay = [], []
    for name, p in model.named_parameters():
        if not p.requires_grad:
            continue
        if p.dim() <= 1 or name.endswith("bias") or "norm" in name.lower() or "embedding" in name.lower():
            no_decay.append(p)
        else:
            decay.append(p)
    return [
        {"params": decay, "weight_decay": weight_decay},
        {"params": no_decay, "weight_decay": 0.0},
    ]
