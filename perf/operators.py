"""Cases for timing the sequence-policy operators: token log probabilities, the gated linear recurrence and the
orthogonalised update.

The three make up what a learner's step of a token or sequence policy does besides its projections: a recurrent core
over (padded, concatenated) trajectories, the log probability / entropy head over a vocabulary or an action set with its
gradient, and the update of the weight matrices. ``own`` chooses between the plain form (elementary torch operations in
32 bits) and the framework's entry points (``ding.rl_utils.token_log_prob``, ``ding.torch_utils.gated_linear_recurrence``,
``ding.torch_utils.orthogonalize``).
"""
import math

import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
IGNORE = -100
NS_COEFFICIENTS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
# the dearest listed case of each operator, which no drawn one passes
MOST_LOGITS = 8 * 2048 * 131072
MOST_STATES = 32768 * 2 * 2048
MOST_PRODUCT = 4096 * 4096 * 16384


def listed():
    return [
        # an on-policy batch of a discrete-action agent (full Atari action set, some actions illegal): many tiny rows
        dict(name='log_prob actions', op='log_prob', batch=32, seq=128, vocab=18, dtype='fp32', live=1.0, masked=0.2,
             temperature=1.0, entropy=True, top_k=0, backward=True),
        # one decoding step of a served token policy that reports its eight best alternatives: latency of few long rows
        dict(name='log_prob step', op='log_prob', batch=32, seq=1, vocab=32000, dtype='bf16', live=1.0, masked=0.0,
             temperature=0.7, entropy=True, top_k=8, backward=False),
        # a frozen reference policy scoring a batch of padded responses, odd length and odd vocabulary
        dict(name='log_prob score', op='log_prob', batch=8, seq=1023, vocab=50001, dtype='bf16', live=0.6, masked=0.0,
             temperature=1.0, entropy=False, top_k=0, backward=False),
        # the learner's loss head on long responses over a large vocabulary, with entropy bonus and gradient
        dict(name='log_prob learn', op='log_prob', batch=8, seq=2048, vocab=131072, dtype='bf16', live=0.75, masked=0.0,
             temperature=1.0, entropy=True, top_k=0, backward=True),
        # a collector's step: one token for each environment
        dict(name='recurrence step', op='recurrence', seq=1, batch=256, dim=512, dtype='fp32', start=True, reset=0.02,
             backward=False),
        # a replayed unroll with stored starting state and episode ends inside
        dict(name='recurrence unroll', op='recurrence', seq=80, batch=64, dim=512, dtype='fp32', start=True, reset=0.01,
             backward=True),
        # odd sizes, rows that are not aligned to wide loads
        dict(name='recurrence odd', op='recurrence', seq=5001, batch=3, dim=777, dtype='fp16', start=True, reset=0.002,
             backward=True),
        # two long token sequences: few columns, so the time axis has to be split
        dict(name='recurrence long', op='recurrence', seq=32768, batch=2, dim=2048, dtype='bf16', start=False, reset=0.0,
             backward=True),
        # the hidden layers of a small agent's network, orthogonalised together
        dict(name='orthogonalize mlp', op='orthogonalize', batch=6, rows=128, cols=128, dtype='fp32'),
        # one square projection in single precision
        dict(name='orthogonalize square', op='orthogonalize', batch=1, rows=2048, cols=2048, dtype='fp32'),
        # tall matrices of odd sizes
        dict(name='orthogonalize tall', op='orthogonalize', batch=3, rows=2731, cols=1001, dtype='bf16'),
        # the feed-forward weight of a wide block
        dict(name='orthogonalize wide', op='orthogonalize', batch=1, rows=4096, cols=16384, dtype='bf16'),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(['log_prob', 'recurrence', 'orthogonalize'])
    dtype = rng.choice(['fp32', 'bf16', 'fp16'])
    if op == 'log_prob':
        vocab = _log_int(rng, 2, 131072)
        batch = _log_int(rng, 1, 64)
        half = MOST_LOGITS // 2 if dtype == 'fp32' else MOST_LOGITS
        seq = _log_int(rng, 1, max(1, min(4096, half // (vocab * batch))))
        top_k = rng.choice([0, 0, 0, 1, 5, 20])
        if batch * seq * vocab > MOST_LOGITS // 16:
            top_k = 0
        return dict(op=op, batch=batch, seq=seq, vocab=vocab, dtype=dtype, live=round(rng.uniform(0.3, 1.0), 2),
                    masked=rng.choice([0.0, 0.0, 0.1]), temperature=rng.choice([1.0, 0.7, 1.3]),
                    entropy=rng.random() < 0.5, top_k=min(top_k, vocab), backward=rng.random() < 0.5)
    if op == 'recurrence':
        half = MOST_STATES // 2 if dtype == 'fp32' else MOST_STATES
        dim = _log_int(rng, 16, 4096)
        batch = _log_int(rng, 1, 256)
        seq = _log_int(rng, 1, max(1, min(32768, half // (dim * batch))))
        return dict(op=op, seq=seq, batch=batch, dim=dim, dtype=dtype, start=rng.random() < 0.5,
                    reset=rng.choice([0.0, 0.002, 0.02]), backward=rng.random() < 0.6)
    rows, cols = _log_int(rng, 24, 4096), _log_int(rng, 24, 8192)
    small = min(rows, cols)
    batch = _log_int(rng, 1, max(1, min(16, MOST_PRODUCT // 2 // (rows * cols * small))))
    return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=dtype)


def _live_rows(case):
    return max(1, int(round(case['live'] * case['batch'] * case['seq'])))


def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    if case['op'] == 'log_prob':
        rows, live, vocab = case['batch'] * case['seq'], _live_rows(case), case['vocab']
        # the logits of the live rows once, the tokens, what comes out; the gradient of every row is written
        moved = live * vocab * size + rows * (8 + 4 + 4 * case['entropy'] + 12 * case['top_k'])
        if case['backward']:
            moved += rows * vocab * size + rows * (4 + 4 * case['entropy'])
        return {'bytes': moved, 'flops': live * vocab * (4 + 4 * case['backward'])}
    if case['op'] == 'recurrence':
        states = case['seq'] * case['batch'] * case['dim']
        moved = 3 * states * size + case['seq'] * case['batch'] * (case['reset'] > 0)
        moved += case['batch'] * case['dim'] * 4 * (1 + case['start'])
        if case['backward']:
            # forward's inputs are read again only because both directions are one pass here: counted once
            moved += 3 * states * size + case['batch'] * case['dim'] * 4 * (1 + case['start'])
        return {'bytes': moved, 'flops': states * (8 + 12 * case['backward'])}
    small, large = min(case['rows'], case['cols']), max(case['rows'], case['cols'])
    # a product that is symmetric needs half its entries; the iteration may run on X or on its Gram matrix alone
    on_x = NS_STEPS * (3 * small**2 * large + small**3)
    on_gram = 3 * small**2 * large + (4 * NS_STEPS - 3) * small**3
    return {'bytes': case['batch'] * 2 * small * large * size, 'flops': case['batch'] * min(on_x, on_gram)}


def prepare(case, seed):
    device = torch.device('cuda')
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    dtype = DTYPES[case['dtype']]
    state = dict(case=dict(case))

    def normal(*shape, scale=1.0, to=torch.float32):
        return torch.empty(shape, device=device, dtype=to).normal_(0.0, scale, generator=gen)

    if case['op'] == 'log_prob':
        batch, seq, vocab = case['batch'], case['seq'], case['vocab']
        # a model's logits for every position; the last one predicts nothing that is scored
        logits = normal(batch, seq + 1, vocab, scale=2.5, to=dtype)
        rows = batch * seq
        index = torch.randint(0, vocab, (batch, seq), device=device, generator=gen)
        if case['masked'] > 0:
            illegal = torch.rand(vocab, device=device, generator=gen) < case['masked']
            illegal[0] = False
            logits.masked_fill_(illegal, float('-inf'))
            legal = torch.nonzero(~illegal).squeeze(-1)
            index = legal[index % legal.numel()]
        live = torch.randperm(rows, device=device, generator=gen)[:_live_rows(case)]
        kept = torch.full((rows, ), IGNORE, device=device, dtype=torch.long)
        kept[live] = index.reshape(-1)[live]
        # gradients of a mean over the tokens; half precision is trained with a scaled loss
        scale = (4096.0 if dtype == torch.float16 else 1.0) / rows
        state.update(logits=logits[:, :-1], index=kept.reshape(batch, seq),
                     grad_log_prob=normal(batch, seq, scale=scale))
        if case['entropy']:
            state.update(grad_entropy=normal(batch, seq, scale=0.1 * scale))
        return state
    if case['op'] == 'recurrence':
        seq, batch, dim = case['seq'], case['batch'], case['dim']
        packed = normal(seq, batch, 2 * dim, to=dtype)  # one projection makes the inputs and the gates
        packed[..., dim:] += 2.0
        state.update(x=packed[..., :dim], gate=packed[..., dim:], h0=None, reset=None)
        if case['start']:
            state['h0'] = normal(batch, dim)
        if case['reset'] > 0:
            state['reset'] = torch.rand(seq, batch, device=device, generator=gen) < case['reset']
        if case['backward']:
            state.update(grad_h=normal(seq, batch, dim, to=dtype), grad_last=normal(batch, dim))
        return state
    batch, rows, cols = case['batch'], case['rows'], case['cols']
    rank = max(1, min(rows, cols) // 8)
    # a momentum buffer: a few strong directions and noise
    strong = normal(batch, rows, rank) * torch.linspace(1.0, 0.05, rank, device=device)
    update = torch.bmm(strong, normal(batch, rank, cols)) / math.sqrt(rank) + normal(batch, rows, cols, scale=0.1)
    state.update(update=(update * 1e-3).to(dtype))
    return state


# ------------------------------------------------------------------------------------------------------ plain forms


def _plain_log_prob(s):
    case, logits, index = s['case'], s['logits'], s['index']
    live = index != IGNORE
    z = logits.float()
    top = None
    if case['top_k']:
        # order by value, then by the lower index: the value's bits as an ordered integer above the index
        bits = (z + 0.0).view(torch.int32)
        order = (bits ^ ((bits >> 31) & 0x7fffffff)).long() << 32
        order += case['vocab'] - 1 - torch.arange(case['vocab'], device=z.device)
        top = torch.topk(order, case['top_k'], dim=-1).indices
        del bits, order
    z = (z - z.amax(-1, keepdim=True)) / case['temperature']
    log_p = z - z.exp().sum(-1, keepdim=True).log()
    del z
    out = {}
    token = index.clamp(min=0).unsqueeze(-1)
    out['log_prob'] = torch.where(live, log_p.gather(-1, token).squeeze(-1), 0.0)
    if top is not None:
        out['top_log_prob'] = torch.where(live.unsqueeze(-1), log_p.gather(-1, top), 0.0)
        out['top_index'] = torch.where(live.unsqueeze(-1), top, -1)
    p = log_p.exp()
    if case['entropy']:
        finite = torch.where(p > 0, log_p, 0.0)
        h = -(p * finite).sum(-1)
        out['entropy'] = torch.where(live, h, 0.0)
    if case['backward']:
        g = torch.where(live, s['grad_log_prob'], 0.0).unsqueeze(-1)
        grad = p * -g
        grad.scatter_add_(-1, token, g)
        if case['entropy']:
            grad -= torch.where(live, s['grad_entropy'], 0.0).unsqueeze(-1) * p * (finite + h.unsqueeze(-1))
        out['grad_logits'] = (grad / case['temperature']).to(logits.dtype)
    return out


def _scan(keep, add):
    """h[t] = keep[t] * h[t-1] + add[t] along dim 0: each pass joins spans twice as long."""
    span = 1
    while span < keep.shape[0]:
        add = torch.cat([add[:span], add[span:] + keep[span:] * add[:-span]])
        keep = torch.cat([keep[:span], keep[span:] * keep[:-span]])
        span *= 2
    return add


def _plain_recurrence(s):
    x, f = s['x'].float(), s['gate'].float()
    a, b = 1 / (1 + torch.exp(-f)), 1 / (1 + torch.exp(f))
    keep = a if s['reset'] is None else torch.where(s['reset'].unsqueeze(-1), 0.0, a)
    add = b * x
    if s['h0'] is not None:
        add[0] += keep[0] * s['h0']
    h = _scan(keep, add)
    out = {'h': h.to(s['x'].dtype), 'last': h[-1].clone()}
    if s['case']['backward']:
        g = s['grad_h'].float()
        g = torch.cat([g[:-1], g[-1:] + s['grad_last']])
        after = torch.cat([torch.zeros_like(keep[:1]), keep[1:].flip(0)])
        dh = _scan(after, g.flip(0)).flip(0)
        first = torch.zeros_like(h[0]) if s['h0'] is None else s['h0']
        before = torch.cat([first.unsqueeze(0), h[:-1]])
        if s['reset'] is not None:
            before = torch.where(s['reset'].unsqueeze(-1), 0.0, before)
        out['grad_x'] = (b * dh).to(s['x'].dtype)
        out['grad_gate'] = (dh * (before - x) * a * b).to(s['x'].dtype)
        if s['h0'] is not None:
            out['grad_h0'] = keep[0] * dh[0]
    return out


def _plain_orthogonalize(s):
    a, b, c = NS_COEFFICIENTS
    x = s['update'].float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1).contiguous()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + NS_EPS)
    for _ in range(NS_STEPS):
        gram = torch.bmm(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    if tall:
        x = x.transpose(-2, -1)
    return {'update': x.to(s['update'].dtype).contiguous()}


# ---------------------------------------------------------------------------------------------- the framework's calls


def _own_log_prob(s):
    from ding.rl_utils import token_log_prob
    case, logits = s['case'], s['logits']
    if case['backward']:
        logits = logits.detach().requires_grad_()
    got = token_log_prob(logits, s['index'], temperature=case['temperature'], ignore_index=IGNORE,
                         entropy=case['entropy'], top_k=case['top_k'])
    out = {'log_prob': got.log_prob}
    if case['entropy']:
        out['entropy'] = got.entropy
    if case['top_k']:
        out['top_log_prob'], out['top_index'] = got.top_log_prob, got.top_index
    if case['backward']:
        heads, grads = [got.log_prob], [s['grad_log_prob']]
        if case['entropy']:
            heads.append(got.entropy)
            grads.append(s['grad_entropy'])
        out['grad_logits'], = torch.autograd.grad(heads, [logits], grads)
    return out


def _own_recurrence(s):
    from ding.torch_utils import gated_linear_recurrence
    if not s['case']['backward']:
        h, last = gated_linear_recurrence(s['x'], s['gate'], h0=s['h0'], reset=s['reset'])
        return {'h': h, 'last': last}
    x, gate = s['x'].detach().requires_grad_(), s['gate'].detach().requires_grad_()
    leaves = [x, gate]
    h0 = s['h0']
    if h0 is not None:
        h0 = h0.detach().requires_grad_()
        leaves.append(h0)
    h, last = gated_linear_recurrence(x, gate, h0=h0, reset=s['reset'])
    grads = torch.autograd.grad([h, last], leaves, [s['grad_h'], s['grad_last']])
    out = {'h': h, 'last': last, 'grad_x': grads[0], 'grad_gate': grads[1]}
    if h0 is not None:
        out['grad_h0'] = grads[2]
    return out


def _own_orthogonalize(s):
    from ding.torch_utils import orthogonalize
    return {'update': orthogonalize(s['update'], steps=NS_STEPS, coefficients=NS_COEFFICIENTS, eps=NS_EPS)}


def run(state):
    op = state['case']['op']
    if op == 'log_prob':
        return _own_log_prob(state) if own else _plain_log_prob(state)
    if op == 'recurrence':
        return _own_recurrence(state) if own else _plain_recurrence(state)
    return _own_orthogonalize(state) if own else _plain_orthogonalize(state)


# ------------------------------------------------------------------------------------- the definitions in 64 bits


def _exact_log_prob(s):
    case, dtype = s['case'], s['logits'].dtype
    out = {k: [] for k, on in (('log_prob', True), ('entropy', case['entropy']), ('top_log_prob', case['top_k']),
                               ('grad_logits', case['backward'])) if on}
    flat = s['logits'].reshape(-1, case['vocab'])
    step = max(1, (1 << 28) // case['vocab'])
    for at in range(0, flat.shape[0], step):
        rows = slice(at, at + step)
        z = flat[rows].double() / case['temperature']
        token = s['index'].reshape(-1)[rows]
        on = (token != IGNORE).double().unsqueeze(-1)
        lse = torch.logsumexp(z, -1, keepdim=True)
        z = z - lse
        p = torch.exp(z)
        hit = token.clamp(min=0).unsqueeze(-1)
        out['log_prob'].append(torch.gather(z, 1, hit).squeeze(-1) * on.squeeze(-1))
        if case['top_k']:
            out['top_log_prob'].append(z.topk(case['top_k'], -1).values * on)
        if case['entropy'] or case['backward']:
            z.masked_fill_(p == 0, 0.0)
            h = (p * z).sum(-1, keepdim=True).neg()
        if case['entropy']:
            out['entropy'].append((h * on).squeeze(-1))
        if case['backward']:
            g = s['grad_log_prob'].reshape(-1, 1)[rows].double()
            grad = torch.zeros_like(p)
            grad.scatter_(1, hit, 1.0)
            grad.sub_(p).mul_(g)
            if case['entropy']:
                grad -= s['grad_entropy'].reshape(-1, 1)[rows].double() * (p * (z + h))
            out['grad_logits'].append(grad.mul_(on / case['temperature']).to(
                torch.float64 if flat.numel() <= MOST_LOGITS // 8 else torch.float32))
        del z, p
    shape = s['index'].shape
    got = {k: torch.cat(v) for k, v in out.items()}
    got = {k: v.reshape(shape + v.shape[1:]) for k, v in got.items()}
    if case['top_k']:
        got['top_index'] = None
    return got


def _exact_recurrence(s):
    x, f = s['x'].double(), s['gate'].double()
    a = torch.sigmoid(f)
    seq = x.shape[0]
    if s['reset'] is not None:
        on = (~s['reset']).double().unsqueeze(-1)
    else:
        on = torch.ones(seq, 1, 1, device=x.device, dtype=torch.float64)
    keep, add = a * on, torch.sigmoid(-f) * x
    state = torch.zeros_like(x[0]) if s['h0'] is None else s['h0'].double()
    h = torch.empty_like(x)
    before = torch.empty_like(x)
    for t in range(seq):
        before[t] = state
        torch.addcmul(add[t], keep[t], state, out=h[t])
        state = h[t]
    out = {'h': h, 'last': h[-1]}
    if s['case']['backward']:
        before *= on
        dh = torch.empty_like(x)
        carry = s['grad_last'].double()
        g = s['grad_h'].double()
        for t in range(seq - 1, -1, -1):
            torch.add(g[t], carry, out=dh[t])
            carry = keep[t] * dh[t]
        out['grad_x'] = torch.sigmoid(-f) * dh
        out['grad_gate'] = dh * (before - x) * torch.sigmoid(f) * torch.sigmoid(-f)
        if s['h0'] is not None:
            out['grad_h0'] = carry
    return out


def _exact_orthogonalize(s):
    """The odd polynomials act on the singular values alone: run them on the Gram matrix, multiply X once."""
    a, b, c = NS_COEFFICIENTS
    got = []
    for x in s['update'].double().unbind(0):
        flip = x.shape[0] > x.shape[1]
        x = x.t().contiguous() if flip else x
        x = x / (torch.linalg.vector_norm(x) + NS_EPS)
        gram = x @ x.t().contiguous()
        eye = torch.eye(gram.shape[0], device=x.device, dtype=torch.float64)
        total = eye
        for _ in range(NS_STEPS):
            factor = a * eye + gram @ (b * eye + c * gram)
            total = factor @ total
            gram = factor @ gram @ factor
            gram = (gram + gram.t()) / 2
        x = total @ x
        got.append(x.t() if flip else x)
    return {'update': torch.stack(got)}


def exact(case, seed):
    s = prepare(case, seed)
    if case['op'] == 'log_prob':
        return _exact_log_prob(s)
    if case['op'] == 'recurrence':
        return _exact_recurrence(s)
    return _exact_orthogonalize(s)
