"""The policy operators over rollout fragments, as measured: drawing actions,
the clipped policy loss with its gradient, the gated linear recurrence and the
advantages it gives, each in plain torch operations (`own` False) and through
abmarl_amd.learning (`own` True)."""
import functools
import math

import torch

own = False

DTYPES = {'f32': torch.float32, 'f16': torch.float16, 'bf16': torch.bfloat16}
BYTES = {'f32': 4, 'f16': 2, 'bf16': 2}
CLIP, KL, ENTROPY = 0.2, 0.2, 0.01
GAMMA, LAM = 0.99, 0.95
END, TRUNCATED, RESET = 1, 2, 4          # marks of a step of an env

# action rows of the programs: move row, move column (Box(-r, r)), attack
TEAM = {'heads': '3,3,2', 'low': '-1,-1,0'}
RTT = {'heads': '5,5,2,2,2,2,2,2,2,2,2', 'low': '-2,-2,0,0,0,0,0,0,0,0,0'}
CROSS = {'heads': '5', 'low': '0'}
# ReachTheTarget's target as one raveled index: 5 x 5 moves x 2^9 attacks
RAVEL = {'heads': '12800', 'low': '0'}


def listed():
    return [
        # one SGD minibatch of 128 agent steps, the autograd form
        {'name': 'loss_minibatch', 'op': 'loss', 'rows': 128, **RTT, 'dtype': 'f32', 'form': 'autograd',
         'ref': True, 'valid': False, 'lanes': 0},
        # the headline fragment: 20 steps x 4096 envs x 64 agents, dead agents' rows left out
        {'name': 'loss_team_fragment', 'op': 'loss', 'rows': 20 * 4096 * 64, **TEAM, 'dtype': 'bf16',
         'form': 'grad', 'ref': True, 'valid': True, 'lanes': 0},
        # ReachTheTarget: 4 steps x 1023 envs x 256 lanes that may choose different things, loss scaling
        {'name': 'loss_rtt_lanes', 'op': 'loss', 'rows': 4 * 1023 * 256, **RTT, 'dtype': 'f16', 'form': 'autograd',
         'ref': False, 'valid': True, 'lanes': 256},
        # raveled actions: the widest softmax that the wrappers give
        {'name': 'loss_ravel', 'op': 'loss', 'rows': 4099, **RAVEL, 'dtype': 'bf16', 'form': 'grad',
         'ref': True, 'valid': False, 'lanes': 0},
        # one env's agents choose (the dict API's step)
        {'name': 'sample_one_env', 'op': 'sample', 'rows': 64, **TEAM, 'dtype': 'f32', 'lanes': 0},
        # the closed loop's step: 4096 envs x 64 agents
        {'name': 'sample_closed_loop', 'op': 'sample', 'rows': 4096 * 64, **TEAM, 'dtype': 'bf16', 'lanes': 0},
        # 1024 targets choose a raveled action
        {'name': 'sample_ravel', 'op': 'sample', 'rows': 1024, **RAVEL, 'dtype': 'f16', 'lanes': 0},
        # a policy memory of 256 channels over a fragment of 20 steps x 4096 envs, forward and backward
        {'name': 'memory_fragment', 'op': 'memory', 'T': 20, 'B': 4096, 'D': 256, 'dtype': 'bf16',
         'shared': False, 'reverse': False, 'cut': True, 'grad': True},
        # one env played for long: few channels, a long axis, a gate shared by the channels
        {'name': 'memory_long', 'op': 'memory', 'T': 65537, 'B': 1, 'D': 96, 'dtype': 'f32',
         'shared': True, 'reverse': False, 'cut': True, 'grad': True},
        # one step of the memory while acting
        {'name': 'memory_step', 'op': 'memory', 'T': 1, 'B': 1024, 'D': 256, 'dtype': 'bf16',
         'shared': False, 'reverse': False, 'cut': True, 'grad': False},
        # the headline fragment of 100 steps
        {'name': 'advantages_fragment', 'op': 'advantages', 'T': 100, 'E': 4096, 'A': 64, 'dtype': 'f32'},
        # few envs, long episodes
        {'name': 'advantages_long', 'op': 'advantages', 'T': 5003, 'E': 3, 'A': 5, 'dtype': 'bf16'},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_heads(rng):
    kind = rng.choice(['moves', 'cells', 'cross', 'one', 'one'])
    if kind == 'moves':
        r, k = rng.randint(1, 7), rng.randint(1, 4)
        return {'heads': '%d,%d,%d' % (2 * r + 1, 2 * r + 1, k + 1), 'low': '%d,%d,0' % (-r, -r)}
    if kind == 'cells':
        r, d, k = rng.randint(1, 4), 2 * rng.randint(0, 3) + 1, rng.randint(1, 3)
        return {'heads': ','.join(['%d' % (2 * r + 1)] * 2 + ['%d' % (k + 1)] * (d * d)),
                'low': ','.join(['%d' % -r] * 2 + ['0'] * (d * d))}
    if kind == 'cross':
        return dict(CROSS)
    return {'heads': '%d' % _log_int(rng, 2, 40000), 'low': '0'}


def draw(rng):
    op = rng.choice(['loss', 'loss', 'sample', 'memory', 'memory', 'advantages'])
    dtype = rng.choice(['f32', 'f16', 'bf16'])
    if op in ('loss', 'sample'):
        h = _draw_heads(rng)
        width = sum(_ints(h['heads']))
        most = max(1, min(20 * 4096 * 64, (20 << 20) // width))
        rows = _log_int(rng, 1, most)
        lanes = rng.choice([0, 0, 1, 7, 64])
        rows = max(1, rows // lanes) * lanes if lanes else rows
        c = {'op': op, 'rows': rows, **h, 'dtype': dtype, 'lanes': lanes}
        if op == 'loss':
            c.update(form=rng.choice(['grad', 'autograd']), ref=rng.random() < 0.6, valid=rng.random() < 0.6)
        return c
    if op == 'memory':
        T, D = _log_int(rng, 1, 65537), _log_int(rng, 1, 512)
        B = _log_int(rng, 1, max(1, min(4096, (20 << 20) // (T * D))))
        return {'op': op, 'T': T, 'B': B, 'D': D, 'dtype': dtype, 'shared': rng.random() < 0.4,
                'reverse': rng.random() < 0.3, 'cut': rng.random() < 0.7, 'grad': rng.random() < 0.7}
    T, A = _log_int(rng, 1, 5003), _log_int(rng, 1, 256)
    E = _log_int(rng, 1, max(1, min(8192, (26 << 20) // (T * A))))
    return {'op': op, 'T': T, 'E': E, 'A': A, 'dtype': rng.choice(['f32', 'bf16'])}


# ------------------------------------------------------------------ layouts
def _ints(text):
    return [int(v) for v in text.split(',')]


@functools.lru_cache(None)
def _layout(heads):
    """Of the heads' sizes: for each head the columns of its choices (padded
    to the widest head), which of them are real, and each column's place."""
    sizes = _ints(heads)
    M, C = max(sizes), sum(sizes)
    off = [sum(sizes[:d]) for d in range(len(sizes))]
    cols = torch.tensor([[min(o + i, C - 1) for i in range(M)] for o in off], device='cuda')
    real = torch.tensor([[i < n for i in range(M)] for n in sizes], device='cuda')
    place = torch.tensor([d * M + i for d, n in enumerate(sizes) for i in range(n)], device='cuda')
    return cols, real, place


@functools.lru_cache(None)
def _heads(heads, low):
    from abmarl_amd.learning import PolicyHeads
    return PolicyHeads(_ints(heads), low=_ints(low))


@functools.lru_cache(None)
def _low(low):
    return torch.tensor(_ints(low), device='cuda', dtype=torch.int32)


def _lane_mask(case, lanes):
    """What each lane may choose: a third of the lanes nothing, a third the
    first two heads (they move), a third the others (they attack)."""
    sizes = _ints(case['heads'])
    lane = torch.arange(lanes, device='cuda') % 3
    which = torch.cat([torch.full((n,), 1 if d < 2 else 2, device='cuda') for d, n in enumerate(sizes)])
    return (lane[:, None] == which[None, :]).to(torch.uint8) if lanes > 1 else \
        torch.ones((1, sum(sizes)), dtype=torch.uint8, device='cuda')


# ------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    return {'case': case, **{'loss': _prepare_loss, 'sample': _prepare_sample, 'memory': _prepare_memory,
                             'advantages': _prepare_advantages}[case['op']](case, g)}


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device='cuda')


def _rand(g, *shape):
    return torch.rand(shape, generator=g, device='cuda')


def _gumbel(g, *shape):
    return -torch.log(torch.empty(shape, device='cuda').exponential_(generator=g))


def _prepare_sample(case, g):
    N, C = case['rows'], sum(_ints(case['heads']))
    return {'logits': (1.5 * _randn(g, N, C)).to(DTYPES[case['dtype']]), 'noise': _gumbel(g, N, C),
            'mask': _lane_mask(case, case['lanes']) if case['lanes'] else None}


def _prepare_loss(case, g):
    s = _prepare_sample(case, g)
    N, z = case['rows'], s['logits']
    s['ref'] = (z.float() + 0.2 * _randn(g, *z.shape)).to(z.dtype) if case['ref'] else None
    # what the behaviour policy chose, and how likely it was to: the ratios lie
    # around 1, none of them next to the border that the clipping has
    choice, logp, _ = _choose(case, z, s.pop('noise'), s['mask'])
    s['actions'] = choice + _low(case['low'])
    d = 0.15 * _randn(g, N)
    for border in (math.log(1 - CLIP), math.log(1 + CLIP)):
        d = torch.where((d - border).abs() < 1e-3, border + 2e-3, d)
    s['old_logp'] = logp - d
    s['advantage'] = _randn(g, N)
    s['valid'] = None
    if case['valid']:
        # agents that are done: no action, and logits of unwritten observations
        s['valid'] = (_rand(g, N) < 0.7).to(torch.uint8)
        s['logits'] = torch.where(((s['valid'] == 0) & (_rand(g, N) < 0.2))[:, None], math.nan, z).to(z.dtype)
    # fp16 gradients of a mean over many rows need the loss scaled
    scale = 2.0 ** round(math.log2(N)) if case['dtype'] == 'f16' else 1.0
    s['scale'] = torch.tensor(scale, device='cuda')
    s['scale_value'] = scale
    return s


def _prepare_memory(case, g):
    T, B, D, t = case['T'], case['B'], case['D'], DTYPES[case['dtype']]
    gate = torch.sigmoid(2 + _randn(g, T, B, 1 if case['shared'] else D)).to(t)
    s = {'gate': gate, 'x': _randn(g, T, B, D).to(t), 'state': _randn(g, B, D),
         'cut': (_rand(g, T, B) < 0.01).to(torch.uint8) if case['cut'] else None}
    if case['grad']:
        s['dh'], s['dlast'] = _randn(g, T, B, D).to(t), _randn(g, B, D)
    return s


def _prepare_advantages(case, g):
    T, E, A = case['T'], case['E'], case['A']
    # episodes that end, or are cut at a horizon, once in about 150 steps;
    # the step behind such a one is the env's reset
    u = _rand(g, T, E)
    last = (u < 1 / 150) & ~torch.cat([torch.zeros_like(u[:1]) > 0, u[:-1] < 1 / 150])
    reset = torch.cat([torch.zeros_like(last[:1]), last[:-1]])
    marks = torch.where(last, torch.where(u < 1 / 300, END, TRUNCATED), 0) + RESET * reset
    # an agent is done from its last step to the reset
    done = _rand(g, T, E, A) < 0.01
    done |= torch.cat([torch.zeros_like(done[:1]), done[:-1]]) & ~reset[:, :, None]
    reward = torch.where(_rand(g, T, E, A) < 0.2, _rand(g, T, E, A) * 2 - 1, -0.01).double()
    return {'reward': reward, 'value': _randn(g, T + 1, E, A).to(DTYPES[case['dtype']]), 'done': done.to(torch.uint8),
            'marks': marks.to(torch.uint8), 'live': (_rand(g, E, A) < 0.9).to(torch.uint8)}


# -------------------------------------------------------------------- plain
def _by_head(case, z, mask):
    """Logits as [rows, heads, widest], choices that are none at -inf."""
    cols, real, _ = _layout(case['heads'])
    if mask is not None:
        z = torch.where(mask.bool().repeat(z.shape[0] // mask.shape[0], 1), z, -math.inf)
    return torch.where(real, z[:, cols], -math.inf)


def _log_softmax(z):
    """Logarithms of the probabilities, and the probabilities; a head that has no choice gives zeros."""
    some = (z > -math.inf).any(-1, keepdim=True)
    top = torch.where(some, z.amax(-1, keepdim=True), 0)
    e = torch.where(z > -math.inf, torch.exp(z - top), 0)
    total = torch.where(some, e.sum(-1, keepdim=True), 1)
    lp = torch.where(z > -math.inf, z - top - torch.log(total), 0)
    return lp, e / total


def _choose(case, logits, noise, mask):
    z = _by_head(case, logits.float(), mask)
    score = z + _by_head(case, noise, None)
    score = torch.where(z > -math.inf, score, -math.inf)
    M = z.shape[-1]
    first = torch.where(score == score.amax(-1, keepdim=True), torch.arange(M, device='cuda'), M).amin(-1)
    first = torch.where((z > -math.inf).any(-1), first, 0)
    lp, p = _log_softmax(z)
    return first.to(torch.int32), lp.gather(-1, first[..., None].long())[..., 0].sum(-1), -(p * lp).sum((-1, -2))


def _plain_loss(s):
    case, z = s['case'], s['logits']
    N, M = z.shape[0], _layout(case['heads'])[2]
    ok = s['valid'].bool() if s['valid'] is not None else torch.ones(N, dtype=torch.bool, device='cuda')
    zh = _by_head(case, torch.where(ok[:, None], z.float(), 0), s['mask'])
    lp, p = _log_softmax(zh)
    choice = (s['actions'] - _low(case['low'])).long()[..., None]
    logp = lp.gather(-1, choice)[..., 0].sum(-1)
    count = ok.sum().float().clamp(min=1)
    ratio = torch.exp(logp - s['old_logp'])
    a = s['advantage']
    free, held = ratio * a, ratio.clamp(1 - CLIP, 1 + CLIP) * a
    entropy = -(p * lp).sum(-1)
    kl = torch.zeros_like(logp)
    pull = torch.where(held < free, 0, -free)[:, None, None]
    chosen = torch.zeros_like(p).scatter_(-1, choice, 1.0) * (zh > -math.inf)
    grad = pull * (chosen - p) + ENTROPY * p * (lp + entropy[..., None])
    if s['ref'] is not None:
        lq, q = _log_softmax(_by_head(case, torch.where(ok[:, None], s['ref'].float(), 0), s['mask']))
        kl = (q * (lq - lp)).sum((-1, -2))
        grad = grad + KL * (p - q)
    entropy = entropy.sum(-1)
    mean = lambda v: torch.where(ok, v, 0).sum() / count  # noqa: E731
    stats = torch.stack([mean(-torch.minimum(free, held)), mean(kl), mean(entropy), mean((held < free).float())])
    loss = stats[0] + KL * stats[1] - ENTROPY * stats[2]
    grad = torch.where(ok[:, None], grad.flatten(1)[:, M], 0) * (s['scale'] / count)
    return {'loss': loss, 'stats': stats, 'logp': torch.where(ok, logp, 0), 'grad': grad.to(z.dtype)}


def _scan(a, b):
    """h[t] = a[t] h[t-1] + b[t] by doubling: log2(T) passes over whole tensors."""
    step = 1
    while step < b.shape[0]:
        b = torch.cat([b[:step], b[step:] + a[step:] * b[:-step]])
        a = torch.cat([a[:step], a[step:] * a[:-step]])
        step *= 2
    return b


def _plain_memory(s):
    case, x = s['case'], s['x']
    gate = s['gate'].float()
    if s['cut'] is not None:
        gate = torch.where(s['cut'].bool()[..., None], 0, gate)
    xs = x.float()
    if case['reverse']:
        gate, xs = gate.flip(0), xs.flip(0)
    h = _scan(gate, torch.cat([xs[:1] + gate[:1] * s['state'], xs[1:]]))
    out = {'h': (h.flip(0) if case['reverse'] else h).to(x.dtype), 'last': h[-1]}
    if case['grad']:
        dh = s['dh'].float()
        dh = dh.flip(0) if case['reverse'] else dh
        dh = torch.cat([dh[:-1], dh[-1:] + s['dlast']])
        after = torch.cat([gate[1:], torch.zeros_like(gate[:1])])
        g = _scan(after.flip(0), dh.flip(0)).flip(0)
        dgate = g * torch.cat([s['state'][None], h[:-1]])
        out['dstate'] = gate[0] * g[0]
        if case['reverse']:
            g, dgate = g.flip(0), dgate.flip(0)
        if s['cut'] is not None:
            dgate = torch.where(s['cut'].bool()[..., None], 0, dgate)
        dgate = dgate.sum(-1, keepdim=True) if case['shared'] else dgate
        out.update(dx=g.to(x.dtype), dgate=dgate.to(x.dtype))
    return out


def _fates(s):
    """Of every step of every lane: whether it acted, whether nothing follows, whether the episode goes on in the next step."""
    marks, done = s['marks'].int()[..., None], s['done'].bool()
    before = torch.cat([s['live'][None].bool(), ~done[:-1] | ((marks[:-1] & END) > 0)])
    acted = before & ((marks & RESET) == 0)
    final = done | ((marks & END) > 0)
    return acted, final, acted & ~final & ((marks & TRUNCATED) == 0)


def _plain_advantages(s):
    acted, final, goes_on = _fates(s)
    v = s['value'].float()
    delta = s['reward'].float() + torch.where(final, 0, GAMMA * v[1:]) - v[:-1]
    delta = torch.where(acted, delta, 0)
    adv = _scan((GAMMA * LAM * goes_on.float()).flip(0), delta.flip(0)).flip(0)
    return {'advantage': adv, 'target': torch.where(acted, adv + v[:-1], 0), 'valid': acted.to(torch.uint8)}


def run(s):
    case = s['case']
    if own:
        return _run_own(s)
    if case['op'] == 'loss':
        return _plain_loss(s)
    if case['op'] == 'sample':
        choice, logp, entropy = _choose(case, s['logits'], s['noise'], s['mask'])
        return {'actions': choice + _low(case['low']), 'logp': logp, 'entropy': entropy}
    return _plain_memory(s) if case['op'] == 'memory' else _plain_advantages(s)


# ------------------------------------------------------------ the framework
def _run_own(s):
    from abmarl_amd import learning
    case = s['case']
    if case['op'] == 'sample':
        r = learning.sample_actions(s['logits'], _heads(case['heads'], case['low']), noise=s['noise'],
                                    choice_mask=s['mask'])
        return {'actions': r.actions, 'logp': r.logp, 'entropy': r.entropy}
    if case['op'] == 'loss':
        kw = dict(ref_logits=s['ref'], valid=s['valid'], choice_mask=s['mask'], clip=CLIP, kl_coef=KL,
                  entropy_coef=ENTROPY)
        args = (s['actions'], s['advantage'], s['old_logp'], _heads(case['heads'], case['low']))
        if case['form'] == 'grad':
            r = learning.policy_loss_grad(s['logits'], *args, grad_scale=s['scale_value'], **kw)
            return {'loss': r.loss, 'stats': r.stats, 'logp': r.logp, 'grad': r.grad}
        z = s['logits'].detach().requires_grad_()
        r = learning.policy_loss(z, *args, **kw)
        grad, = torch.autograd.grad(r.loss, z, s['scale'])
        return {'loss': r.loss.detach(), 'stats': r.stats, 'logp': r.logp, 'grad': grad}
    if case['op'] == 'memory':
        kw = dict(cut=s['cut'], reverse=case['reverse'])
        if not case['grad']:
            h, last = learning.linear_recurrence(s['gate'], s['x'], s['state'], **kw)
            return {'h': h, 'last': last}
        leaves = [s[k].detach().requires_grad_() for k in ('gate', 'x', 'state')]
        h, last = learning.linear_recurrence(*leaves, **kw)
        dgate, dx, dstate = torch.autograd.grad((h, last), leaves, (s['dh'], s['dlast']))
        return {'h': h.detach(), 'last': last.detach(), 'dx': dx, 'dgate': dgate, 'dstate': dstate}
    r = learning.advantages(s['reward'], s['value'], s['done'], s['marks'], s['live'], gamma=GAMMA, lam=LAM)
    return {'advantage': r.advantage, 'target': r.target, 'valid': r.valid}


# --------------------------------------------------------------------- work
def work(case):
    b = BYTES[case['dtype']]
    if case['op'] in ('loss', 'sample'):
        N, sizes = case['rows'], _ints(case['heads'])
        C, D = sum(sizes), len(sizes)
        lanes = case['lanes'] * C
        if case['op'] == 'sample':
            return {'bytes': N * (C * (b + 4) + 4 * D + 8) + lanes, 'flops': 10 * N * C}
        row = C * b * (3 if case['ref'] else 2) + 4 * D + 12 + (1 if case['valid'] else 0)
        return {'bytes': N * row + lanes, 'flops': N * C * (26 if case['ref'] else 16)}
    T = case['T']
    if case['op'] == 'memory':
        B, n = case['B'], case['B'] * case['D']
        gates = B if case['shared'] else n
        fwd = T * (2 * n * b + gates * b + (B if case['cut'] else 0)) + 8 * n
        # backward: gate, x and dh in, dx and dgate out
        bwd = T * (3 * n * b + 2 * gates * b + (B if case['cut'] else 0)) + 12 * n
        return {'bytes': fwd + (bwd if case['grad'] else 0), 'flops': T * n * (7 if case['grad'] else 2)}
    n = case['E'] * case['A']
    return {'bytes': T * (n * (8 + b + 1 + 4 + 4 + 1) + case['E']) + n * (1 + b), 'flops': 8 * T * n}


# -------------------------------------------------------------------- exact
def _split(case, z, mask):
    """One [rows, size] matrix of logits in 64 bits for each head, -inf where a choice is none."""
    z = z.double()
    if mask is not None:
        z = z.masked_fill(mask.repeat(z.shape[0] // mask.shape[0], 1) == 0, -math.inf)
    return z.split(_ints(case['heads']), dim=1)


def _softmax64(z):
    none = torch.isinf(z)
    dead = none.all(1, keepdim=True)
    lp = torch.log_softmax(z.masked_fill(dead, 0.0), 1).masked_fill(none, 0.0)
    return lp, lp.exp().masked_fill(none, 0.0), none


def exact(case, seed):
    s = prepare(case, seed)
    return {'loss': _exact_loss, 'sample': _exact_sample, 'memory': _exact_memory,
            'advantages': _exact_advantages}[case['op']](case, s)


def _exact_sample(case, s):
    logp = entropy = 0
    for z, noise, zf in zip(_split(case, s['logits'], s['mask']), s['noise'].split(_ints(case['heads']), 1),
                            s['logits'].float().split(_ints(case['heads']), 1)):
        # the choice is by the sums as 32 bits hold them: that is its definition
        choice = (zf + noise).masked_fill(torch.isinf(z), -math.inf).argmax(1, keepdim=True)
        lp, p, _ = _softmax64(z)
        logp = logp + lp.gather(1, choice)[:, 0]
        entropy = entropy - (p * lp).sum(1)
    return {'actions': None, 'logp': logp, 'entropy': entropy}


def _exact_loss(case, s):
    valid = torch.ones(case['rows'], device='cuda') if s['valid'] is None else s['valid']
    rows = torch.nonzero(valid)[:, 0]
    lanes = s['mask'][rows % s['mask'].shape[0]] if s['mask'] is not None else None
    heads = list(zip(_split(case, s['logits'][rows], lanes), _ints(case['low'])))
    refs = _split(case, s['ref'][rows], lanes) if s['ref'] is not None else [None] * len(heads)
    chosen = [(s['actions'][rows, d].long() - low)[:, None] for d, (_, low) in enumerate(heads)]
    logp = sum(_softmax64(z)[0].gather(1, c)[:, 0] for (z, _), c in zip(heads, chosen))
    n, a = max(1, len(rows)), s['advantage'][rows].double()
    ratio = torch.exp(logp - s['old_logp'][rows].double())
    held = torch.where(ratio < 1 - CLIP, 1 - CLIP, torch.where(ratio > 1 + CLIP, 1 + CLIP, ratio))
    clipped = held * a < ratio * a
    kl = entropy = 0
    grads = []
    for (z, _), r, c in zip(heads, refs, chosen):
        lp, p, none = _softmax64(z)
        h = -(p * lp).sum(1, keepdim=True)
        entropy = entropy + h[:, 0]
        one = torch.zeros_like(p).scatter_(1, c, 1.0).masked_fill(none, 0.0)
        gz = (ratio * a).masked_fill(clipped, 0.0)[:, None] * (p - one) + ENTROPY * p * (lp + h)
        if r is not None:
            lq, q, _ = _softmax64(r)
            kl = kl + (q * (lq - lp)).sum(1)
            gz = gz + KL * (p - q)
        grads.append(gz * (s['scale_value'] / n))
    pg = -torch.where(clipped, held * a, ratio * a)
    stats = torch.stack([v.sum() / n if torch.is_tensor(v) else torch.zeros((), dtype=torch.float64, device='cuda')
                         for v in (pg, kl, entropy, clipped.double())])
    grad = torch.zeros(s['logits'].shape, dtype=torch.float64, device='cuda')
    grad[rows] = torch.cat(grads, 1)
    whole = torch.zeros(case['rows'], dtype=torch.float64, device='cuda')
    whole[rows] = logp
    return {'loss': stats[0] + KL * stats[1] - ENTROPY * stats[2], 'stats': stats, 'logp': whole, 'grad': grad}


def _exact_memory(case, s):
    if case['T'] * (2 if case['grad'] else 1) > 140000:
        return None
    order = list(range(case['T']))
    order = order[::-1] if case['reverse'] else order
    gate = s['gate'].double()
    if s['cut'] is not None:
        gate = gate.masked_fill(s['cut'][..., None] != 0, 0.0)
    x, h = s['x'].double(), s['state'].double()
    hs, prev = torch.empty_like(x), torch.empty_like(x)
    for t in order:
        prev[t] = h
        h = torch.addcmul(x[t], gate[t], h)
        hs[t] = h
    out = {'h': hs, 'last': h}
    if case['grad']:
        dh, g = s['dh'].double(), s['dlast'].double()
        gs = torch.empty_like(x)
        for t in order[::-1]:
            gs[t] = dh[t] + g
            g = gate[t] * gs[t]
        dgate = gs * prev
        if s['cut'] is not None:
            dgate = dgate.masked_fill(s['cut'][..., None] != 0, 0.0)
        out.update(dx=gs, dgate=dgate.sum(-1, keepdim=True) if case['shared'] else dgate, dstate=g)
    return out


def _exact_advantages(case, s):
    acted, final, goes_on = _fates(s)
    v, r = s['value'].double(), s['reward']
    adv, carry = torch.empty_like(r), torch.zeros_like(r[0])
    for t in reversed(range(case['T'])):
        d = r[t] - v[t] + GAMMA * v[t + 1].masked_fill(final[t], 0.0)
        carry = (d + GAMMA * LAM * carry.masked_fill(~goes_on[t], 0.0)).masked_fill(~acted[t], 0.0)
        adv[t] = carry
    return {'advantage': adv, 'target': (adv + v[:-1]).masked_fill(~acted, 0.0), 'valid': None}
