"""The policy operators in 64 bits on the CPU, written from their definitions
(one row, one head, one step at a time), and the tolerances that float32
arithmetic and a rounding to the output's type allow."""
import math

import torch

U = 2.0 ** -24                     # half a step of float32, relative


def head_slices(heads):
    off, out = 0, []
    for n in heads.sizes:
        out.append(slice(off, off + n))
        off += n
    return out


def exists(z, mask):
    """Which choices there are: not masked, logit not -inf."""
    m = torch.ones(z.shape, dtype=torch.bool) if mask is None else (mask != 0).expand(z.shape)
    return m & (z != -math.inf)


def softmax_row(z, there):
    """(log p, p, H) of one head of one row in 64 bits; zeros where nothing is."""
    lp, p = torch.zeros_like(z), torch.zeros_like(z)
    if there.any():
        v = z[there] - z[there].max()          # first: beside -3e38 a logarithm of 2 would be lost
        lp[there] = v - torch.logsumexp(v, 0)
        p[there] = torch.exp(lp[there])
    return lp, p, -(p * lp).sum()


def sample(logits, heads, noise=None, mask=None):
    """(actions, logp, entropy, error of logp, error of entropy)."""
    N = logits.shape[0]
    z32, z = logits.float(), logits.double()
    there = exists(z32, mask)
    actions = torch.zeros((N, heads.act_dim), dtype=torch.int32)
    logp, entropy, err = torch.zeros(N).double(), torch.zeros(N).double(), torch.zeros(N).double()
    for r in range(N):
        for d, s in enumerate(head_slices(heads)):
            t = there[r, s]
            choice = 0
            if t.any():
                score = z32[r, s] + noise[r, s] if noise is not None else z32[r, s].clone()   # float32, as defined
                score[~t] = -math.inf
                choice = int(torch.nonzero(t & (score == score[t].max()))[0])
                lp, p, h = softmax_row(z[r, s], t)
                logp[r] += lp[choice]
                entropy[r] += h
                err[r] += softmax_error(z[r, s], t)
            actions[r, heads.slots[d]] = heads.low[d] + choice
    return actions, logp, entropy, err + 4 * U * heads.n_heads * (logp.abs() + entropy.abs()), \
        2 * err + 4 * U * heads.n_heads * (logp.abs() + entropy.abs())


def softmax_error(z, there):
    """How far float32 may have a log-probability of one head: n terms of a sum,
    each with an exponential of 2 ulp (and one rounding of its argument, up to
    the largest difference), the logarithm's 2 ulp, two subtractions."""
    v = z[there]
    # differences so large that their exponentials vanish do not count
    span = min(float(v.max() - v.min()), 100.0) if len(v) else 0.0
    return U * (len(v) + 8 + 4 * span + 2 * math.log(max(1, len(v))))


def loss_rows(z, actions, advantage, old_logp, heads, ref, mask, clip, kl_coef, entropy_coef):
    """Per row (differentiable by z, 64 bits): loss, policy term, KL, H, clipped, L."""
    lo, hi = clip if isinstance(clip, tuple) else (clip, clip)
    there = exists(z.detach(), mask)
    cols = []
    for r in range(z.shape[0]):
        L = kl = H = torch.zeros((), dtype=torch.float64)
        possible = True
        for d, s in enumerate(head_slices(heads)):
            t = there[r, s]
            if not t.any():
                continue
            idx = torch.nonzero(t)[:, 0]
            lp = torch.log_softmax(z[r, s][idx], 0)
            c = int(actions[r, heads.slots[d]]) - heads.low[d]
            where = torch.nonzero(idx == c)[:, 0]
            if len(where):
                L = L + lp[where[0]]
            else:
                possible = False
            p = torch.exp(lp)
            H = H - (p * lp).sum()
            if ref is not None:
                v = ref[r, s][idx]
                if (v != -math.inf).any():
                    lq = torch.log_softmax(v, 0)
                    k = v != -math.inf
                    kl = kl + (torch.exp(lq[k]) * (lq[k] - lp[k])).sum()
        a = float(advantage[r])
        ratio = torch.exp(L - float(old_logp[r])) if possible else 0 * L
        # the lower of the two; where they are equal the free one, whose gradient it has
        free, held = ratio * a, ratio.detach().clamp(1 - lo, 1 + hi) * a
        clipped = bool(held < free)
        pg = -(held if clipped else free)
        cols.append((pg + kl_coef * kl - entropy_coef * H, pg, kl, H, float(clipped),
                     float(L.detach()) if possible else -math.inf))
    return cols


def policy_loss(logits, actions, advantage, old_logp, heads, ref=None, valid=None, mask=None, clip=0.2, kl_coef=0.0,
                entropy_coef=0.0, denominator=None, scale=1.0):
    """dict of loss, stats, count, logp, grad (64 bits, by autograd over the
    rows) and the absolute errors that float32 allows them."""
    N, C = logits.shape
    rows = [r for r in range(N) if valid is None or valid[r]]
    m = (mask if mask is None or mask.shape[0] == 1 else mask.repeat(N // mask.shape[0], 1))
    at = torch.tensor(rows, dtype=torch.long)
    z = logits[at].double()
    there = exists(z, None if m is None else (m if m.shape[0] == 1 else m[at]))
    z = torch.where(there, z, -math.inf).requires_grad_()
    k = None if ref is None else ref[at].double()
    cols = loss_rows(z, actions[at], advantage[at], old_logp[at], heads, k, None, clip, kl_coef, entropy_coef)
    M = float(len(rows)) if denominator is None else float(denominator)
    inv = 1 / M if M > 0 else 0.0
    grad = torch.zeros((N, C), dtype=torch.float64)
    logp = torch.zeros(N, dtype=torch.float64)
    total = sum((c[0] for c in cols), torch.zeros((), dtype=torch.float64)) * inv
    if rows and total.requires_grad:
        g, = torch.autograd.grad(total, z)
        grad[at] = torch.where(there, g, 0.0) * scale
    for r, c in zip(rows, cols):
        logp[r] = c[5]
    stats = torch.tensor([sum(float(torch.as_tensor(c[i]).detach()) for c in cols) * inv for i in (1, 2, 3, 4)], dtype=torch.float64)
    # errors: of each row's L, of its ratio, of its terms
    e_logp, e_grad, e_terms = torch.zeros(N).double(), torch.zeros((N, C)).double(), [0.0, 0.0, 0.0]
    for i, r in enumerate(rows):
        e = sum(softmax_error(z.detach()[i, s], there[i, s]) for s in head_slices(heads))
        e_ref = 0.0
        if ref is not None:
            for s in head_slices(heads):
                t = there[i, s] & (k[i, s] != -math.inf)
                e_ref += softmax_error(k[i, s], t) + U * 4 * float(
                    (z.detach()[i, s][t] - k[i, s][t]).abs().max() if t.any() else 0)
        size = abs(cols[i][5]) if math.isfinite(cols[i][5]) else 0.0
        e_logp[r] = e + 4 * U * len(heads.sizes) * size
        A = abs(float(advantage[r]))
        ratio = math.exp(cols[i][5] - float(old_logp[r])) if math.isfinite(cols[i][5]) else 0.0
        e_ratio = ratio * (e_logp[r] + U * (4 + abs(size) + abs(float(old_logp[r]))))
        e_pg = A * (e_ratio + 4 * U * ratio)
        H = float(cols[i][3].detach())
        e_kl, e_h = e + e_ref + 8 * U * (1 + abs(float(cols[i][2].detach()))), 2 * e + 8 * U * (1 + H)
        e_terms = [e_terms[0] + e_pg, e_terms[1] + e_kl, e_terms[2] + e_h]
        # p, q within e; log p + H up to their sizes
        big = max(1.0, H) + 20.0
        e_grad[r] = (e_pg + ratio * A * (2 * e + 8 * U) + abs(kl_coef) * (2 * e + 2 * e_ref + 8 * U)
                     + abs(entropy_coef) * big * (2 * e + 16 * U)) * inv * scale
    e_terms = [v * inv + 4 * U * abs(float(s)) for v, s in zip(e_terms, stats)]
    e_loss = e_terms[0] + abs(kl_coef) * e_terms[1] + abs(entropy_coef) * e_terms[2] + 4 * U * abs(float(total.detach()))
    return dict(loss=float(total.detach()), stats=stats, count=M, logp=logp, grad=grad, e_loss=e_loss,
                e_stats=e_terms + [4 * U], e_logp=e_logp, e_grad=e_grad)


def near(got, want, err, dtype=torch.float32):
    """|got - want| within err and half a step of the type that got was rounded to
    (its smallest step included)."""
    got, want = got.detach().double().cpu(), want.double()
    info = torch.finfo(dtype)
    room = torch.as_tensor(err).double() + info.eps / 2 * want.abs() + info.smallest_normal * info.eps
    same = (got == want) | (torch.isnan(got) & torch.isnan(want))
    off = torch.where(same, 0.0, (got - want).abs() / room)
    return float(off.max()) if off.numel() else 0.0


# ---------------------------------------------------------------- recurrence
def _per_channel(t, x, dtype):
    """t's values for each element of x [T, ...] (t: like x, its first
    dimensions, or those with a last dimension of 1)."""
    t = t.to(dtype)
    while t.dim() < x.dim():
        t = t[..., None]
    return t.expand(x.shape)


def recurrence(gate, x, state=None, cut=None, reverse=False):
    """(h, last) in 64 bits, differentiable."""
    T = x.shape[0]
    xs = x.double()
    a = _per_channel(gate, x, torch.float64) if isinstance(gate, torch.Tensor) else torch.full_like(xs, gate)
    drop = None if cut is None else _per_channel(cut, x, torch.bool)
    h = torch.zeros(x.shape[1:], dtype=torch.float64) if state is None else state.double()
    out = [None] * T
    for t in (reversed(range(T)) if reverse else range(T)):
        # a gate of 0 drops the state, whatever it holds; its own gradient remains
        kept = a[t] * h
        if drop is not None:
            kept = torch.where(drop[t], torch.zeros_like(kept), kept)
        h = kept + xs[t]
        out[t] = h
    return (torch.stack(out) if T else xs.clone()), h


def recurrence_error(gate, x, state=None, cut=None, reverse=False):
    """A bound of float32's error of every h: each step rounds the product and
    the sum, and carries the error before it (the joined form of a split axis
    rounds products of gates too: three roundings a step are allowed, and one
    for each of the up to 64 pieces joined)."""
    T = x.shape[0]
    a = _per_channel(gate, x, torch.float64).abs() if isinstance(gate, torch.Tensor) else \
        torch.full(x.shape, abs(gate), dtype=torch.float64)
    if cut is not None:
        a = torch.where(_per_channel(cut, x, torch.bool), 0.0, a)
    big = torch.zeros(x.shape[1:], dtype=torch.float64) if state is None else state.double().abs()
    err = torch.zeros_like(big)
    out = [None] * T
    for t in (reversed(range(T)) if reverse else range(T)):
        err = a[t] * err + 4 * U * a[t] * big
        big = a[t] * big + x[t].double().abs()
        err = err + 4 * U * big
        out[t] = err
    return (torch.stack(out) if T else x.double()), err


# ---------------------------------------------------------------- advantages
def marks(all_done, steps, horizon, autoreset, before=None, err=None):
    K, E = all_done.shape
    out = torch.zeros((K, E), dtype=torch.uint8)
    for e in range(E):
        n = int(steps[e]) if steps is not None else 0
        ended = bool(before[e]) if before is not None else False
        for t in range(K):
            m = 8 if err is not None and int(err[e]) else 0
            if autoreset == 'next_step' and (ended or (horizon and n >= horizon)):
                m, n, ended = m | 4, 0, False
            else:
                n, ended = n + 1, bool(all_done[t, e])
                over = bool(horizon) and n >= horizon
                if autoreset == 'same_step':
                    m |= 1 if ended or over else 0
                    n = 0 if ended or over else n
                else:
                    m |= 1 if ended else 2 if over else 0
            out[t, e] = m
    return out


def advantages(reward, value, done, mark, live, gamma, lam, acts=None):
    """(advantage, target, valid, error) in 64 bits, a lane at a time."""
    K, E, A = reward.shape
    adv, target, err = (torch.zeros((K, E, A), dtype=torch.float64) for _ in range(3))
    valid = torch.zeros((K, E, A), dtype=torch.uint8)
    r, v = reward.double(), value.double()
    for e in range(E):
        for a in range(A):
            if acts is not None and not acts[a]:
                continue
            carry = bad = 0.0
            for t in reversed(range(K)):
                m = int(mark[t, e])
                before = bool(live[e, a]) if t == 0 else bool(int(mark[t - 1, e]) & 1) or not bool(done[t - 1, e, a])
                if not before or m & (4 | 8):
                    carry = bad = 0.0
                    continue
                final = bool(done[t, e, a]) or bool(m & 1)
                nxt = 0.0 if final else gamma * float(v[t + 1, e, a])
                back = 0.0 if final or m & 2 else gamma * lam
                size = abs(float(r[t, e, a])) + abs(float(v[t, e, a])) + abs(nxt) + abs(back * carry)
                carry = float(r[t, e, a]) + nxt - float(v[t, e, a]) + back * carry
                bad = abs(back) * bad + 8 * U * size
                adv[t, e, a], valid[t, e, a], err[t, e, a] = carry, 1, bad
                target[t, e, a] = carry + float(v[t, e, a])
    return adv, target, valid, err
