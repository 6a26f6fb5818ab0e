"""The policy operators at the ends of their range, against the same 64-bit
definitions and counted bounds."""
import ctypes as C
import math

import pytest
import torch
import torch.autograd.forward_ad as fwad

from abmarl_amd import _native, learning
from abmarl_amd.learning import PolicyHeads
from tests import learning_reference as ref
from tests.test_learning import DTYPES, LAYOUTS, _all_calls, _gradients, check_loss, cuda, fragment, gen, gumbel

gpu = pytest.mark.gpu

NARROW = ['team', 'rtt', 'odd', 'w47']


def offsets(dtype):
    far = [1e3, 6e4] if dtype == torch.float16 else [1e3, 6e4, 1e6, 1.3e8, 2.6e8, 1e10, 1e20, 1e38]
    return far + [-v for v in far]


def far_inputs(heads, dtype, offset, seed, N, masked):
    """Rows around `offset` (row 0 equal to it throughout, row 1 around 0), ref
    logits, masks, actions, advantages and what the actions' log-probabilities
    were a little before."""
    g = gen(seed)
    shape = (N, heads.n_choices)
    z = offset + 1.7 * torch.randn(shape, generator=g, dtype=torch.float64)
    z[0] = offset
    z[1] -= offset
    z = z.to(dtype)
    k = (z.double() + 0.3 * torch.randn(shape, generator=g, dtype=torch.float64)).to(dtype)
    mask = None
    if masked:
        mask = (torch.rand(shape, generator=g) < 0.7).to(torch.uint8)
        mask[:2] = 1
        z = torch.where(mask == 0, torch.tensor(math.nan, dtype=dtype), z)
    noise = gumbel(shape, g)
    act, logp, _, _, _ = ref.sample(z, heads, noise, mask)
    old = (logp - 0.1 * torch.rand(N, generator=g)).float()      # no ratio at the border of the clipping
    valid = (torch.rand(N, generator=g) < 0.7).to(torch.uint8)
    valid[0] = 1
    return z, k, mask, noise, act, torch.randn(N, generator=g), old, valid


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('name', NARROW)
def test_loss_of_logits_of_any_size(name, masked, dtype):
    """Only differences of a head's logits count, however large they are."""
    heads = LAYOUTS[name]
    kw = dict(kl_coef=0.3, entropy_coef=0.02)
    for i, offset in enumerate(offsets(dtype)):
        z, k, mask, _, act, adv, old, valid = far_inputs(heads, dtype, offset, i, 67, masked)
        for r, v in ((None, valid), (k, None)):
            want = ref.policy_loss(z, act, adv, old, heads, r, v, mask, **kw)
            zc, actc, advc, oldc, rc, vc, mc = cuda(z, act, adv, old, r, v, mask)
            got = learning.policy_loss_grad(zc, actc, advc, oldc, heads, ref_logits=rc, valid=vc, choice_mask=mc, **kw)
            check_loss(got, want, dtype)


WIDE = {'w65': 67, 'w300': 31, 'w513': 9, 'w4100': 5, 'w12801': 5}


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('name', list(WIDE))
def test_wide_rows_of_any_size(name, masked, dtype):
    """One wide head: the waves and lanes of a row count its differences alike,
    whether or not a choice of theirs is masked, and a row that is not valid
    changes nothing for its neighbours; what is drawn has the loss's own log-probability."""
    heads, N = PolicyHeads([int(name[1:])]), WIDE[name]
    kw = dict(kl_coef=0.3, entropy_coef=0.02)
    near = [100.7, -12345.6, 31000.0]
    for i, offset in enumerate(near + offsets(dtype)):
        z, k, _, noise, _, adv, _, valid = far_inputs(heads, dtype, offset, i, N, False)
        mask = None
        if masked:                                               # the first choices of some rows: one wave's
            mask = torch.ones(z.shape, dtype=torch.uint8)
            mask[2:, 1:4] = 0
            z = torch.where(mask == 0, torch.tensor(math.nan, dtype=dtype), z)
        act, logp, entropy, e, e_h = ref.sample(z, heads, noise, mask)
        old = (logp - 0.05).float()
        zc, kc, mc, nc, advc, oldc = cuda(z, k, mask, noise, adv, old)
        got = learning.sample_actions(zc, heads, nc, mc)
        assert got.actions.cpu().equal(act), offset
        assert ref.near(got.logp, logp, e) <= 1, offset
        assert ref.near(got.entropy, entropy, e_h) <= 1, offset
        for r, v in ((None, valid), (k, None)):
            want = ref.policy_loss(z, act, adv, old, heads, r, v, mask, **kw)
            loss = learning.policy_loss_grad(zc, got.actions, advc, oldc, heads, ref_logits=None if r is None else kc,
                                             valid=None if v is None else v.cuda(), choice_mask=mc, **kw)
            check_loss(loss, want, dtype)


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('name', ['team', 'rtt', 'odd', 'w65', 'w4100', 'w200', 'mixed', 'cells', 'two_wide'])
def test_differences_past_the_largest_number(name, dtype):
    """Logits whose difference float32 does not hold: the far ones have
    probability 0, and nothing is NaN."""
    heads = LAYOUTS[name]
    N = 5
    z = torch.randn(N, heads.n_choices, generator=gen(4)).to(dtype)
    first = [s.start for s in ref.head_slices(heads)]
    z[0] = -3e38
    z[0, first] = 3e38
    z[1] = -1e38
    z[1, first] = 3e38
    z[2] = 3e38
    z[3] = -3e38
    act, logp, entropy, e, e_h = ref.sample(z, heads)
    zc = z.cuda()
    got = learning.sample_actions(zc, heads)
    assert got.actions.cpu().equal(act)
    assert ref.near(got.logp, logp, e) <= 1 and ref.near(got.entropy, entropy, e_h) <= 1
    adv = torch.randn(N, generator=gen(5))
    want = ref.policy_loss(z, act, adv, logp.float(), heads, z, kl_coef=0.5, entropy_coef=0.1)
    got = learning.policy_loss_grad(zc, *cuda(act, adv, logp.float()), heads, ref_logits=zc, kl_coef=0.5, entropy_coef=0.1)
    check_loss(got, want, dtype)


@gpu
@pytest.mark.parametrize('n,dtype', [(1 << 29, torch.float32), (1 << 30, torch.float32), (1 << 30, torch.bfloat16)])
def test_the_widest_heads(n, dtype):
    """Rows of 2 and 4 GiB, whose sizes in bytes pass 31 and 32 bits.  All logits are 0 but
    the last, -3: the sums are n - 1 ones, exact in float32 joined by parts, and e^-3."""
    heads = PolicyHeads([n])
    z = torch.zeros((1, n), dtype=dtype, device='cuda')
    z[0, n - 1] = -3.0
    total = n - 1 + math.exp(-3)
    logp, entropy = -math.log(total), math.log(total) + 3 * math.exp(-3) / total
    room = 16 * 2.0 ** -24 * entropy                             # the joined parts, the logarithm, the result
    got = learning.sample_actions(z, heads)
    assert got.actions.item() == 0
    assert abs(got.logp.item() - logp) <= room and abs(got.entropy.item() - entropy) <= room
    act = torch.full((1, 1), n - 2, dtype=torch.int32, device='cuda')
    one = torch.ones(1, device='cuda')
    g = learning.policy_loss_grad(z, act, one, got.logp, heads, grad_scale=float(n // 2))
    assert abs(g.logp.item() - logp) <= room and abs(g.loss.item() + 1) <= 2 * room
    half = torch.finfo(dtype).eps / 2
    for j, want in ((0, 1 / total), (100, 1 / total), (n // 2, 1 / total), (n - 3, 1 / total), (n - 2, 1 / total - 1),
                    (n - 1, math.exp(-3) / total)):
        want *= n // 2
        assert abs(g.grad[0, j].item() - want) <= abs(want) * (half + 4 * room), j
    assert int((g.grad > 0).sum()) == n - 1
    del g
    z[0, n - 2] = 90.0                                           # the only one left
    got = learning.sample_actions(z, heads)
    assert got.actions.item() == n - 2 and got.logp.item() == 0.0


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('bad', [math.nan, math.inf])
@pytest.mark.parametrize('name', ['team', 'rtt', 'odd', 'w47', 'w65', 'w4100', 'w200', 'cells', 'mixed'])
def test_a_bad_logit_at_the_chosen_place_shows(name, bad, dtype):
    """A NaN or +inf logit that was chosen gives NaN in its row's
    log-probability, policy term and gradient; other rows are as without it."""
    heads = LAYOUTS[name]
    N = 5
    z = torch.randn(N, heads.n_choices, generator=gen(6)).to(dtype)
    act, logp, _, _, _ = ref.sample(z, heads)
    args = cuda(act, torch.randn(N, generator=gen(7)), logp.float())
    kw = dict(entropy_coef=0.0, denominator=1.0)
    clean = learning.policy_loss_grad(z.cuda(), *args, heads, **kw)
    s, d = ref.head_slices(heads)[0], heads.slots[0]
    z[2, s.start + int(act[2, d]) - heads.low[0]] = bad
    got = learning.policy_loss_grad(z.cuda(), *args, heads, **kw)
    assert math.isnan(got.logp[2].item()) and math.isnan(got.stats[0].item()) and math.isnan(got.loss.item())
    assert torch.isnan(got.grad[2].float()).all().item()
    rest = [0, 1, 3, 4]
    # a bad row may send its wave another way round: equal within two roundings of the sums
    assert torch.allclose(got.logp[rest], clean.logp[rest], rtol=0, atol=heads.n_heads * 2.0 ** -20)
    assert torch.isfinite(got.grad[rest].float()).all().item()


@gpu
def test_shared_gates_of_no_channels():
    """A batch of no envs or lanes is no error, and its gates' gradients are 0."""
    for shape, gshape, cshape in (((5, 0), (5,), (5,)), ((5, 3, 0), (5, 3), (5, 3)), ((5, 0, 4), (5, 0), (5,)),
                                  ((5, 3, 0), (5, 3, 1), (5, 3, 0))):
        x = torch.zeros(shape, device='cuda', requires_grad=True)
        gate = torch.ones(gshape, device='cuda', requires_grad=True)
        state = torch.zeros(shape[1:], device='cuda', requires_grad=True)
        cut = torch.zeros(cshape, dtype=torch.uint8, device='cuda')
        junk = torch.full(gshape, 7.0, device='cuda')            # what freed memory may hold
        del junk
        h, last = learning.linear_recurrence(gate, x, state, cut=cut)
        assert h.shape == shape and last.shape == shape[1:]
        dg, dx, ds = torch.autograd.grad((h, last), (gate, x, state), (torch.ones_like(h), torch.ones_like(last)))
        assert dg.shape == gshape and not dg.any().item() and dx.shape == shape and ds.shape == shape[1:]


def test_forward_mode_refused():
    """A tangent would be lost: the call says so (before it looks for a GPU)."""
    with fwad.dual_level():
        x = torch.ones(4, 3)
        dual = fwad.make_dual(x, x)
        for args in ((0.5, dual), (dual, x), (0.5, x, fwad.make_dual(x[0], x[0]))):
            with pytest.raises(NotImplementedError, match='forward'):
                learning.linear_recurrence(*args)
        z = torch.zeros(4, 8)
        rest = torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4), torch.zeros(4), LAYOUTS['team']
        with pytest.raises(NotImplementedError, match='forward'):
            learning.policy_loss_grad(fwad.make_dual(z, z), *rest)
        with pytest.raises(RuntimeError, match='no CPU fallback'):          # no tangent, no complaint
            learning.policy_loss_grad(z, *rest)


@pytest.mark.parametrize('mode', ['next_step', 'same_step'])
def test_memory_is_cut_where_episodes_begin(mode):
    """Against the envs' own step counters: an observation is an episode's
    first where no step was taken in it.  The one behind an END, before the
    reset (next_step), is cut too."""
    K, E, horizon = 60, 40, 7
    _, _, _, all_done, before, steps, _, _, _ = fragment(K, E, 2, 3, mode, horizon)
    marks = ref.marks(all_done, steps, horizon, mode, before)
    want = torch.zeros((K + 1, E), dtype=torch.uint8)
    for e in range(E):
        n, ended = int(steps[e]), bool(before[e])
        for t in range(K + 1):
            want[t, e] = n == 0 or (mode == 'next_step' and t > 0 and bool(all_done[t - 1, e]) and not reset)
            if t == K:
                break
            reset = mode == 'next_step' and (ended or n >= horizon)
            n, ended = (0, False) if reset else (n + 1, bool(all_done[t, e]))
            if mode == 'same_step' and (ended or n >= horizon):
                n = 0
    got = learning.fragment_cuts(marks, steps)
    assert got.equal(want)
    assert learning.fragment_cuts(marks)[1:].equal(want[1:]) and not learning.fragment_cuts(marks)[0].any()
    assert learning.fragment_cuts(marks[:0], steps).equal(want[:1])


@pytest.mark.parametrize('kw,word', [
    (dict(marks=torch.zeros(3, 2)), 'marks'), (dict(marks=torch.zeros(3, dtype=torch.uint8)), 'marks'),
    (dict(steps=torch.zeros(2)), 'steps'), (dict(steps=torch.zeros(3, dtype=torch.int32)), 'steps')])
def test_cuts_refused(kw, word):
    with pytest.raises(ValueError, match=word):
        learning.fragment_cuts(**{**dict(marks=torch.zeros(3, 2, dtype=torch.uint8)), **kw})


@gpu
def test_two_streams_at_once_give_their_own_numbers():
    """Every round's outputs of two streams that run at once, bit for bit."""
    a, _ = _all_calls(11)
    b, _ = _all_calls(12)
    want = [[t.clone() for t in f()] for f in (a, b)]
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(6):
        for i, (s, f) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i].append(f())
    torch.cuda.synchronize()
    for w, rounds in zip(want, got):
        for out in rounds:
            assert len(out) == len(w)
            for x, y in zip(w, out):
                assert (x == y).logical_or(torch.isnan(x.float()) & torch.isnan(y.float())).all().item()


@gpu
def test_two_to_the_32_shared_gates():
    """More gates than a launch has threads.  Only the last steps' inputs are not 0,
    so their gradients are those of the last steps alone, and the others 0."""
    T, tail = 1 << 31, 40
    if torch.cuda.mem_get_info()[0] < 160e9:
        pytest.skip('132 GB are needed')
    g = gen(8)
    part = torch.randn((tail, 2, 3), generator=g).bfloat16()
    dlast = torch.randn((2, 3), generator=g)
    x = torch.zeros((T, 2, 3), dtype=torch.bfloat16, device='cuda')
    x[-tail:] = part.cuda()
    gate = torch.full((T, 2), 0.5, dtype=torch.bfloat16, device='cuda', requires_grad=True)
    _, last = learning.linear_recurrence(gate, x, torch.zeros((2, 3), device='cuda'))
    dg, = torch.autograd.grad(last, gate, dlast.cuda())
    (want, _, _), e, _, _ = _gradients(torch.full((tail, 2), 0.5), part, torch.zeros((2, 3)), None, False,
                                       torch.zeros((tail, 2, 3)), dlast)
    assert ref.near(dg[-tail:], want, e, torch.bfloat16) <= 1 and want.any()
    assert not (dg[:-tail] != 0).any().item()
    del x, gate, last, dg
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize('name', ['team', 'rtt', 'w65', 'w4100', 'cells'])
def test_no_advantage_beside_a_ratio_past_the_largest_number(name):
    """A row without an advantage has no policy term, however far its action's
    probability has risen; with one, the clipped term."""
    heads = LAYOUTS[name]
    N = 6
    z = torch.randn(N, heads.n_choices, generator=gen(9))
    act, logp, _, _, _ = ref.sample(z, heads)
    old = (logp - torch.tensor([200.0, 0.05, 5.0, 300.0, 0.0, 89.0])).float()
    adv = torch.tensor([0.0, 1.0, 2.0, 0.0, 0.0, 0.0])
    want = ref.policy_loss(z, act, adv, old, heads, entropy_coef=0.1)
    args = cuda(act, adv, old)
    check_loss(learning.policy_loss_grad(z.cuda(), *args, heads, entropy_coef=0.1), want, torch.float32)
    old[0] = old[3] = -math.inf                                  # impossible before, now drawn
    check_loss(learning.policy_loss_grad(z.cuda(), *cuda(act, adv, old), heads, entropy_coef=0.1), want, torch.float32)


@pytest.mark.parametrize('change,word', [
    (dict(denominator=1e-60), 'denominator'), (dict(denominator=1e39), 'denominator'), (dict(kl_coef=1e39), 'kl_coef'),
    (dict(entropy_coef=-1e39), 'entropy_coef'), (dict(clip=1e39), 'clip'), (dict(clip=(0.2, 1e300)), 'clip')])
def test_numbers_that_float32_does_not_hold_are_refused(change, word):
    """A denominator that float32 rounds to 0 would have been the number of
    valid rows in its place."""
    args = (torch.zeros(4, 8), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4), torch.zeros(4), LAYOUTS['team'])
    for fn in (learning.policy_loss, learning.policy_loss_grad):
        with pytest.raises(ValueError, match=word):
            fn(*args, **change)
    with pytest.raises(ValueError, match='gate'):
        learning.linear_recurrence(1e39, torch.zeros(3, 2))


def test_c_entry_refuses_values_past_int32():
    """Heads whose values an int32 action does not hold, given past PolicyHeads' own check."""
    _native.build_learn()
    L = _native.learn_lib()
    one = C.c_void_p(8)
    ints = C.c_int32 * 2
    heads = learning._Heads(2, 2, ints(3, 5), ints(0, 2 ** 31 - 4), ints(0, 1))
    args = C.addressof(heads), 0, 4, one, 8, None, None, 0, one, None, None, None
    assert L.gw_policy_sample(*args) == -1 and b'int32' in L.gw_learn_last_error()


@gpu
@pytest.mark.parametrize('name', ['team', 'rtt', 'w65', 'w300', 'w4100', 'cells'])
def test_ref_of_another_size_than_the_logits(name):
    """KL does not change when all of ref's logits, or all of the policy's, move together."""
    heads = LAYOUTS[name]
    N = 40 if heads.n_choices < 400 else 5
    z0, k0 = (8 * torch.randn(N, heads.n_choices, generator=gen(i)).round() for i in (1, 2))
    act = ref.sample(z0, heads)[0]
    adv, valid = torch.randn(N, generator=gen(3)), (torch.rand(N, generator=gen(4)) < 0.7).to(torch.uint8)
    for dz, dk in ((0.0, 2.0 ** 26), (-2.0 ** 26, 0.0), (2.0 ** 14, -2.0 ** 26), (2.0 ** 26, 2.0 ** 26)):
        z, k = z0 + dz, k0 + dk                                  # (steps of 8: exact)
        want = ref.policy_loss(z, act, adv, torch.full((N,), -3.0), heads, k, valid, kl_coef=0.3, entropy_coef=0.02)
        got = learning.policy_loss_grad(*cuda(z, act, adv), torch.full((N,), -3.0).cuda(), heads, ref_logits=k.cuda(),
                                        valid=valid.cuda(), kl_coef=0.3, entropy_coef=0.02)
        # the bounds count |logits - ref| beside each other: here of the rows as they were
        near = ref.policy_loss(z0, act, adv, torch.full((N,), -3.0), heads, k0, valid, kl_coef=0.3, entropy_coef=0.02)
        assert abs(near['loss'] - want['loss']) <= 1e-9 * (1 + abs(near['loss']))
        check_loss(got, near, torch.float32)


@gpu
def test_policy_loss_refuses_forward_mode():
    with fwad.dual_level():
        z = torch.zeros(4, 8, device='cuda')
        rest = torch.zeros(4, 3, dtype=torch.int32).cuda(), torch.zeros(4).cuda(), torch.zeros(4).cuda(), LAYOUTS['team']
        with pytest.raises(NotImplementedError):
            learning.policy_loss(fwad.make_dual(z, z), *rest)
