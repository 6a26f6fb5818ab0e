"""The policy operators (abmarl_amd.learning) against their definitions in 64
bits (learning_reference.py): every layout, type, mask and edge; refusals on
the CPU.  Actions, valid flags and marks are compared exactly; numbers within
what float32 arithmetic and one rounding to the output's type allow, from
bounds counted in learning_reference.py."""
import ctypes as C
import math
import os
import re

import pytest
import torch

from abmarl_amd import _native, learning
from abmarl_amd.learning import PolicyHeads
from tests import learning_reference as ref

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

TEAM = PolicyHeads([3, 3, 2], low=[-1, -1, 0])
RTT = PolicyHeads([5, 5] + [2] * 9, low=[-2, -2] + [0] * 9)
CROSS = PolicyHeads([5], slots=[0], act_dim=3)


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def gumbel(shape, g):
    return -torch.log(torch.empty(shape).exponential_(generator=g))


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


# ------------------------------------------------------------ CPU: refusals
def test_header_symbols_are_exported_and_mirrored():
    _native.build_learn()
    L = _native.learn_lib()
    txt = re.sub(r'/\*.*?\*/', '', open(os.path.join(ROOT, 'include', 'gw_learn.h')).read(), flags=re.S)
    names = sorted(set(re.findall(r'\b(gw_[a-z_]+)\s*\(', txt)))
    assert len(names) >= 10 and set(names) == set(_native.LEARN_SIGNATURES)
    assert all(hasattr(L, n) for n in names)
    defines = dict(re.findall(r'#define\s+(GW_\w+)\s+(\d+)', txt))
    assert int(defines['GW_RECURRENCE_SEGMENT']) == learning.SEGMENT
    assert int(defines['GW_MAX_HEADS']) == learning.MAX_HEADS
    assert [int(defines['GW_MARK_' + k]) for k in ('END', 'TRUNCATED', 'RESET', 'SKIP')] == \
        [learning.MARK_END, learning.MARK_TRUNCATED, learning.MARK_RESET, learning.MARK_SKIP]
    assert L.gw_learn_abi_version() == 1


@pytest.mark.parametrize('kw,word', [
    (dict(sizes=[]), 'heads'), (dict(sizes=[2] * 257), 'heads'), (dict(sizes=[3, 0]), 'at least one'),
    (dict(sizes=[3], low=[0, 0]), 'one value per head'), (dict(sizes=[3, 3], slots=[1, 1]), 'different columns'),
    (dict(sizes=[3], slots=[-1]), 'different columns'), (dict(sizes=[3], slots=[2], act_dim=2), 'different columns'),
    (dict(sizes=[2 ** 30, 1]), 'at most'), (dict(sizes=[5], low=[2 ** 31 - 2]), 'int32')])
def test_heads_refused(kw, word):
    with pytest.raises(ValueError, match=word):
        PolicyHeads(**kw)


def test_loss_of_actions_far_outside():
    """Differences of actions and lows past int32 are no choice either."""
    z = torch.zeros(2, 3)
    heads = PolicyHeads([3], low=[2 ** 31 - 4])
    act = torch.tensor([[-2 ** 31], [2 ** 31 - 3]], dtype=torch.int32)
    want = ref.policy_loss(z, act, torch.ones(2), torch.zeros(2), heads)
    assert want['logp'][0] == -math.inf and abs(float(want['logp'][1]) + math.log(3)) < 1e-12


def _loss_kw(N=4, heads=TEAM):
    return dict(logits=torch.zeros(N, heads.n_choices), actions=torch.zeros(N, heads.act_dim, dtype=torch.int32),
                advantage=torch.zeros(N), old_logp=torch.zeros(N), heads=heads)


@pytest.mark.parametrize('change,word', [
    (dict(logits=torch.zeros(4, 7)), 'logits'), (dict(logits=torch.zeros(4, 8).double()), 'logits'),
    (dict(logits=torch.zeros(8, 4).t()), 'side by side'), (dict(logits=[1.0]), 'tensor'),
    (dict(logits=torch.zeros(1, 8).expand(4, 8)), 'overlap'),
    (dict(actions=torch.zeros(4, 3)), 'actions'), (dict(actions=torch.zeros(4, 2, dtype=torch.int32)), 'actions'),
    (dict(advantage=torch.zeros(5)), 'advantage'), (dict(advantage=torch.zeros(4).half()), 'advantage'),
    (dict(advantage=torch.zeros(8)[::2]), 'contiguous'), (dict(old_logp=torch.zeros(4, 1)), 'old_logp'),
    (dict(old_logp=torch.zeros(4, requires_grad=True)), 'no gradient'),
    (dict(ref_logits=torch.zeros(4, 8).half()), 'ref_logits'), (dict(ref_logits=torch.zeros(3, 8)), 'ref_logits'),
    (dict(valid=torch.zeros(4)), 'valid'), (dict(valid=torch.zeros(3, dtype=torch.uint8)), 'valid'),
    (dict(choice_mask=torch.ones(3, 8, dtype=torch.uint8)), 'choice_mask'),
    (dict(choice_mask=torch.ones(8)), 'choice_mask'), (dict(choice_mask=5), 'choice_mask'),
    (dict(clip=-0.1), 'clip'), (dict(clip=(0.1, math.inf)), 'clip'), (dict(clip=math.nan), 'clip'),
    (dict(kl_coef=math.nan), 'kl_coef'), (dict(entropy_coef=math.inf), 'entropy_coef'),
    (dict(denominator=0), 'denominator'), (dict(denominator=torch.zeros(1)), 'denominator')])
def test_loss_refused(change, word):
    for fn in (learning.policy_loss, learning.policy_loss_grad):
        with pytest.raises(ValueError, match=word):
            fn(**{**_loss_kw(), **change})


def test_no_cpu_fallback():
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        learning.policy_loss(**_loss_kw())
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        learning.sample_actions(torch.zeros(4, 8), TEAM)
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        learning.linear_recurrence(0.5, torch.zeros(3, 2))
    with pytest.raises(RuntimeError, match='no CPU fallback'):
        learning.fragment_marks(torch.zeros(2, 3, dtype=torch.uint8))


@pytest.mark.parametrize('kw,word', [
    (dict(noise=torch.zeros(4, 8).half()), 'noise'), (dict(noise=torch.zeros(4, 7)), 'noise'),
    (dict(out=torch.zeros(4, 3)), 'out'), (dict(out=torch.zeros(4, 4, dtype=torch.int32)), 'out')])
def test_sample_refused(kw, word):
    with pytest.raises(ValueError, match=word):
        learning.sample_actions(torch.zeros(4, 8), TEAM, **kw)


@pytest.mark.parametrize('gate,x,kw,word', [
    (0.5, torch.zeros(3), {}, 'x'), (0.5, torch.zeros(3, 2).double(), {}, 'x'),
    (0.5, torch.zeros(3, 4)[:, ::2], {}, 'contiguous'),
    (math.inf, torch.zeros(3, 2), {}, 'gate'), (torch.zeros(3, 3), torch.zeros(3, 2), {}, 'gate'),
    (torch.zeros(3, 2).half(), torch.zeros(3, 2).bfloat16(), {}, 'gate'),
    (0.5, torch.zeros(3, 2), dict(state=torch.zeros(3)), 'state'),
    (0.5, torch.zeros(3, 2).half(), dict(state=torch.zeros(2).half()), 'state'),
    (0.5, torch.zeros(3, 2, 2), dict(cut=torch.zeros(3, 1, 2, dtype=torch.uint8)), 'cut'),
    (0.5, torch.zeros(3, 2), dict(cut=torch.zeros(3)), 'cut')])
def test_recurrence_refused(gate, x, kw, word):
    with pytest.raises(ValueError, match=word):
        learning.linear_recurrence(gate, x, **kw)


def _adv_kw(K=3, E=2, A=2):
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    return dict(reward=torch.zeros(K, E, A).double(), value=torch.zeros(K + 1, E, A), done=u8(K, E, A),
                marks=u8(K, E), live=u8(E, A))


@pytest.mark.parametrize('change,word', [
    (dict(reward=torch.zeros(3, 2, 2).half()), 'reward'), (dict(reward=torch.zeros(3, 4)), 'reward'),
    (dict(value=torch.zeros(3, 2, 2)), 'value'), (dict(done=torch.zeros(3, 2, 2)), 'done'),
    (dict(marks=torch.zeros(3, 2)), 'marks'), (dict(live=torch.zeros(2, dtype=torch.uint8)), 'live'),
    (dict(acts=torch.zeros(3, dtype=torch.uint8)), 'acts'), (dict(gamma=math.nan), 'gamma')])
def test_advantages_refused(change, word):
    with pytest.raises(ValueError, match=word):
        learning.advantages(**{**_adv_kw(), **change})


@pytest.mark.parametrize('kw,word', [
    (dict(all_done=torch.zeros(3, dtype=torch.uint8)), 'all_done'), (dict(autoreset='none'), 'autoreset'),
    (dict(horizon=-1), 'horizon'), (dict(steps=torch.zeros(2)), 'steps'),
    (dict(err=torch.zeros(3, dtype=torch.int32)), 'err')])
def test_marks_refused(kw, word):
    with pytest.raises(ValueError, match=word):
        learning.fragment_marks(**{**dict(all_done=torch.zeros(3, 2, dtype=torch.uint8)), **kw})


def test_c_entries_refuse_without_a_gpu():
    """The C-ABI's own checks come before anything touches a device."""
    _native.build_learn()
    L = _native.learn_lib()
    one = C.c_void_p(8)
    heads = TEAM._p
    bad = [
        (L.gw_policy_sample, (None, 0, 4, one, 8, None, None, 0, one, None, None, None), 'heads'),
        (L.gw_policy_sample, (heads, 3, 4, one, 8, None, None, 0, one, None, None, None), 'dtype'),
        (L.gw_policy_sample, (heads, 0, -1, one, 8, None, None, 0, one, None, None, None), 'rows'),
        (L.gw_policy_sample, (heads, 0, 4, None, 8, None, None, 0, one, None, None, None), 'logits'),
        (L.gw_policy_sample, (heads, 0, 4, one, 7, None, None, 0, one, None, None, None), 'apart'),
        (L.gw_policy_sample, (heads, 0, 4, one, 8, None, one, 3, one, None, None, None), 'mask'),
        (L.gw_policy_sample, (heads, 0, 4, one, 8, None, None, 0, None, None, None, None), 'actions')]
    loss = [heads, 0, 4, one, 8, None, 0, one, one, one, None, None, 0, 0.2, 0.2, 0.0, 0.0, 0.0, None, 1.0, None,
            one, one, one, one, one, 1 << 20, None]
    for i, v, word in [(7, None, 'actions'), (13, -1.0, 'clip'), (15, math.nan, 'coefficient'), (25, None, 'workspace'),
                       (26, 8, 'workspace'), (25, C.c_void_p(12), 'workspace'), (22, None, 'both')]:
        bad.append((L.gw_policy_loss, loss[:i] + [v] + loss[i + 1:], word))
    bad.append((L.gw_policy_loss, loss[:21] + [None, None, None, None] + loss[25:], 'nothing'))
    rec = [0, 0, 3, 4, one, one, 1, 0.0, None, 1, None, 0, one, one, None, one, 1 << 30, None]
    for i, v, word in [(0, 5, 'dtype'), (1, 2, 'gate_dtype'), (2, -1, 'steps'), (4, None, 'x'), (6, 3, 'gate_span'),
                       (12, None, 'h')]:
        bad.append((L.gw_recurrence, rec[:i] + [v] + rec[i + 1:], word))
    bad.append((L.gw_recurrence, rec[:8] + [one, 3] + rec[10:], 'cut_span'))
    back = [0, 0, 3, 6, one, one, 3, 0.0, None, 1, one, 0, None, None, one, one, None, None, 0, None]
    bad.append((L.gw_recurrence_backward, back, 'workspace'))
    bad.append((L.gw_recurrence_backward, back[:5] + [None] + back[6:], 'dgate'))
    bad.append((L.gw_recurrence_backward, back[:10] + [None] + back[11:], 'carry'))
    bad.append((L.gw_fragment_marks, (2, 2, one, None, None, None, 0, 0, one, None), 'autoreset'))
    bad.append((L.gw_fragment_marks, (2, 2, None, None, None, None, 0, 1, one, None), 'null'))
    bad.append((L.gw_advantages, (0, 1, 2, 2, 0, *[one] * 5, None, .9, .9, one, one, one, one, 1 << 30, None), 'lanes'))
    bad.append((L.gw_advantages, (0, 1, 2, 2, 2, *[one] * 4, None, None, .9, .9, one, one, one, one, 1 << 30, None), 'null'))
    for fn, args, word in bad:
        assert fn(*args) == -1, (fn.__name__, word)
        assert word in L.gw_learn_last_error().decode(), (fn.__name__, word, L.gw_learn_last_error())


def test_reference_gradients_against_differences():
    """The 64-bit definition's own gradients, by central differences."""
    g = gen(3)
    N, heads = 5, TEAM
    z = torch.randn(N, 8, generator=g, dtype=torch.float64)
    k = z + 0.3 * torch.randn(N, 8, generator=g, dtype=torch.float64)
    act, logp, _, _, _ = ref.sample(z.float(), heads, gumbel((N, 8), g))
    adv, old = torch.randn(N, generator=g), (logp - 0.1).float()
    kw = dict(ref=k, kl_coef=0.3, entropy_coef=0.05)
    want = ref.policy_loss(z, act, adv, old, heads, **kw)['grad']
    for r in range(N):
        for j in range(8):
            h = 1e-5
            d = torch.zeros_like(z)
            d[r, j] = h
            up, dn = (ref.policy_loss(z + s * d, act, adv, old, heads, **kw)['loss'] for s in (1, -1))
            assert abs((up - dn) / (2 * h) - float(want[r, j])) < 1e-8


# --------------------------------------------------------------- GPU: sample
LAYOUTS = {
    'team': TEAM, 'rtt': RTT, 'cross': CROSS, 'one': PolicyHeads([1]), 'two': PolicyHeads([1, 2], slots=[2, 0]),
    'odd': PolicyHeads([7, 1, 31], low=[-3, 5, 0], slots=[3, 0, 1], act_dim=6),
    'pairs20': PolicyHeads([2] * 20), 'ones48': PolicyHeads([1] * 48),
    'w63': PolicyHeads([63]), 'w64': PolicyHeads([64]), 'w65': PolicyHeads([65]), 'w200': PolicyHeads([129, 71]),
    'w513': PolicyHeads([513]), 'w1031': PolicyHeads([1031]), 'w4100': PolicyHeads([4100]),
    'w40003': PolicyHeads([40003]), 'two_wide': PolicyHeads([5000, 3, 5000]),
    'many': PolicyHeads([15, 15] + [2] * 225), 'cells': PolicyHeads([17, 17] + [4] * 49), 'mixed': PolicyHeads([3, 1500, 2, 700]),
    'w19': PolicyHeads([7, 7, 5]), 'w24': PolicyHeads([11, 11, 2]), 'w33': PolicyHeads([15, 15, 3]), 'w47': PolicyHeads([9, 31, 7]),
    'w129': PolicyHeads([129]), 'w250': PolicyHeads([250]), 'w257': PolicyHeads([257]), 'w300': PolicyHeads([300]),
    'w1023': PolicyHeads([1000, 23]), 'w1024': PolicyHeads([1000, 24]),
}
ROWS = {'w513': 9, 'w1031': 5, 'w4100': 3, 'many': 7, 'mixed': 4, 'w200': 13, 'w40003': 2, 'two_wide': 2, 'cells': 11,
        'w1023': 5, 'w1024': 5}


def inputs(name, dtype, seed, masked, lanes=None):
    heads = LAYOUTS[name]
    g = gen(seed)
    N = ROWS.get(name, 67)
    z = (1.7 * torch.randn(N, heads.n_choices, generator=g)).to(dtype)
    mask = None
    if masked:
        M = N if lanes is None else lanes
        mask = (torch.rand(M, heads.n_choices, generator=g) < 0.7).to(torch.uint8)
        for d, s in enumerate(ref.head_slices(heads)):           # some heads have nothing left
            mask[d % M, s] = 0
        mask[-1] = 0
        mask[0, 0] = 1
        m = mask.repeat(N // M, 1)
        bad = torch.tensor([math.nan, math.inf, -math.inf, 1.0])[torch.randint(4, z.shape, generator=g)].to(dtype)
        z = torch.where(m == 0, bad, z)                          # what stands there is never used
        low = torch.rand(z.shape, generator=g) < 0.05
        z = torch.where((m != 0) & low, torch.tensor(torch.finfo(dtype).min, dtype=dtype), z)
        low = torch.rand(z.shape, generator=g) < 0.05
        z = torch.where((m != 0) & low, torch.tensor(-math.inf, dtype=dtype), z)
    return heads, z, mask, gumbel(z.shape, g), g


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('name', list(LAYOUTS))
def test_sample(name, masked, dtype):
    heads, z, mask, noise, _ = inputs(name, dtype, 1, masked)
    for n in (noise, None):
        want, logp, entropy, e_logp, e_h = ref.sample(z, heads, n, None if mask is None else mask)
        zc, nc, mc = cuda(z, n, mask)
        got = learning.sample_actions(zc, heads, nc, mc)
        assert got.actions.cpu().equal(want)
        assert ref.near(got.logp, logp, e_logp) <= 1
        assert ref.near(got.entropy, entropy, e_h) <= 1


@gpu
def test_sample_ties_take_the_lowest():
    heads = PolicyHeads([300, 5])
    z = torch.zeros(4, 305)
    z[1, 7] = z[1, 70] = z[1, 299] = 2.0
    z[2, 300:] = -1.0
    got = learning.sample_actions(z.cuda(), heads).actions.cpu()
    assert got.tolist() == [[0, 0], [7, 0], [0, 0], [0, 0]]


@gpu
def test_sample_lane_masks_strides_and_out():
    """A mask per lane, rows of a wider matrix, actions into a buffer that a
    user keeps; the columns between rows are left alone."""
    g = gen(4)
    E, A = 5, 6
    wide = torch.randn(E * A, 20, generator=g).cuda()
    z = wide[:, 3:11].view(E, A, 8)
    mask = (torch.rand(A, 8, generator=g) < 0.6).to(torch.uint8)
    noise = gumbel((E, A, 8), g)
    want, logp, _, e, _ = ref.sample(z.cpu().reshape(-1, 8), TEAM, noise.reshape(-1, 8), mask.repeat(E, 1))
    out = torch.full((E, A, 3), 77, dtype=torch.int32, device='cuda')
    got = learning.sample_actions(z, TEAM, noise.cuda(), mask.cuda(), out=out)
    assert got.actions is out and out.cpu().reshape(-1, 3).equal(want)
    assert ref.near(got.logp.reshape(-1), logp, e) <= 1


@gpu
def test_sample_many_rows():
    """More rows than one launch has workgroups, the last one alone."""
    for name, N in (('team', 70001), ('w200', 20001), ('w1031', 9001)):
        heads = LAYOUTS[name]
        z = torch.randn(N, heads.n_choices, generator=gen(5))
        noise = gumbel(z.shape, gen(6))
        got = learning.sample_actions(z.cuda(), heads, noise.cuda()).actions.cpu()
        want = torch.stack([(z + noise)[:, s].argmax(1).int() + lo for s, lo in zip(ref.head_slices(heads), heads.low)], 1)
        assert got.equal(want)


# ----------------------------------------------------------------- GPU: loss
def loss_inputs(name, dtype, seed, masked, lanes=None):
    heads, z, mask, noise, g = inputs(name, dtype, seed, masked, lanes)
    N = z.shape[0]
    m = None if mask is None else mask.repeat(N // mask.shape[0], 1)
    act, logp, _, _, _ = ref.sample(z, heads, noise, m)
    k = (torch.where(torch.isfinite(z.float()), z.float(), 0) + 0.3 * torch.randn(z.shape, generator=g)).to(dtype)
    d = 0.3 * torch.randn(N, generator=g)
    for b in (math.log(0.8), math.log(1.2)):                     # no ratio next to the border of the clipping
        d = torch.where((d - b).abs() < 1e-3, b + 2e-3, d)
    return heads, z, mask, k, act, torch.randn(N, generator=g), (logp - d).float(), \
        (torch.rand(N, generator=g) < 0.7).to(torch.uint8), g


def check_loss(got, want, dtype, grad=None):
    assert ref.near(got.loss, torch.tensor(want['loss'], dtype=torch.float64), want['e_loss']) <= 1
    assert ref.near(got.stats, want['stats'], torch.tensor(want['e_stats'], dtype=torch.float64)) <= 1
    assert float(got.count) == want['count']
    assert ref.near(got.logp, want['logp'], want['e_logp']) <= 1
    grad = got.grad if grad is None else grad
    assert grad.dtype == dtype and ref.near(grad, want['grad'], want['e_grad'], dtype) <= 1


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('masked', [False, True])
@pytest.mark.parametrize('name', list(LAYOUTS))
def test_policy_loss(name, masked, dtype):
    heads, z, mask, k, act, adv, old, valid, _ = loss_inputs(name, dtype, 2, masked)
    kw = dict(kl_coef=0.3, entropy_coef=0.02)
    for use_ref, use_valid in ((True, False), (False, True), (True, True)):
        r, v = k if use_ref else None, valid if use_valid else None
        want = ref.policy_loss(z, act, adv, old, heads, r, v, mask, **kw)
        zc, actc, advc, oldc, rc, vc, mc = cuda(z, act, adv, old, r, v, mask)
        got = learning.policy_loss_grad(zc, actc, advc, oldc, heads, ref_logits=rc, valid=vc, choice_mask=mc, **kw)
        check_loss(got, want, dtype)
        zc.requires_grad_()
        got = learning.policy_loss(zc, actc, advc, oldc, heads, ref_logits=rc, valid=vc, choice_mask=mc, **kw)
        got.loss.backward()
        check_loss(got, want, dtype, zc.grad)


@gpu
def test_policy_loss_small_rows_and_nothing():
    """One row; no row; no valid row; a row whose every choice is masked."""
    for N, valid in ((1, None), (0, None), (3, [0, 0, 0]), (2, [0, 1])):
        g = gen(N)
        z = torch.randn(N, 8, generator=g)
        act, logp, _, _, _ = ref.sample(z, TEAM, None)
        v = None if valid is None else torch.tensor(valid, dtype=torch.bool)
        want = ref.policy_loss(z, act, torch.ones(N), logp.float(), TEAM, valid=v, entropy_coef=0.1)
        zc, actc, advc, oldc, vc = cuda(z, act, torch.ones(N), logp.float(), v)
        got = learning.policy_loss_grad(zc, actc, advc, oldc, TEAM, valid=vc, entropy_coef=0.1)
        check_loss(got, want, torch.float32)
        zc.requires_grad_()
        got = learning.policy_loss(zc, actc, advc, oldc, TEAM, valid=vc, entropy_coef=0.1)
        got.loss.backward()
        check_loss(got, want, torch.float32, zc.grad)
    z = torch.full((2, 8), math.nan)
    mask = torch.zeros(1, 8, dtype=torch.uint8)
    zero = torch.zeros(2, 3, dtype=torch.int32)
    got = learning.policy_loss_grad(*cuda(z, zero, torch.ones(2), torch.zeros(2)), TEAM, choice_mask=mask.cuda(),
                                    ref_logits=z.cuda(), kl_coef=1.0)
    # nothing to choose: L = 0, ratio 1, no KL, no entropy, no gradient
    assert got.loss.item() == -1.0 and got.stats.tolist() == [-1.0, 0.0, 0.0, 0.0]
    assert not got.grad.any().item() and got.logp.tolist() == [0.0, 0.0]


@gpu
def test_policy_loss_impossible_actions():
    """Actions outside their heads, or of masked choices, have probability 0."""
    z = torch.randn(5, 8, generator=gen(1))
    act = torch.tensor([[-1, -1, 2], [5, 0, 0], [-2 ** 31, 0, 1], [1, 1, 1], [2 ** 31 - 1, 0, 0]], dtype=torch.int32)
    mask = torch.ones(5, 8, dtype=torch.uint8)
    mask[3, 2] = 0                                               # row 3's first choice
    adv = torch.tensor([1.0, -1.0, 1.0, -2.0, 0.5])
    want = ref.policy_loss(z, act, adv, torch.zeros(5), TEAM, mask=mask, entropy_coef=0.1)
    got = learning.policy_loss_grad(*cuda(z, act, adv, torch.zeros(5)), TEAM, choice_mask=mask.cuda(), entropy_coef=0.1)
    assert (got.logp == -math.inf).all().item()
    check_loss(got, want, torch.float32)
    for sizes in ([3], [100], [3, 100]):                         # differences past int32, in every kernel
        heads = PolicyHeads(sizes, low=[2 ** 31 - 1 - n for n in sizes])
        act = torch.tensor([[-2 ** 31] * len(sizes), [2 ** 31 - 2] * len(sizes)], dtype=torch.int32)
        z = torch.randn(2, sum(sizes), generator=gen(2))
        want = ref.policy_loss(z, act, torch.ones(2), torch.zeros(2), heads)
        check_loss(learning.policy_loss_grad(*cuda(z, act, torch.ones(2), torch.zeros(2)), heads), want, torch.float32)


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_policy_loss_lanes_strides_denominator_scale(dtype):
    heads, z, mask, k, act, adv, old, valid, g = loss_inputs('odd', dtype, 7, True, lanes=67)
    N, Cn = z.shape
    wide = torch.full((N, Cn + 13), math.nan, dtype=dtype)
    wide[:, 5:5 + Cn] = z
    zs = wide.cuda()[:, 5:5 + Cn]
    ks = torch.cat([k, k], 1).cuda()[:, Cn:]
    actc, advc, oldc, vc, mc = cuda(act, adv, old, valid.bool(), mask.bool())
    nothing = learning.policy_loss_grad(zs, actc, advc, oldc, heads, valid=vc, choice_mask=mc,
                                        denominator=torch.tensor(-1.0).cuda())
    assert nothing.loss.item() == 0.0 and nothing.count.item() == 0.0 and not nothing.grad.any().item()
    for den in (1000.0, torch.tensor(1000.0).cuda()):
        want = ref.policy_loss(z, act, adv, old, heads, k, valid, mask, clip=(0.1, 0.3), kl_coef=0.1, entropy_coef=0.0,
                               denominator=1000.0, scale=4096.0)
        kw = dict(ref_logits=ks, valid=vc, choice_mask=mc, clip=(0.1, 0.3), kl_coef=0.1, denominator=den)
        got = learning.policy_loss_grad(zs, actc, advc, oldc, heads, grad_scale=4096.0, **kw)
        check_loss(got, want, dtype)
        leaf = zs.detach().requires_grad_()
        got = learning.policy_loss(leaf, actc, advc, oldc, heads, **kw)
        grad, = torch.autograd.grad(got.loss * 4096.0, leaf)
        check_loss(got, want, dtype, grad)


@gpu
def test_policy_loss_many_rows():
    """Many workgroups, with the valid rows counted on the device; the rows'
    own values against a short run, the means against sums in 64 bits."""
    for name, N in (('team', 300007), ('w200', 20001)):
        heads = LAYOUTS[name]
        g = gen(8)
        z = torch.randn(N, heads.n_choices, generator=g)
        act = torch.stack([torch.randint(n, (N,), generator=g).int() + lo for n, lo in zip(heads.sizes, heads.low)], 1)
        adv, valid = torch.randn(N, generator=g), (torch.rand(N, generator=g) < 0.5).to(torch.uint8)
        logp = sum(torch.log_softmax(z[:, s].double(), 1).gather(1, (act[:, d:d + 1] - heads.low[d]).long())[:, 0]
                   for d, s in enumerate(ref.head_slices(heads)))
        old = (logp - 0.1).float()                               # every ratio exp(0.1): not clipped
        args = cuda(z, act.contiguous(), adv, old)
        got = learning.policy_loss_grad(*args, heads, valid=valid.cuda(), entropy_coef=0.0)
        m = float(valid.sum())
        want = float((-torch.exp(logp - old.double()) * adv.double())[valid.bool()].sum()) / m
        assert got.count.item() == m
        assert abs(got.loss.item() - want) <= 64 * ref.U * float(adv.abs().double().mean())
        for r in (0, 1, N // 2, N - 2, N - 1):
            part = ref.policy_loss(z[r:r + 1], act[r:r + 1], adv[r:r + 1], old[r:r + 1], heads, valid=valid[r:r + 1],
                                   denominator=m)
            assert ref.near(got.grad[r:r + 1], part['grad'], part['e_grad']) <= 1
        again = learning.policy_loss_grad(*args, heads, valid=valid.cuda(), entropy_coef=0.0)
        assert all(a.equal(b) for a, b in zip(got, again)), "the same inputs, other bits"


@gpu
def test_policy_loss_gradient_against_differences():
    """The kernel's own loss along a direction, by central differences."""
    heads, z, _, k, act, adv, old, _, g = loss_inputs('rtt', torch.float32, 9, False)
    args = cuda(act, adv, old)
    kw = dict(ref_logits=k.cuda(), kl_coef=0.3, entropy_coef=0.05)
    got = learning.policy_loss_grad(z.cuda(), *args, heads, **kw)
    v = torch.randn(z.shape, generator=g)
    h = 2.0 ** -9
    up, dn = (learning.policy_loss((z + s * h * v).cuda(), *args, heads, **kw).loss.item() for s in (1, -1))
    slope = float((got.grad.cpu().double() * v.double()).sum())
    up64, dn64 = (ref.policy_loss(z + s * h * v, act, adv, old, heads, k, **{a: b for a, b in kw.items() if a != 'ref_logits'})
                  for s in (1, -1))
    # the kernel's two values have e_loss each; the 64-bit difference says what h itself costs
    room = (up64['e_loss'] + dn64['e_loss']) / (2 * h) + abs((up64['loss'] - dn64['loss']) / (2 * h) - slope)
    assert abs((up - dn) / (2 * h) - slope) <= room
    assert abs((up64['loss'] - dn64['loss']) / (2 * h) - slope) < 1e-3 * float(v.norm())


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('name,N,lanes', [('team', 700, 7), ('team', 1000, 100), ('rtt', 640, 64), ('odd', 130, 130),
                                          ('w65', 90, 30), ('w513', 12, 4), ('cells', 12, 3)])
def test_lane_masks_wrap(name, N, lanes, dtype):
    """Mask rows that repeat inside and across tiles of rows."""
    heads = LAYOUTS[name]
    g = gen(N + lanes)
    z = torch.randn(N, heads.n_choices, generator=g).to(dtype)
    mask = (torch.rand(lanes, heads.n_choices, generator=g) < 0.6).to(torch.uint8)
    noise = gumbel(z.shape, g)
    act, logp, _, e, _ = ref.sample(z, heads, noise, mask.repeat(N // lanes, 1))
    got = learning.sample_actions(z.cuda(), heads, noise.cuda(), mask.cuda())
    assert got.actions.cpu().equal(act) and ref.near(got.logp, logp, e) <= 1
    old = (logp + 0.1).float()
    adv = torch.randn(N, generator=g)
    want = ref.policy_loss(z, act, adv, old, heads, z, None, mask, kl_coef=0.1, entropy_coef=0.01)
    zc, actc, advc, oldc, mc = cuda(z, act, adv, old, mask)
    got = learning.policy_loss_grad(zc, actc, advc, oldc, heads, ref_logits=zc, choice_mask=mc, kl_coef=0.1,
                                    entropy_coef=0.01)
    check_loss(got, want, dtype)


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('name', ['team', 'rtt', 'odd', 'w65', 'w513', 'w4100', 'mixed'])
def test_odd_addresses_and_strides(name, dtype):
    """Rows that begin at any element and lie any stride apart; a gradient is
    still side by side."""
    heads = LAYOUTS[name]
    g = gen(7)
    N, Cn = 5, heads.n_choices
    for shift, pad in ((1, 0), (3, 1), (0, 7)):
        flat = torch.full((shift + N * (Cn + pad),), math.nan, dtype=dtype)
        z = torch.randn(N, Cn, generator=g).to(dtype)
        view = flat[shift:].view(N, Cn + pad)[:, :Cn]
        view.copy_(z)
        zc = flat.cuda()[shift:].view(N, Cn + pad)[:, :Cn]
        noise = gumbel(z.shape, g)
        act, logp, _, e, _ = ref.sample(z, heads, noise)
        got = learning.sample_actions(zc, heads, noise.cuda())
        assert got.actions.cpu().equal(act) and ref.near(got.logp, logp, e) <= 1
        adv, old = torch.randn(N, generator=g), (logp - 0.05).float()
        want = ref.policy_loss(z, act, adv, old, heads, z, None, None, kl_coef=0.1, entropy_coef=0.01)
        got = learning.policy_loss_grad(zc, *cuda(act, adv, old), heads, ref_logits=zc, kl_coef=0.1, entropy_coef=0.01)
        check_loss(got, want, dtype)


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('sizes', [[5, 5] + [2] * 9, [2] * 30, [100]], ids=['narrow', 'heads', 'wide'])
def test_log_probabilities_lean_nowhere(sizes, dtype):
    """Errors that point one way add up over heads and rows: the mean
    error of a log-probability and of the KL is under half a rounding at 1
    (2^-25) per head.  What may lean: log2(e) and log(2), 1.4e-8 and 3e-9 of the
    logits' distance from their mean, and 3e-9 of the exponentials."""
    N, g = 65536, gen(5)
    heads = PolicyHeads(sizes)
    z = (1.5 * torch.randn(N, sum(sizes), generator=g)).to(dtype)
    r = (z + 0.2 * torch.randn(z.shape, generator=g)).to(dtype)
    acts, lp, kl, first = [], 0., 0., 0
    for n in sizes:
        p, q = (t[:, first:first + n].double().log_softmax(1) for t in (z, r))
        acts.append((p + gumbel(p.shape, g)).argmax(1))
        lp = lp + p.gather(1, acts[-1][:, None])[:, 0]
        kl = kl + (q.exp() * (q - p)).sum(1)
        first += n
    args = cuda(z, torch.stack(acts, 1).int(), torch.randn(N, generator=g), lp.float())
    got = learning.policy_loss_grad(*args, heads, ref_logits=r.cuda(), kl_coef=1.0)
    bound = len(sizes) * 2. ** -25
    assert abs((got.logp.cpu().double() - lp).mean()) <= bound
    # (the mean itself is rounded to float32)
    assert abs(got.stats[1].cpu().double() - kl.mean()) <= bound + 2. ** -24 * kl.mean()


@gpu
def test_masked_by_the_lowest_value():
    """Choices masked by their type's lowest number, as some policies do, with
    a large loss scale: probability 0, gradient 0, nothing infinite."""
    for name in ('team', 'rtt', 'w65', 'w4100', 'cells'):
        heads = LAYOUTS[name]
        for dtype in DTYPES:
            g = gen(5)
            z = torch.randn(6, heads.n_choices, generator=g)
            hide = torch.rand(z.shape, generator=g) < 0.4
            for s in ref.head_slices(heads):
                hide[:, s.start] = False
            low = torch.finfo(dtype).min
            zl = torch.where(hide, low, z.to(dtype).float()).to(dtype)
            mask = (~hide).to(torch.uint8)
            act, logp, _, _, _ = ref.sample(z.to(dtype), heads, None, mask)
            args = cuda(act, torch.randn(6, generator=g), logp.float())
            kw = dict(entropy_coef=0.1, grad_scale=2.0 ** 14, denominator=1.0)
            a = learning.policy_loss_grad(zl.cuda(), *args, heads, **kw)
            b = learning.policy_loss_grad(z.to(dtype).cuda(), *args, heads, choice_mask=mask.cuda(), **kw)
            assert torch.isfinite(a.grad.float()).all().item() and torch.isfinite(a.loss).item()
            assert not a.grad.cpu()[hide].any().item()
            size = float(b.grad.float().abs().max())
            assert (a.grad.float() - b.grad.float()).abs().max().item() <= size * (2.0 ** -18 + torch.finfo(dtype).eps)


@gpu
def test_more_than_two_to_the_31_elements():
    """Offsets past 32 bits: the last rows and channels as on their own."""
    N = (1 << 28) + 130
    z = torch.zeros(N, 8, dtype=torch.bfloat16, device='cuda')
    tail = torch.randn(130, 8, generator=gen(1)).bfloat16().cuda()
    z[-130:] = tail
    act = torch.zeros(N, 3, dtype=torch.int32, device='cuda')
    adv = torch.ones(N, device='cuda')
    old = torch.zeros(N, device='cuda')
    got = learning.policy_loss_grad(z, act, adv, old, TEAM, entropy_coef=0.1, denominator=1.0)
    own = learning.policy_loss_grad(tail, act[-130:], adv[-130:], old[-130:], TEAM, entropy_coef=0.1, denominator=1.0)
    assert got.grad[-130:].equal(own.grad) and got.logp[-130:].equal(own.logp) and got.count.item() == 1.0
    del got
    r = learning.sample_actions(z, TEAM, out=act)
    assert r.actions[-130:].equal(learning.sample_actions(tail, TEAM).actions)
    del z, r, act, adv, old
    wide = torch.zeros(170000, 12801, dtype=torch.bfloat16, device='cuda')
    heads = PolicyHeads([12801])
    wide[-3:] = torch.randn(3, 12801, generator=gen(2)).bfloat16().cuda()
    assert learning.sample_actions(wide, heads).actions[-3:].equal(learning.sample_actions(wide[-3:].clone(), heads).actions)
    del wide
    n = 1 << 29
    x = torch.zeros(5, n, dtype=torch.bfloat16, device='cuda')
    part = torch.randn(5, 200, generator=gen(3)).bfloat16().cuda()
    x[:, -200:] = part
    h, last = learning.linear_recurrence(0.5, x)
    own, own_last = learning.linear_recurrence(0.5, part)
    assert h[:, -200:].equal(own) and last[-200:].equal(own_last)


# ----------------------------------------------------------- GPU: recurrence
SHAPES = [(1, 1), (1, 7), (2, 64), (15, 3), (16, 65), (17, 130), (33, 2, 5), (100, 4, 3, 2), (257, 96), (1000, 2),
          (4099, 5), (40, 300, 17)]


def recurrence_inputs(shape, dtype, gate_kind, cut_kind, seed=0):
    g = gen(seed)
    x = torch.randn(shape, generator=g).to(dtype)
    gshape = {'full': shape, 'f32': shape, 'shared': shape[:-1] + (1,), 'steps': shape[:1], 'value': None}[gate_kind]
    if gshape is None:
        gate = 0.97
    else:
        gate = torch.sigmoid(2 + torch.randn(gshape, generator=g)) * (torch.rand(gshape, generator=g) < 0.95)
        gate = gate.to(torch.float32 if gate_kind == 'f32' else dtype)
    cshape = {'none': None, 'envs': shape[:2] if len(shape) > 2 else shape[:1], 'full': shape}[cut_kind]
    cut = None if cshape is None else (torch.rand(cshape, generator=g) < 0.1).to(torch.uint8)
    return gate, x, torch.randn(shape[1:], generator=g), cut, g


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_recurrence(shape, dtype):
    for i, (gk, ck, reverse) in enumerate([('full', 'none', False), ('shared', 'envs', True), ('value', 'full', False),
                                           ('f32', 'envs', True), ('steps', 'none', False), ('full', 'full', True)]):
        gate, x, state, cut, _ = recurrence_inputs(shape, dtype, gk, ck, i)
        state = state if i % 3 else None
        want, last = ref.recurrence(gate, x, state, cut, reverse)
        e, e_last = ref.recurrence_error(gate, x, state, cut, reverse)
        gc = gate.cuda() if isinstance(gate, torch.Tensor) else gate
        xc, sc, cc = cuda(x, state, cut)
        h, l = learning.linear_recurrence(gc, xc, sc, cut=cc, reverse=reverse)
        assert h.dtype == dtype and ref.near(h, want, e, dtype) <= 1, (gk, ck, reverse)
        assert ref.near(l, last, e_last) <= 1


def _gradients(gate, x, state, cut, reverse, dh, dlast):
    """64-bit gradients by autograd, and bounds of float32's errors."""
    leaves = [t.double().requires_grad_() for t in (gate, x, state)]
    h, last = ref.recurrence(*leaves, cut, reverse)
    want = torch.autograd.grad((h, last), leaves, (dh.double(), dlast.double()))
    # the error of g = dx is a recurrence's over |dh|; dgate's follows from both
    T = x.shape[0]
    a = ref._per_channel(gate, x, torch.float64).abs()
    if cut is not None:
        a = torch.where(ref._per_channel(cut, x, torch.bool), 0.0, a)
    order = list(range(T))[::-1] if reverse else list(range(T))
    eh, _ = ref.recurrence_error(gate, x, state, cut, reverse)
    hs = h.detach()
    eg, big = torch.zeros_like(hs), dlast.double().abs()
    err = torch.zeros_like(big)
    e_gate = torch.zeros_like(hs)
    for i in reversed(range(T)):
        t = order[i]
        big = big + dh[t].double().abs()
        err = err + 4 * ref.U * big
        eg[t] = err
        before = hs[order[i - 1]] if i else state.double()
        e_before = eh[order[i - 1]] if i else torch.zeros_like(err)
        e_gate[t] = torch.where(a[t] > 0, 1.0, 1.0) * (err * before.abs() + big * e_before + 4 * ref.U * big * before.abs())
        err, big = a[t] * err + 4 * ref.U * a[t] * big, a[t] * big
    while e_gate.dim() > gate.dim():
        e_gate = e_gate.sum(-1) * 1.0
    if e_gate.shape != gate.shape:
        e_gate = e_gate.sum(-1, keepdim=True)
    # the sum over the channels of a shared gate rounds at each of them
    n = x.numel() / gate.numel()
    full = (ref._per_channel(gate, x, torch.float64) * 0 + 1)
    size = torch.zeros_like(hs)
    for i in range(T):
        size[order[i]] = (want[1][order[i]].abs() * (hs[order[i - 1]] if i else state.double()).abs())
    size = size * full
    while size.dim() > gate.dim():
        size = size.sum(-1)
    if size.shape != gate.shape:
        size = size.sum(-1, keepdim=True)
    return want, e_gate + (n + 4) * ref.U * size, eg, err


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_recurrence_backward(shape, dtype):
    for i, (gk, ck, reverse) in enumerate([('full', 'none', False), ('shared', 'envs', True), ('f32', 'full', False),
                                           ('steps', 'envs', False), ('full', 'envs', True)]):
        gate, x, state, cut, g = recurrence_inputs(shape, dtype, gk, ck, 10 + i)
        dh, dlast = torch.randn(shape, generator=g).to(dtype), torch.randn(shape[1:], generator=g)
        (wg, wx, ws), e_gate, e_x, e_s = _gradients(gate, x, state, cut, reverse, dh, dlast)
        leaves = [t.cuda().requires_grad_() for t in (gate, x, state)]
        h, last = learning.linear_recurrence(*leaves, cut=None if cut is None else cut.cuda(), reverse=reverse)
        dg, dx, ds = torch.autograd.grad((h, last), leaves, (dh.cuda(), dlast.cuda()))
        assert ref.near(dx, wx, e_x, dtype) <= 1, (gk, ck, reverse)
        assert ref.near(ds, ws, e_s) <= 1
        assert dg.shape == gate.shape and ref.near(dg, wg, e_gate, gate.dtype) <= 1, (gk, ck, reverse)


@gpu
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('shape,gk,ck,reverse', [
    ((18, 2048, 258), 'full', 'envs', False), ((18, 2048, 258), 'shared', 'envs', True),
    ((16, 4096, 130), 'f32', 'none', True), ((3, 4096, 130), 'steps', 'none', False),
    ((5, 4096, 129), 'shared', 'envs', False), ((1, 524288, 1), 'full', 'none', False),
    ((2, 262144, 2), 'shared', 'full', False)])
def test_recurrence_many_channels(shape, gk, ck, reverse, dtype):
    """So many channels that they alone fill the device: pairs of 16-bit
    channels, and what cannot be paired (odd spans, a cut for each channel)."""
    gate, x, state, cut, g = recurrence_inputs(shape, dtype, gk, ck, 20)
    dh, dlast = torch.randn(shape, generator=g).to(dtype), torch.randn(shape[1:], generator=g)
    want, last = ref.recurrence(gate, x, state, cut, reverse)
    e, e_last = ref.recurrence_error(gate, x, state, cut, reverse)
    (wg, wx, ws), e_gate, e_x, e_s = _gradients(gate, x, state, cut, reverse, dh, dlast)
    leaves = [t.cuda().requires_grad_() for t in (gate, x, state)]
    h, l = learning.linear_recurrence(*leaves, cut=None if cut is None else cut.cuda(), reverse=reverse)
    dg, dx, ds = torch.autograd.grad((h, l), leaves, (dh.cuda(), dlast.cuda()))
    assert ref.near(h, want.detach(), e, dtype) <= 1 and ref.near(l, last.detach(), e_last) <= 1
    assert ref.near(dx, wx, e_x, dtype) <= 1 and ref.near(ds, ws, e_s) <= 1
    assert ref.near(dg, wg, e_gate, gate.dtype) <= 1
    if gk == 'full':                                             # a gate of one number, no state
        want, last = ref.recurrence(0.9, x, None, cut, reverse)
        e, _ = ref.recurrence_error(0.9, x, None, cut, reverse)
        h, _ = learning.linear_recurrence(0.9, x.cuda(), cut=None if cut is None else cut.cuda(), reverse=reverse)
        assert ref.near(h, want, e, dtype) <= 1


@gpu
def test_recurrence_partial_gradients():
    """Only h or only last has a gradient; leaves that need none; an expanded
    gradient (of a sum)."""
    gate, x, state, cut, g = recurrence_inputs((33, 2, 5), torch.float32, 'full', 'envs', 3)
    zero_h, zero_l = torch.zeros(x.shape), torch.zeros(state.shape)
    for which in ('h', 'last'):
        dh = torch.ones(x.shape) if which == 'h' else zero_h
        dl = torch.ones(state.shape) if which == 'last' else zero_l
        (wg, wx, ws), e_g, e_x, e_s = _gradients(gate, x, state, cut, False, dh, dl)
        leaves = [t.cuda().requires_grad_() for t in (gate, x, state)]
        h, last = learning.linear_recurrence(*leaves, cut=cut.cuda())
        (h if which == 'h' else last).sum().backward()
        assert ref.near(leaves[1].grad, wx, e_x) <= 1 and ref.near(leaves[2].grad, ws, e_s) <= 1
        assert ref.near(leaves[0].grad, wg, e_g) <= 1
    only = x.cuda().requires_grad_()
    h, _ = learning.linear_recurrence(gate.cuda(), only, cut=cut.cuda())
    h.sum().backward()
    (_, wx, _), _, e_x, _ = _gradients(gate, x, torch.zeros_like(state), cut, False, torch.ones(x.shape), zero_l)
    assert ref.near(only.grad, wx, e_x) <= 1


@gpu
def test_recurrence_gradient_against_differences():
    gate, x, state, cut, g = recurrence_inputs((20, 6), torch.float32, 'shared', 'envs', 5)
    leaves = [t.cuda().requires_grad_() for t in (gate, x, state)]
    h, last = learning.linear_recurrence(*leaves, cut=cut.cuda())
    w = torch.randn(h.shape, generator=g)
    grads = torch.autograd.grad((h.double() * w.cuda()).sum(), leaves)
    d = [torch.randn(t.shape, generator=g) for t in (gate, x, state)]
    step = 2.0 ** -8
    val, err = [], 0.0
    for s in (1, -1):
        moved = [t + s * step * v for t, v in zip((gate, x, state), d)]
        hk, _ = learning.linear_recurrence(*[t.cuda() for t in moved], cut=cut.cuda())
        val.append(float((hk.cpu().double() * w).sum()))
        e, _ = ref.recurrence_error(*moved, cut)
        err += float((e * w.abs()).sum())
    slope = sum(float((a.cpu().double() * v).sum()) for a, v in zip(grads, d))
    h64 = [float((ref.recurrence(*[t + s * step * v for t, v in zip((gate, x, state), d)], cut)[0] * w).sum()) for s in (1, -1)]
    assert abs((val[0] - val[1]) / (2 * step) - slope) <= err / (2 * step) + abs((h64[0] - h64[1]) / (2 * step) - slope)
    assert abs((h64[0] - h64[1]) / (2 * step) - slope) < 0.05 * (1 + abs(slope))


@gpu
def test_recurrence_cut_and_zero_gates_drop_infinities():
    x = torch.ones(6, 3)
    x[1] = math.inf
    x[3] = math.nan
    gate = torch.full((6, 3), 0.5)
    cut = torch.zeros(6, dtype=torch.uint8)
    cut[2] = 1
    gate[4] = 0.0
    h, last = learning.linear_recurrence(gate.cuda(), x.cuda(), cut=cut.cuda())
    assert h[2].tolist() == [1.0] * 3 and h[4].tolist() == [1.0] * 3 and last.tolist() == [1.5] * 3
    assert torch.isnan(h[3]).all().item() and torch.isinf(h[1]).all().item()


@gpu
def test_recurrence_no_steps_or_channels():
    state = torch.randn(4, generator=gen(1)).cuda()
    h, last = learning.linear_recurrence(0.5, torch.zeros(0, 4).cuda(), state)
    assert h.shape == (0, 4) and last.equal(state)
    h, last = learning.linear_recurrence(0.5, torch.zeros(3, 0).cuda())
    assert h.shape == (3, 0) and last.shape == (0,)
    s = state.clone().requires_grad_()
    learning.linear_recurrence(0.5, torch.zeros(0, 4).cuda(), s)[1].sum().backward()
    assert s.grad.tolist() == [1.0] * 4


# ----------------------------------------------------------- GPU: advantages
def fragment(K, E, A, seed, mode='next_step', horizon=9):
    """Slabs of a made-up rollout that keep gw_rollout's rules."""
    g = gen(seed)
    steps0 = torch.randint(0, max(1, horizon), (E,), generator=g).int()
    before = (torch.rand(E, generator=g) < 0.2).to(torch.uint8)
    all_done = torch.zeros((K, E), dtype=torch.uint8)
    n, ended = steps0.clone(), before.bool().clone()
    for t in range(K):
        reset = (ended | (n >= horizon)) if mode == 'next_step' else torch.zeros(E, dtype=torch.bool)
        end = (torch.rand(E, generator=g) < 0.1) & ~reset
        n = torch.where(reset, 0, n + 1)
        ended = end
        if mode == 'same_step':
            n = torch.where(end | (n >= horizon), 0, n)
        all_done[t] = end
    done = (torch.rand((K, E, A), generator=g) < 0.3).to(torch.uint8)
    reward = torch.randn((K, E, A), generator=g).double()
    value = torch.randn((K + 1, E, A), generator=g)
    live = (torch.rand((E, A), generator=g) < 0.8).to(torch.uint8)
    acts = (torch.rand(A, generator=g) < 0.8).to(torch.uint8)
    err = (torch.rand(E, generator=g) < 0.1).int() * 4
    return reward, value, done, all_done, before, steps0, live, acts, err


@gpu
@pytest.mark.parametrize('mode', ['next_step', 'same_step'])
@pytest.mark.parametrize('K,E,A', [(1, 1, 1), (2, 3, 5), (16, 7, 64), (17, 33, 3), (40, 5, 2), (300, 2, 3), (100, 40, 7)])
def test_advantages(K, E, A, mode):
    horizon = 9
    reward, value, done, all_done, before, steps0, live, acts, err = fragment(K, E, A, K + E, mode, horizon)
    for h, b, s, e in ((horizon, before, steps0, err), (0, None, None, None)):
        want = ref.marks(all_done, s, h, mode, b, e)
        ac, bc, sc, ec = cuda(all_done, b, s, e)
        marks = learning.fragment_marks(ac, sc, h, mode, bc, ec)
        assert marks.cpu().equal(want)
        for dtype, rdtype, a in ((torch.float32, torch.float64, acts), (torch.bfloat16, torch.float32, None),
                                 (torch.float16, torch.float64, acts)):
            v, r = value.to(dtype), reward.to(rdtype)
            adv, target, valid, e_adv = ref.advantages(r, v, done, want, live, 0.99, 0.95, a)
            # rows of steps in which nothing acted may hold anything
            r = torch.where(valid == 0, torch.tensor(math.nan, dtype=rdtype), r)
            rc, vc, dc, lc, aac = cuda(r, v, done, live, a)
            got = learning.advantages(rc, vc, dc, marks, lc, 0.99, 0.95, aac)
            assert got.valid.cpu().equal(valid)
            assert ref.near(got.advantage, adv, e_adv) <= 1
            assert ref.near(got.target, target, e_adv + 2 * ref.U * (adv.abs() + value[:-1].abs().double())) <= 1


@gpu
def test_advantages_nothing():
    k = _adv_kw(0, 2, 2)
    got = learning.advantages(**{a: b.cuda() for a, b in k.items()})
    assert got.advantage.shape == (0, 2, 2)


# --------------------------------------------- GPU: streams, graphs, devices
def _all_calls(seed):
    """Each operator's call on its own inputs, as a closure returning tensors."""
    heads, z, mask, k, act, adv, old, valid, g = loss_inputs('rtt', torch.bfloat16, seed, True)
    zc, mc, kc, actc, advc, oldc, vc = cuda(z, mask, k, act, adv, old, valid)
    noise = gumbel(z.shape, g).cuda()
    gate, x, state, cut, _ = recurrence_inputs((700, 3, 5), torch.bfloat16, 'shared', 'envs', seed)
    gc, xc, sc, cc = cuda(gate, x, state, cut)
    reward, value, done, all_done, before, steps0, live, acts, err = fragment(300, 5, 7, seed)
    rc, valc, dc, adc, lc = cuda(reward, value, done, all_done, live)

    def calls():
        s = learning.sample_actions(zc, heads, noise, mc)
        p = learning.policy_loss_grad(zc, actc, advc, oldc, heads, ref_logits=kc, valid=vc, choice_mask=mc, kl_coef=0.1)
        h, last = learning.linear_recurrence(gc, xc, sc, cut=cc)
        m = learning.fragment_marks(adc, horizon=9)
        a = learning.advantages(rc, valc, dc, m, lc)
        return list(s) + list(p) + [h, last, m] + list(a)
    return calls, (zc, xc, rc)


@gpu
def test_on_another_stream_and_two_at_once():
    a, _ = _all_calls(1)
    b, _ = _all_calls(2)
    want = [t.clone() for t in a()], [t.clone() for t in b()]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(3):
        for i, (s, f) in enumerate(((s1, a), (s2, b))):
            with torch.cuda.stream(s):
                got[i] = f()
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(x.equal(y) or (torch.isnan(x.float()) == torch.isnan(y.float())).all() for x, y in zip(w, o))


@gpu
def test_captured_and_replayed():
    """Forward calls and the one-pass gradient in a graph, replayed on new
    inputs between eager work; every replay against the eager result."""
    calls, (zc, xc, rc) = _all_calls(3)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        calls()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = calls()
    for i in range(4):
        zc.copy_(zc.roll(1, 0) if i else zc)
        xc.mul_(-1)
        rc.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        want = calls()
        torch.cuda.synchronize()
        for x, y in zip(want, out):
            assert (x == y).logical_or(torch.isnan(x.float()) & torch.isnan(y.float())).all().item()


@gpu
def test_backward_captured():
    """Autograd's backward inside a graph (torch.autograd.grad: no leaf
    accumulation), replayed against the eager gradients."""
    heads, z, mask, k, act, adv, old, valid, g = loss_inputs('team', torch.float32, 4, False)
    zc, kc, actc, advc, oldc, vc = cuda(z, k, act, adv, old, valid)
    gate, x, state, cut, _ = recurrence_inputs((50, 4, 8), torch.float32, 'shared', 'envs', 4)
    rec = cuda(gate, x, state)
    cc, = cuda(cut)

    def step():
        leaf = zc.detach().requires_grad_()
        r = learning.policy_loss(leaf, actc, advc, oldc, heads, ref_logits=kc, valid=vc, kl_coef=0.1)
        leaves = [t.detach().requires_grad_() for t in rec]
        h, last = learning.linear_recurrence(*leaves, cut=cc)
        return list(torch.autograd.grad(r.loss, leaf)) + list(torch.autograd.grad(
            (h, last), leaves, (torch.ones_like(h), torch.ones_like(last))))

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        zc.mul_(-1)
        rec[1].add_(0.25)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(step(), out):
            assert a.equal(b)


@gpu
def test_autograd_refuses_changed_inputs():
    z = torch.randn(4, 8, generator=gen(1)).cuda().requires_grad_()
    args = cuda(torch.zeros(4, 3, dtype=torch.int32), torch.ones(4), torch.zeros(4))
    r = learning.policy_loss(z, *args, TEAM)
    args[1].add_(1)
    with pytest.raises(RuntimeError, match='inplace'):
        r.loss.backward()


def test_kernels_call_nothing():
    """Every helper is inlined (a called function would need a stack of its
    own) and no kernel spills more than a few scalars."""
    pytest.importorskip('msgpack')
    from tests.test_kernel_resources import kernel_metadata
    _native.build_learn()
    md = kernel_metadata(_native.LIB_LEARN)
    assert len(md) > 50
    bad = {k: v['.private_segment_fixed_size'] for k, v in md.items()
           if v['.private_segment_fixed_size'] > 64 or v.get('.uses_dynamic_stack')}
    assert not bad, bad
