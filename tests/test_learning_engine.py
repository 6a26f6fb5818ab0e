"""The policy operators on the engine's own rollouts: heads and lane masks from
the agents' parameters, a closed loop of drawn actions, whole fragments with
their marks, advantages, loss and gradient, against the 64-bit definitions and
the engine's own count of acting agents."""
import numpy as np
import pytest

from tests import learning_reference as ref
from tests.cases import RTT_CONFIG4, build_maze, build_rtt, build_sim, load_golden, team_battle

pytestmark = pytest.mark.gpu


def _engine(cc, E, run=0):
    from abmarl_amd.engine import GridWorldEngine, env_seeds
    eng = GridWorldEngine(cc, E, seeds=env_seeds(E, run=run))
    eng.reset()
    eng.all_done.zero_()
    eng.err.zero_()
    return eng


def _gumbel(shape, g):
    import torch
    return -torch.log(torch.empty(shape, device='cuda').exponential_(generator=g))


def _policy(obs, C, seed):
    """Logits from the observations by a fixed random linear map (dead lanes'
    rows are -2 throughout: any finite logits)."""
    import torch
    g = torch.Generator(device='cuda').manual_seed(seed)
    flat = obs.reshape(obs.shape[:-2] + (-1,)).float()
    w = 0.3 * torch.randn((flat.shape[-1], C), generator=g, device='cuda')
    return flat @ w


def _small_team():
    return team_battle(rows=8, cols=8, n_agents=12, n_teams=2,
                       agent=dict(move_range=1, attack_range=1, attack_strength=1, attack_accuracy=1, view_range=2))


CASES = {
    'team': (_small_team, 24, 7), 'team_headline': (team_battle, 64, 40),
    'rtt_small': (lambda: build_rtt(load_golden('rtt_7')['case']).compiled(), 32, 9),
    'rtt_256': (lambda: build_rtt({**RTT_CONFIG4}).compiled(), 8, 6),
    'maze': (lambda: build_maze(load_golden('maze_16')['case']).compiled(), 40, 11),
}


@pytest.mark.parametrize('name', list(CASES))
def test_heads_follow_the_agents(name):
    import torch
    from abmarl_amd import _abi
    cc = CASES[name][0]()
    eng = _engine(cc, 4)
    heads, mask, acts = eng.policy_heads()
    assert heads.act_dim == eng.act_dim and mask.shape == (eng.A, heads.n_choices)
    for lane, e in enumerate(eng.lane_entities):
        s = cc.specs[e]
        assert bool(acts[lane]) == bool(s.kind & _abi.GW_K_ACTING)
        can = mask[lane].cpu().split(list(heads.sizes))
        values = [[heads.low[d] + i for i in range(n) if can[d][i]] for d, n in enumerate(heads.sizes)]
        m = s.move_range if s.kind & _abi.GW_K_MOVING else 0
        assert values[0] == values[1] == list(range(-m, m + 1))
        k = s.simultaneous_attacks if s.kind & _abi.GW_K_ATTACKING else 0
        cells = 1 if eng.act_dim == 3 else (2 * s.attack_range + 1) ** 2
        for q in range(eng.act_dim - 2):
            assert values[2 + q] == (list(range(k + 1)) if q < cells else [0])
    # every draw is one of the lane's own choices, and what the random policy
    # plays is one of them too
    g = torch.Generator(device='cuda').manual_seed(1)
    first = torch.tensor([sum(heads.sizes[:d]) for d in range(heads.n_heads)], device='cuda')
    low = torch.tensor(heads.low, device='cuda')
    lanes = torch.arange(eng.A, device='cuda').view(1, -1, 1)
    for t in range(20):
        z = torch.zeros((4, eng.A, heads.n_choices), device='cuda')
        for rows in (eng.sample_actions(z, _gumbel(z.shape, g)).actions, eng.random_actions(3, t)):
            assert mask[lanes, (rows - low + first).long()].all().item()


def test_pacman_heads():
    from abmarl_amd.examples.pacman import build_pacman
    cc = build_pacman().compiled()
    eng = _engine(cc, 2)
    heads, mask, acts = eng.policy_heads()
    assert heads.sizes == (5,) and heads.slots == (0,) and heads.act_dim == eng.act_dim
    assert mask.shape == (eng.A, 5) and bool(mask[:, 0].all())
    with pytest.raises(ValueError, match='turn'):
        import torch
        eng.advantages(dict(returned=None), torch.zeros(3, 2, eng.A, device='cuda'), {})


@pytest.mark.parametrize('mode', ['next_step', 'same_step'])
@pytest.mark.parametrize('name', list(CASES))
def test_fragments_together(name, mode):
    """Draw, step, mark, advantages, loss, gradient: two fragments in a row."""
    import torch
    make, E, horizon = CASES[name]
    eng = _engine(make(), E, run=5)
    A = eng.A
    heads, mask, acts = eng.policy_heads()
    C = heads.n_choices
    g = torch.Generator(device='cuda').manual_seed(7)
    step = eng.step_autoreset_next if mode == 'next_step' else eng.step_autoreset
    obs = eng.obs
    for fragment, K in enumerate((13, 5)):
        eng.err.zero_()
        start = eng.fragment_start()
        acting0 = eng.acting.clone()
        out = eng.rollout_buffers(K)
        logits, drawn, logps = [], [], []
        for t in range(K):
            z = _policy(obs, C, 11)
            r = eng.sample_actions(z, _gumbel(z.shape, g))
            assert r.actions is eng.actions
            a = r.actions.cpu().numpy()
            for d, lo in enumerate(heads.low):
                assert (a[..., d] >= lo).all() and (a[..., d] < lo + heads.sizes[d]).all()
            logits.append(z)
            drawn.append(r.actions.clone())
            logps.append(r.logp)
            obs, rew, done, ad = step(r.actions, horizon=horizon)
            for k, v in (('reward', rew), ('done', done), ('all_done', ad), ('obs', obs)):
                out[k][t].copy_(v)
        value = torch.randn((K + 1, E, A), generator=g, device='cuda')
        adv = eng.advantages(out, value, start, 0.99, 0.95, horizon, mode)
        # the engine's own count of agents that acted
        ok = (eng.err == 0).cpu()
        assert ok.any()
        per_env = adv.valid.sum((0, 2)).cpu().long()
        assert per_env[ok].equal((eng.acting - acting0).cpu()[ok]), (name, mode, fragment)
        assert not per_env[~ok].any()
        marks = ref.marks(out['all_done'].cpu(), start['steps'].cpu(), horizon, mode, start['all_done'].cpu(), eng.err.cpu())
        want = ref.advantages(out['reward'].cpu(), value.cpu(), out['done'].cpu(), marks, start['live'].cpu(), 0.99, 0.95,
                              acts.cpu())
        assert adv.valid.cpu().equal(want[2])
        assert ref.near(adv.advantage, want[0], want[3]) <= 1
        # the same steps in one launch give the same slabs, so the same advantages: rollout() on a twin is
        # tested elsewhere; here the loss on what was collected
        z, act, old = torch.stack(logits), torch.stack(drawn), torch.stack(logps)
        r = eng.policy_loss_grad(z, act, adv.advantage, old, valid=adv.valid, ref_logits=z, kl_coef=0.1, entropy_coef=0.01)
        assert r.count.item() == float(adv.valid.sum())
        # the policy has not moved: every ratio 1, no KL, nothing clipped
        assert r.stats[3].item() == 0.0 and abs(r.stats[1].item()) < 1e-6
        assert torch.allclose(r.logp[adv.valid.bool()], old[adv.valid.bool()], rtol=0, atol=2e-5)
        mean = float(-(adv.advantage.double() * adv.valid).sum() / adv.valid.sum())
        assert abs(r.stats[0].item() - mean) <= 1e-4 * float(adv.advantage.abs().double().sum() / adv.valid.sum())
        leaf = z.clone().requires_grad_()
        auto = eng.policy_loss(leaf, act, adv.advantage, old, valid=adv.valid, ref_logits=z, kl_coef=0.1, entropy_coef=0.01)
        auto.loss.backward()
        assert torch.equal(leaf.grad, r.grad) and auto.loss.item() == r.loss.item()
        # some rows against the 64-bit definition
        flat = lambda t: t.reshape((-1,) + tuple(t.shape[3:])).cpu()  # noqa: E731
        rows = torch.randperm(K * E * A, generator=torch.Generator().manual_seed(1))[:40]
        m = mask.cpu().repeat(K * E, 1)
        part = ref.policy_loss(flat(z)[rows], flat(act)[rows], flat(adv.advantage)[rows], flat(old)[rows], heads,
                               flat(z)[rows], flat(adv.valid)[rows], m[rows], kl_coef=0.1, entropy_coef=0.01,
                               denominator=float(adv.valid.sum()))
        assert ref.near(flat(r.grad)[rows], part['grad'], part['e_grad']) <= 1


def test_rollout_slabs_give_the_same_advantages():
    """One gw_rollout launch and the same steps one by one: equal marks,
    advantages and valid rows."""
    import torch
    a, b = _engine(_small_team(), 48, run=2), _engine(_small_team(), 48, run=2)
    K, horizon = 21, 8
    acts = torch.stack([a.random_actions(5, t).clone() for t in range(K)])
    value = torch.randn((K + 1, 48, a.A), device='cuda')
    start = a.fragment_start()
    out = a.rollout(acts, horizon=horizon)
    slabs = b.rollout_buffers(K)
    for t in range(K):
        obs, rew, done, ad = b.step_autoreset_next(acts[t].contiguous(), horizon=horizon)
        slabs['reward'][t], slabs['done'][t], slabs['all_done'][t] = rew, done, ad
    x = a.advantages(out, value, start, horizon=horizon)
    y = b.advantages(slabs, value, start, horizon=horizon)
    assert all(p.equal(q) for p, q in zip(x, y))
    assert x.valid.any().item() and not x.valid.all().item()


@pytest.mark.parametrize('encoding', ['array', 'ravel'])
@pytest.mark.parametrize('name', ['tb_small', 'rtt_7'])
def test_batched_env_sample(name, encoding):
    """BatchedMultiAgentEnv.sample gives actions that its step() takes, in
    either encoding, inside every agent's space."""
    import torch
    from abmarl_amd.external import BatchedMultiAgentEnv
    case = load_golden(name)['case']
    sim = build_sim(case) if name.startswith('tb') else build_rtt(case)
    env = BatchedMultiAgentEnv(sim, 16, horizon=9, auto_reset='next_step', action_encoding=encoding)
    env.reset()
    heads, mask = env.policy_heads()
    g = torch.Generator(device='cuda').manual_seed(2)
    A = env.engine.A
    for t in range(12):
        z = torch.randn((16, A, heads.n_choices), generator=g, device='cuda')
        r = env.sample(z, _gumbel(z.shape, g))
        assert r.logp.shape == (16, A)
        if encoding == 'ravel':
            assert r.actions.shape == (16, A)
            assert mask.bool().gather(1, r.actions.long().t()).all().item()
            rows = env.decode_actions(r.actions).cpu().numpy()
        else:
            rows = r.actions.cpu().numpy()
        for lane, aid in enumerate(env.agent_ids):
            space = env.action_space.spaces.get(aid)
            if space is None:
                continue
            sub = space.spaces
            if 'move' in sub:
                assert (np.abs(rows[:, lane, :2]) <= sub['move'].high.max()).all()
        obs, rew, done, ad = env.step(r.actions)
        env.engine.err.zero_()
    assert obs.shape[0] == 16
