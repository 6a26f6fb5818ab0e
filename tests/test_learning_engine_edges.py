"""The policy operators' methods on engines and batched envs at their edges."""
import pytest

from tests import learning_reference as ref
from tests.cases import build_rtt, build_sim, load_golden
from tests.test_learning_engine import _engine, _gumbel, _small_team

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('encoding', ['array', 'ravel'])
@pytest.mark.parametrize('name', ['tb_small', 'rtt_7'])
def test_drawn_actions_can_be_collected(name, encoding):
    """What BatchedMultiAgentEnv.sample returned stays as it was after the next draws and steps."""
    import torch
    from abmarl_amd.external import BatchedMultiAgentEnv
    case = load_golden(name)['case']
    env = BatchedMultiAgentEnv(build_sim(case) if name.startswith('tb') else build_rtt(case), 16, horizon=9,
                               auto_reset='next_step', action_encoding=encoding)
    env.reset()
    heads, mask = env.policy_heads()
    g = torch.Generator(device='cuda').manual_seed(3)
    kept, copies = [], []
    for t in range(5):
        z = torch.randn((16, env.engine.A, heads.n_choices), generator=g, device='cuda')
        r = env.sample(z, _gumbel(z.shape, g))
        kept.append(r)
        copies.append([v.clone() for v in r])
        env.step(r.actions)
        env.engine.err.zero_()
    for r, c in zip(kept, copies):
        assert all(a.equal(b) for a, b in zip(r, c))
    assert not torch.stack([r.actions for r in kept]).eq(kept[-1].actions).all().item()


@pytest.mark.parametrize('mode', ['next_step', 'same_step'])
def test_memory_over_fragments(mode):
    """engine.linear_recurrence over two fragments in a row, against a memory in 64 bits that starts
    anew whenever the engine's own step counter of an env is 0."""
    import torch
    E, horizon, D = 40, 7, 5
    eng = _engine(_small_team(), E, run=3)
    step = eng.step_autoreset_next if mode == 'next_step' else eng.step_autoreset
    g = torch.Generator(device='cuda').manual_seed(4)
    state = torch.zeros((E, eng.A, D), device='cuda')
    begun = 0
    for fragment, K in enumerate((19, 6)):
        eng.err.zero_()
        start = eng.fragment_start()
        out = eng.rollout_buffers(K + 2)                         # slabs may hold more steps than the fragment
        first = []
        for t in range(K + 1):
            first.append(eng.fragment_start()['steps'] == 0)
            if t < K:
                out['all_done'][t] = step(eng.random_actions(9, 100 * fragment + t), horizon=horizon)[3]
        first = torch.stack(first)
        x = torch.randn((K + 1, E, eng.A, D), generator=g, device='cuda')
        gate = torch.rand((K + 1, E, eng.A, 1), generator=g, device='cuda')
        h, _ = eng.linear_recurrence(gate, x, out, start, state, horizon=horizon, autoreset=mode)
        part, last = eng.linear_recurrence(gate[:K], x[:K], out, start, state, horizon=horizon, autoreset=mode)
        cut = first.cpu().to(torch.uint8)
        want, _ = ref.recurrence(gate.cpu(), x.cpu(), state.cpu(), cut)
        err, _ = ref.recurrence_error(gate.cpu(), x.cpu(), state.cpu(), cut)
        used = torch.ones((K + 1, E), dtype=torch.bool)
        if mode == 'next_step':                                  # behind an episode's end, before the reset: not used
            used[1:] = (out['all_done'][:K] == 0).cpu() | cut[1:].bool()
        assert used.any(1).all().item() and cut.any().item()
        begun += int(cut[1:].sum())
        assert ref.near(h[used.cuda()], want[used], err[used]) <= 1, fragment
        assert ref.near(part[used[:K].cuda()], want[:K][used[:K]], err[:K][used[:K]]) <= 1
        # (the last state is joined of the steps' maps, not walked: the same bound)
        assert ref.near(last[used[K - 1].cuda()], want[K - 1][used[K - 1]], err[K - 1][used[K - 1]]) <= 1
        state = last
    assert begun > E


def test_memory_of_turn_based_slabs_refused():
    import torch
    from abmarl_amd.examples.pacman import build_pacman
    eng = _engine(build_pacman().compiled(), 2)
    with pytest.raises(ValueError, match='turn'):
        eng.linear_recurrence(0.5, torch.zeros((3, 2, eng.A), device='cuda'), dict(returned=None), {})
