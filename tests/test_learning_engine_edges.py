"""The policy operators' methods on engines and batched envs at their edges."""
import pytest

from tests.cases import build_rtt, build_sim, load_golden
from tests.test_learning_engine import _gumbel

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
