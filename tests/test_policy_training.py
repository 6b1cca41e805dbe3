"""Training the grasp policy over rounds (agent.PolicyLearner, BatchedGraspAgent(objective="policy")): what rounds without a signal do, what one scene learns, empty batches, resuming."""
import collections
import types

import pytest
import torch

from mujoco_rl_ur5_amd import qnet
from mujoco_rl_ur5_amd.agent import BASELINE_GRASPS, BatchedGraspAgent, PolicyLearner
from mujoco_rl_ur5_amd.envs import GraspEnv


def _agent(model, n, rewards, seed=20, learning_rate=0.001, **options):
    """An agent of n scenes whose grasps are answered with the given rewards, a list per round: its learning alone."""
    env = GraspEnv(file=model, n_envs=n, show_obs=False, observation="render", check_mode=1, image_width=24, image_height=24)
    env.reset()
    agent = BatchedGraspAgent(env=env, device="cuda", objective="policy", seed=seed, learning_rate=learning_rate, **options)
    left = iter(rewards)
    env.step_device = lambda action, depth, device=None, sync=True: (torch.tensor(next(left), dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.bool, device="cuda"))
    return agent


def _weights(agent):
    return torch.cat([p.detach().flatten() for p in agent.policy_net.parameters()])


@pytest.mark.gpu
@pytest.mark.parametrize("reward", [0, 1])
@pytest.mark.parametrize("n", [1, 3])
def test_rounds_of_one_reward_leave_the_weights(model_it1, n, reward):
    """Rewards that are all the same say nothing: weights may shrink by the decay, 30 x 0.001 x 0.00002 of themselves, no more. (The first round of rewards above the start's baseline of
    nothing is a signal; it is not counted.)"""
    agent = _agent(model_it1, n, [[reward] * n] * 40)
    for _ in range(10 if reward else 0):
        agent.round(learn=False)
    before = _weights(agent)
    for _ in range(30):
        agent.round()
    after = _weights(agent)
    assert float((after - before).norm() / before.norm()) < 1e-5


@pytest.mark.gpu
def test_one_scene_learns_from_a_lone_reward(model_it1):
    agent = _agent(model_it1, 1, [[0], [0], [1]], learning_rate=1e-5)
    seen = {}
    update = agent.learner.update
    agent.learner.update = lambda state, action, logp, advantage, mask: seen.update(state=state, action=action, logp=logp, advantage=advantage, mask=mask) or update(state, action, logp, advantage, mask)
    for _ in range(3):
        agent.round()
    assert float(seen["advantage"]) > 0.5
    assert float(agent.learner.log_probs(seen["state"], seen["action"], seen["mask"])) > float(seen["logp"])


@pytest.mark.gpu
def test_advantages_compare_with_the_other_scenes_and_earlier_rounds(model_it1):
    """Every scene against the mean of the round's other rewards and of what earlier rounds brought, weighted by how many these are: its own reward does not enter, so the gradient has the
    expected direction whatever the baseline is."""
    rewards = [[1, 0, 0, 1], [0, 0, 1, 0], [1, 1, 1, 0]]
    agent = _agent(model_it1, 4, rewards)
    seen = []
    agent.learner.update = lambda state, action, logp, advantage, mask: seen.append(advantage.tolist()) or []
    for _ in rewards:
        agent.round()
    before = []
    for round_rewards, got in zip(rewards, seen):
        for i, r in enumerate(round_rewards):
            others = before + round_rewards[:i] + round_rewards[i + 1:]
            assert abs(got[i] - (r - sum(others) / len(others))) < 1e-6
        before = before + round_rewards


def test_a_baseline_forgets_old_rounds():
    """Whole rounds are dropped once the later ones hold as many grasps as wanted; the last one always counts."""
    agent = types.SimpleNamespace(_rewards=collections.deque())
    advantage = lambda *r: BatchedGraspAgent._advantage(agent, torch.tensor(r, dtype=torch.int32)).tolist()  # noqa: E731
    assert advantage(1) == [1.0] and advantage(1) == [0.0] and advantage(0) == [-1.0]
    many = [1] * BASELINE_GRASPS
    assert advantage(*many)[0] == pytest.approx(1 - (2 + BASELINE_GRASPS - 1) / (3 + BASELINE_GRASPS - 1)) and len(agent._rewards) == 1
    assert advantage(0) == [-1.0] and len(agent._rewards) == 2
    for _ in range(BASELINE_GRASPS - 2):
        advantage(0)
    assert advantage(0)[0] < 0 and advantage(0) == [0.0] and len(agent._rewards) == BASELINE_GRASPS


# ------------------------------------------------------------------ the learner alone
def _learner(**kw):
    torch.manual_seed(1)
    return PolicyLearner(qnet.MULTIDISCRETE_POLICY_RESNET(3).cuda(), "cuda", **kw)


@pytest.mark.gpu
def test_empty_batches():
    learner = _learner()
    state, none = torch.empty(0, 4, 24, 20, device="cuda"), torch.empty(0, dtype=torch.long, device="cuda")
    for mask in (None, torch.empty(0, 24, 20, dtype=torch.bool, device="cuda")):
        action, logp = learner.act(state, 9, none, 0, mask)
        assert action.shape == logp.shape == (0,) and action.dtype == torch.int64 and logp.dtype == torch.float32 and action.is_cuda
        logp = learner.log_probs(state, none, mask)
        assert logp.shape == (0,) and logp.dtype == torch.float32 and logp.is_cuda


@pytest.mark.gpu
def test_batches_in_which_no_row_counts_leave_the_weights():
    learner = _learner(batch_size=2)
    state, action, zero = torch.rand(4, 4, 24, 20, device="cuda"), torch.full((4,), -1, device="cuda"), torch.zeros(4, device="cuda")
    before = torch.cat([p.detach().flatten() for p in learner.policy_net.parameters()])
    for _ in range(15):
        learner.update(state, action, zero, zero + 1)
    after = torch.cat([p.detach().flatten() for p in learner.policy_net.parameters()])
    assert float((after - before).norm() / before.norm()) < 1e-5


# ------------------------------------------------------------------ saving and resuming
@pytest.mark.gpu
def test_a_resumed_run_is_held_to_the_policy_it_started_from(model_it1, tmp_path):
    path = str(tmp_path / "policy.pt")
    options = dict(policy_options=dict(kl_coef=0.1, batch_size=2))
    agent = _agent(model_it1, 2, [[1, 0], [0, 0], [0, 1]], **options)
    start = {k: v.clone() for k, v in agent.learner.reference.state_dict().items()}
    for _ in range(3):
        agent.round()
    agent.save(path)
    resumed = _agent(model_it1, 2, [[0, 0], [0, 1]], seed=21, load_path=path, **options)
    kept = resumed.learner.reference.state_dict()
    assert all(torch.equal(v, kept[k]) for k, v in start.items())
    assert any(not torch.equal(v, kept[k]) for k, v in resumed.policy_net.state_dict().items())
    assert not any(p.requires_grad for p in resumed.learner.reference.parameters()) and resumed.optimizer.param_groups[0]["decoupled_weight_decay"]
    # and the same advantages follow
    seen = []
    for a in (agent, resumed):
        a.env.step_device = lambda action, depth, device=None, sync=True: (torch.tensor([0, 1], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.bool, device="cuda"))
        a.learner.update = lambda state, action, logp, advantage, mask: seen.append(advantage.clone()) or []
        a.round()
    assert torch.equal(seen[0], seen[1])
    # a file without them (of a Q run, or of a run without an anchor): the reference is the network that is loaded
    plain = torch.load(path, map_location="cuda")
    for key in [k for k in plain if k.startswith("policy")]:
        del plain[key]
    torch.save(plain, path)
    other = _agent(model_it1, 2, [[0, 0]], load_path=path, **options)
    assert all(torch.equal(v, other.learner.reference.state_dict()[k]) for k, v in other.policy_net.state_dict().items())
