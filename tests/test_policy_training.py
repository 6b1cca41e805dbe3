"""Training the grasp policy over rounds (agent.PolicyLearner, BatchedGraspAgent(objective="policy")): what rounds without a signal do, what one scene learns, empty batches, resuming."""
import pytest
import torch

from mujoco_rl_ur5_amd import qnet
from mujoco_rl_ur5_amd.agent import BatchedGraspAgent, PolicyLearner
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


# ------------------------------------------------------------------ the learner alone
def _learner(**kw):
    torch.manual_seed(1)
    return PolicyLearner(qnet.MULTIDISCRETE_POLICY_RESNET(3).cuda(), "cuda", **kw)


@pytest.mark.gpu
def test_batches_in_which_no_row_counts_leave_the_weights():
    learner = _learner(batch_size=2)
    state, action, zero = torch.rand(4, 4, 24, 20, device="cuda"), torch.full((4,), -1, device="cuda"), torch.zeros(4, device="cuda")
    before = torch.cat([p.detach().flatten() for p in learner.policy_net.parameters()])
    for _ in range(15):
        learner.update(state, action, zero, zero + 1)
    after = torch.cat([p.detach().flatten() for p in learner.policy_net.parameters()])
    assert float((after - before).norm() / before.norm()) < 1e-5
