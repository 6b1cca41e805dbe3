"""The policy operators as they are used: PolicyLearner (agent.py) on the grasp network, 8-bit checkpoints in both learners, and BatchedGraspAgent(objective="policy")."""
import numpy as np
import pytest
import torch

from mujoco_rl_ur5_amd import checkpoint8, policy, qnet
from mujoco_rl_ur5_amd.agent import BatchedGraspAgent, Learner, PolicyLearner
from mujoco_rl_ur5_amd.envs import GraspEnv


def test_refusals_on_the_host(model_it1, emul_lib):
    net = torch.nn.Conv2d(4, 6, 1)
    with pytest.raises(ValueError, match="activations"):
        Learner(net, 8, 8, "cpu", activations="int4")
    with pytest.raises(ValueError, match="activations"):
        PolicyLearner(net, "cpu", activations="int4")
    env = GraspEnv(file=model_it1, n_envs=1, show_obs=False, observation="render", image_width=8, image_height=8, _lib_path=emul_lib)
    for kw, what in ((dict(objective="v"), "objective"), (dict(objective="policy"), "GPU"), (dict(objective="policy", pipeline_groups=2), "one group")):
        with pytest.raises(ValueError, match=what):
            BatchedGraspAgent(env=env, device="cpu", **kw)
    learner = PolicyLearner(net, "cpu")
    with pytest.raises(ValueError, match="no CPU fallback"):
        learner.act(torch.zeros(2, 4, 8, 8), 1, torch.arange(2), 0)


def test_learner_on_the_host_is_unchanged_by_the_option():
    """On the host nothing is packed: the same losses and weights with and without activations="int8"."""
    out = []
    for activations in (None, "int8"):
        torch.manual_seed(3)
        learner = Learner(qnet.MULTIDISCRETE_RESNET(2), 16, 16, "cpu", mem_size=40, batch_size=4, activations=activations)
        g = torch.Generator().manual_seed(4)
        learner.memory.push(torch.rand(12, 4, 16, 16, generator=g), torch.randint(0, 512, (12,), generator=g), torch.randint(0, 2, (12,), generator=g))
        out.append(([learner.learn() for _ in range(2)], [p.detach().clone() for p in learner.policy_net.parameters()]))
    assert out[0][0] == out[1][0] and all(torch.equal(a, b) for a, b in zip(out[0][1], out[1][1]))


def _transitions(n=10, h=24, w=20):
    g = torch.Generator().manual_seed(7)
    state = torch.rand(n, 4, h, w, generator=g).cuda()
    mask = (torch.rand(n, h, w, generator=g) < 0.5).cuda()
    mask[:, 0, 0] = True
    return state, mask, torch.arange(n).cuda() + 5, torch.randn(n, generator=g).cuda()


def _learner(**kw):
    torch.manual_seed(1)
    return PolicyLearner(qnet.MULTIDISCRETE_POLICY_RESNET(3).cuda(), "cuda", **kw)


@pytest.mark.gpu
def test_sampling_scoring_and_training_fit_together():
    state, mask, gids, advantage = _transitions()
    learner = _learner(batch_size=4)
    action, logp = learner.act(state, 9, gids, 2, mask)
    again, logp2 = learner.act(state, 9, gids, 2, mask, chunk=3)                              # chunks choose the same actions
    # (a library convolution may add in another order for another batch: log-probabilities agree to its rounding, and a draw changes only where two scores are as near)
    assert (action == again).sum() >= 9 and torch.allclose(logp, logp2, atol=1e-3)
    assert mask.flatten(1).gather(1, (action % (24 * 20))[:, None]).all()
    assert torch.allclose(learner.log_probs(state, action, mask), logp, atol=1e-3)
    # one batch: the gradient that reaches the weights is that of the loss written out
    part = slice(0, 4)
    old = logp[part] + 0.05
    params = list(learner.policy_net.parameters())
    logits = learner.logits(state[part])
    terms, grad = policy.clipped_policy_grad(logits, action[part], old, advantage[part], mask[part], entropy_coef=0.01)
    got = torch.autograd.grad(logits, params, grad, retain_graph=True)
    lp = torch.log_softmax(logits.double().masked_fill(~mask[part].flatten(1).repeat(1, 3), -1e30), 1)
    ratio = torch.exp(lp.gather(1, action[part, None])[:, 0] - old.double())
    a = advantage[part].double()
    loss = (-torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a) + 0.01 * (lp.exp() * lp.clamp(min=-1e6)).sum(1)).mean()
    want = torch.autograd.grad(loss, params)
    assert abs(float(terms.loss) - float(loss)) < 1e-5
    most = max(float(w.norm()) for w in want)
    for x, y in zip(got, want):
        assert float((x - y).norm()) < 1e-4 * float(y.norm()) + 1e-5 * most


@pytest.mark.gpu
@pytest.mark.parametrize("activations", [None, "int8"])
def test_updates_run_and_move_the_policy(activations):
    state, mask, gids, advantage = _transitions()
    learner = _learner(batch_size=4, epochs=2, kl_coef=0.01, entropy_coef=0.001, activations=activations, learning_rate=1e-4)
    action, logp = learner.act(state, 9, gids, 0, mask)
    frozen = [p.clone() for p in learner.reference.parameters()]
    before = [p.detach().clone() for p in learner.policy_net.parameters()]
    losses = learner.update(state, action, logp, advantage, mask)
    assert len(losses) == learner.updates_done == 6 and np.isfinite(losses).all() and not checkpoint8.active()
    assert all(torch.equal(a, b) for a, b in zip(frozen, learner.reference.parameters()))
    assert any(not torch.equal(a, b) for a, b in zip(before, learner.policy_net.parameters()))
    assert all(p.grad is None or not p.grad.any() for p in learner.policy_net.parameters())
    loss, margin = learner.prefer(state, action, logp, torch.tensor([0, 3, 5, 9, 9]).cuda(), mask)
    assert np.isfinite(loss) and margin.shape == (2,) and learner.updates_done == 7
    assert learner.update(state[:0], action[:0], logp[:0], advantage[:0], mask[:0]) == []


@pytest.mark.gpu
def test_q_learner_with_packed_activations_on_gpu():
    """The reference's learner: the same first loss, and first-step weights that moved the same way wherever Adam's first step (the gradient's sign) is decided."""
    out = []
    for activations in (None, "int8"):
        torch.manual_seed(3)
        learner = Learner(qnet.MULTIDISCRETE_RESNET(6).cuda(), 40, 40, "cuda", mem_size=40, activations=activations)
        g = torch.Generator().manual_seed(4)
        learner.memory.push(torch.rand(24, 4, 40, 40, generator=g), torch.randint(0, 9600, (24,), generator=g), torch.randint(0, 2, (24,), generator=g))
        start = [p.detach().clone() for p in learner.policy_net.parameters()]
        loss = learner.learn()
        out.append((loss, torch.cat([(p.detach() - s).flatten() for p, s in zip(learner.policy_net.parameters(), start)])))
    assert abs(out[0][0] - out[1][0]) < 1e-5
    assert float((out[0][1].sign() == out[1][1].sign()).float().mean()) > 0.9


@pytest.mark.gpu
def test_policy_agent_rounds(model_it1):
    env = GraspEnv(file=model_it1, n_envs=6, show_obs=False, observation="render", check_mode=1, image_width=40, image_height=40)
    env.reset()
    agent = BatchedGraspAgent(env=env, device="cuda", objective="policy", activations="int8", policy_options=dict(batch_size=4, entropy_coef=0.01))
    for k in range(2):
        obs = env.observation_device("cuda")
        table = agent._on_table(obs, env)
        out = agent.round()
        assert out["reward"].shape == (6,) and set(out["reward"].tolist()) <= {0, 1} and out["outcomes"].shape == (6, 4)
        assert table.gather(1, (out["action"] % 1600)[:, None]).all() and ((out["action"] >= 0) & (out["action"] < 9600)).all()
        assert len(out["losses"]) == 2 and np.isfinite(out["losses"]).all()
    assert agent.rounds_done == 2 and agent.steps_done == 12
    with pytest.raises(RuntimeError, match="within round"):
        agent.learn()
