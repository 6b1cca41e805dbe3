"""The policy operators at the ends of their ranges: infinite log-probabilities of a reference."""
import math

import pytest
import torch

from mujoco_rl_ur5_amd import policy


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [4, 60, 200])
@pytest.mark.parametrize("eps", [0.0, 0.1])
@pytest.mark.parametrize("side", [0, 1])
def test_a_preference_over_an_action_that_the_reference_rules_out(side, eps, rows):
    """action_log_probs gives -inf for such an action. In the preferred episode the margin is +inf and its term eps inf, nothing without smoothing; in the other one it is -inf and the
    loss inf. The other pairs' margins and gradients are what they are without it, and the pair's own gradient is its limit."""
    g = torch.Generator().manual_seed(rows)
    z, a = torch.randn(rows, 50, generator=g).cuda(), torch.randint(0, 50, (rows,), generator=g).cuda()
    rl = (-4 + 0.1 * torch.randn(rows, generator=g)).cuda()
    half = rows // 4
    off = torch.tensor([0, half, 2 * half, 3 * half, rows]).cuda()
    ruled = rl.clone()
    ruled[side * half] = -math.inf
    beta = 0.3
    want, wgrad = policy.preference_grad(z, a, rl, off, beta=beta, label_smoothing=eps)
    got, grad = policy.preference_grad(z, a, ruled, off, beta=beta, label_smoothing=eps)
    assert float(got.margin[0]) == (math.inf if side == 0 else -math.inf) and torch.equal(got.margin[1], want.margin[1])
    m = want.margin[1].double()
    other = (1 - eps) * torch.nn.functional.softplus(-m) + eps * torch.nn.functional.softplus(m)
    if side == 0 and eps == 0:
        assert abs(float(got.loss) - float(other) / 2) < 1e-6
    else:
        assert float(got.loss) == math.inf
    # the pair's weight: -beta / pairs times (1 - eps) sigmoid(-margin) - eps sigmoid(margin), here 0 or 1 each
    w = -beta / 2 * (-eps if side == 0 else 1 - eps)
    weight = torch.cat((torch.full((half,), w), torch.full((half,), -w))).double().cuda()[:, None]
    one = torch.nn.functional.one_hot(a[:2 * half], 50).double()
    exact = weight * (one - torch.softmax(z[:2 * half].double(), 1))
    assert torch.isfinite(grad).all() and ((grad[:2 * half].double() - exact).abs() <= 1e-4 * exact.abs() + 1e-7 * beta).all() and torch.equal(grad[2 * half:], wgrad[2 * half:])
    leaf = z.clone().requires_grad_()
    terms = policy.preference_loss(leaf, a, ruled, off, beta=beta, label_smoothing=eps)
    terms.loss.backward()
    assert torch.equal(terms.loss.detach(), got.loss) and torch.equal(terms.margin, got.margin) and torch.equal(leaf.grad, grad)
