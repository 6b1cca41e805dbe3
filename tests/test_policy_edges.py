"""The policy operators at the ends of their ranges: infinite log-probabilities of a reference, and the longest sums that one thread adds up."""
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


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(16, 16384, 1, 8), (8, 40000, 1, 9), (64, 4096, 2, 8)])
def test_the_longest_sums_of_a_thread(shape, dtype):
    """Up to 64 turns of 8 values, and one more where the mask's length is no multiple of 8: 520 terms in 32 bits, 520 x 2^-24 of their sum at the worst, and 1.4e-6 of each term by the
    hardware's 2^x within 20 of the maximum; everything after that is 64 bits wide."""
    n, maps, h, w = shape
    LONG = 520 * 2.0 ** -24 + 1.4e-6
    g = torch.Generator().manual_seed(n)
    z = (2 * torch.randn(shape, generator=g)).to(dtype).cuda()
    mask = torch.rand((n, h, w), generator=g) < 0.9
    mask[:, 0, 0] = True
    mask = mask.cuda()
    action = (torch.randint(0, maps, (n,), generator=g) * h * w).cuda()
    ok = mask[:, None].expand(shape).reshape(n, -1)
    x = torch.where(ok, z.reshape(n, -1).double(), -math.inf)
    lp = torch.log_softmax(x, 1)
    p, inside = lp.exp(), torch.where(ok, lp, 0.0)
    h64 = -(p * inside).sum(1)
    logp, entropy = policy.action_log_probs(z, action, mask)
    want = lp.gather(1, action[:, None])[:, 0]
    assert ((logp.double() - want).abs() <= LONG + want.abs() * 2.0 ** -24).all()
    assert ((entropy.double() - h64).abs() <= LONG * (1 + h64) + h64 * 2.0 ** -24).all()
    drawn, drawn_logp = policy.sample_actions(z, 3, torch.arange(n).cuda(), 0, mask)
    want = lp.gather(1, drawn[:, None])[:, 0]
    assert ok.gather(1, drawn[:, None]).all() and ((drawn_logp.double() - want).abs() <= LONG + want.abs() * 2.0 ** -24).all()
    old, adv = logp - 0.1, torch.ones(n).cuda()
    ref = (z.float() + 0.5 * torch.randn(shape, generator=g).cuda()).to(dtype)
    y = torch.where(ok, ref.reshape(n, -1).double(), -math.inf)
    apart = torch.where(ok, lp - torch.log_softmax(y, 1), 0.0)
    kl = (p * apart).sum(1)
    scale = 4096.0
    terms, grad = policy.clipped_policy_grad(z, action, old, adv, mask, ref, kl_coef=0.5, entropy_coef=0.01, grad_scale=scale)
    # |z - q| stays below 4; a KL is a sum of terms of that size
    assert ((terms.kl.double() - kl).abs() <= 4 * LONG + kl * 2.0 ** -24).all()
    ratio = torch.exp(lp.gather(1, action[:, None])[:, 0] - old.double())
    take = torch.where(ratio <= 1.2, -ratio, 0.0)
    one = torch.zeros_like(p).scatter_(1, action[:, None], take[:, None])
    parts = [(-take)[:, None].expand_as(p), 0.5 * (apart - kl[:, None]), 0.01 * (inside + h64[:, None])]
    exact = (p * sum(parts) + one) * scale / n
    made_of = (p * (sum(t.abs() for t in parts) + 0.5 * 4 + 0.01 * 20) + one.abs()) * scale / n
    half = torch.finfo(dtype).eps / 2
    # a probability is 2 LONG off, the sum it is multiplied with one more, and the rounding to the type is half a step, or half of the smallest
    tol = 5 * LONG * made_of + exact.abs() * half * (1 + 1e-3) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((grad.reshape(n, -1).double() - exact).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,ends", [(8, [0, 5, 8]), (9, [0, 2, 9]), (12, [0, 1, 4, 6, 7, 9, 12]), (12, [0, 3, 6, 9, 12]), (12, [0, 12, 12])])
def test_preferences_of_long_rows_on_both_sides_of_the_rule_for_few(rows, ends):
    """Rows of more than 64 records, in pairs that the gradient ends by itself and in longer ones: the bits of the form that takes the gradient later, which always ends them first."""
    g = torch.Generator().manual_seed(rows)
    z = (2 * torch.randn(rows, 6, 200, 200, generator=g)).cuda()
    mask = (torch.rand(rows, 200, 200, generator=g) < 0.5).cuda()
    mask[:, 0, 0] = True
    action = torch.zeros(rows, dtype=torch.long).cuda()
    rl, off = policy.action_log_probs(z, action, mask)[0] + 0.5 * torch.randn(rows, generator=g).cuda(), torch.tensor(ends).cuda()
    got, grad = policy.preference_grad(z, action, rl, off, mask, beta=0.4, label_smoothing=0.1)
    leaf = z.clone().requires_grad_()
    terms = policy.preference_loss(leaf, action, rl, off, mask, beta=0.4, label_smoothing=0.1)
    terms.loss.backward()
    assert torch.equal(terms.loss.detach(), got.loss) and torch.equal(terms.margin, got.margin) and torch.equal(leaf.grad, grad)
