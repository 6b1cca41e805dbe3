"""The policy operators (mujoco_rl_ur5_amd/policy.py, include/ur5learn.h) against plain implementations in 64 bits, their refusals, and what a caller may do with them
(streams, graphs, strides, padded batches).

Tolerances, from the kernels' arithmetic. A term of a softmax's sum is 2^(d log2 e) by the hardware: the product rounds to |d| 2^-24 in the exponent and the function is good
to 2^-23; with logits within 20 of the maximum that is 1.4e-6. A thread adds at most 128 such terms in 32 bits (128 x 2^-24 = 7.7e-6 at the worst), everything after that is 64 bits
wide. So a sum is right to SUM = 1e-5 of it, and log-probabilities to SUM plus their own rounding; sums weighted by something of size w to SUM w.
"""
import ctypes as C
import math
import os
import re

import pytest
import torch

from conftest import ROOT
from mujoco_rl_ur5_amd import native, policy, sharding

SUM = 1e-5
TYPES = [torch.float32, torch.float16, torch.bfloat16]
half_step = lambda t: torch.finfo(t).eps / 2  # noqa: E731

# [N, R, H, W]: one action, a single tile's part, masks that wrap inside 8 actions, a mask length that is no multiple of 8, whole tiles, several pieces per row
SHAPES = [(1, 1, 1, 1), (3, 1, 1, 7), (4, 5, 1, 3), (2, 6, 5, 9), (3, 1, 33, 67), (5, 2, 32, 32), (2, 6, 40, 40), (67, 3, 9, 9), (1, 6, 200, 200)]


# ------------------------------------------------------------------ host side
def test_header_and_binding_agree():
    src = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ur5learn.h")).read(), flags=re.S)
    assert sorted(set(re.findall(r"\b(ur5_[a-z0-9_]+)\s*\(", src))) == sorted(native.LEARN_EXPORTS)
    if os.path.exists(native.DEFAULT_LIB):
        lib = C.CDLL(native.DEFAULT_LIB)
        for sym in native.LEARN_EXPORTS:
            assert hasattr(lib, sym), sym


def _good_rows(**kw):
    lib = native.load()
    n, a = kw.pop("rows", 4), kw.pop("actions", 90)
    d = dict(logits=4096, ref=None, mask=None, stride=a, ref_stride=0, mask_stride=0, rows=n, actions=a, mask_len=0, dtype=0, device=0, stream=None, work=4096,
             work_bytes=max(16, lib.ur5_policy_work_bytes(n, a, 0, 1)))   # (most of all)
    d.update(kw)
    return native.Rows(*[d[f] for f, _ in native.Rows._fields_])


@pytest.mark.parametrize("change", [dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(actions=0), dict(actions=1 << 31), dict(rows=1 << 26), dict(stride=89), dict(logits=None),
                                    dict(actions=90000, work=None), dict(actions=90000, work=4100), dict(actions=90000, work_bytes=16), dict(mask=4096, mask_len=0), dict(mask=4096, mask_len=7),
                                    dict(mask=4096, mask_len=45, mask_stride=-1), dict(ref=4096, ref_stride=1)])
def test_entry_points_refuse_bad_rows(change):
    """Every check runs before the device is asked for anything: no pointer below is ever used."""
    lib = native.load()
    r = _good_rows(**change)
    c, p = native.Clip(4096, 4096, 4096, 0.2, 0.2, 0.0, 0.0, 1.0, None), native.Prefer(4096, 4096, 4096, 1, 0.1, 0.0, 1.0, None)
    for rc in (lib.ur5_policy_sample(C.byref(r), 1, 4096, 4096, 4096), lib.ur5_policy_logp(C.byref(r), 4096, 4096, 4096), lib.ur5_policy_clip_loss(C.byref(r), C.byref(c), *[4096] * 4),
               lib.ur5_policy_clip_grad(C.byref(r), C.byref(c), 4096), lib.ur5_policy_clip_loss_grad(C.byref(r), C.byref(c), *[4096] * 5),
               lib.ur5_policy_prefer_loss(C.byref(r), C.byref(p), 4096, 4096), lib.ur5_policy_prefer_grad(C.byref(r), C.byref(p), 4096),
               lib.ur5_policy_prefer_loss_grad(C.byref(r), C.byref(p), 4096, 4096, 4096)):
        assert rc == -1 and b"ur5_policy_" in lib.ur5_last_error()


def test_entry_points_refuse_bad_numbers_and_missing_outputs():
    lib = native.load()
    r = _good_rows()
    clip = lambda **kw: C.byref(native.Clip(*[{**dict(action=4096, old_logp=4096, advantage=4096, clip_low=0.2, clip_high=0.2, kl_coef=0.0, entropy_coef=0.0, grad_scale=1.0, upstream=None), **kw}[f]
                                              for f, _ in native.Clip._fields_]))  # noqa: E731
    for kw in (dict(action=None), dict(old_logp=None), dict(advantage=None), dict(clip_low=-0.1), dict(clip_low=1.5), dict(clip_high=-1), dict(clip_low=math.nan), dict(kl_coef=-1),
               dict(kl_coef=0.1), dict(entropy_coef=math.nan)):
        assert lib.ur5_policy_clip_loss(C.byref(r), clip(**kw), *[4096] * 4) == -1, kw
        assert lib.ur5_policy_clip_grad(C.byref(r), clip(**kw), 4096) == -1, kw
    pref = lambda **kw: C.byref(native.Prefer(*[{**dict(action=4096, ref_logp=4096, offsets=4096, pairs=1, beta=0.1, label_smoothing=0.0, grad_scale=1.0, upstream=None), **kw}[f]
                                                for f, _ in native.Prefer._fields_]))  # noqa: E731
    for kw in (dict(action=None), dict(ref_logp=None), dict(offsets=None), dict(pairs=0), dict(beta=0.0), dict(beta=math.nan), dict(label_smoothing=0.6), dict(label_smoothing=-0.1)):
        assert lib.ur5_policy_prefer_loss(C.byref(r), pref(**kw), 4096, 4096) == -1, kw
        assert lib.ur5_policy_prefer_grad(C.byref(r), pref(**kw), 4096) == -1, kw
    assert lib.ur5_policy_clip_loss(C.byref(r), clip(), None, 4096, 4096, 4096) == -1 and lib.ur5_policy_clip_grad(C.byref(r), clip(), None) == -1
    assert lib.ur5_policy_prefer_loss(C.byref(r), pref(), 4096, None) == -1 and lib.ur5_policy_prefer_grad(C.byref(r), pref(), None) == -1
    assert lib.ur5_policy_sample(C.byref(r), 0, None, 4096, 4096) == -1 and lib.ur5_policy_logp(C.byref(r), 4096, None, None) == -1 and lib.ur5_policy_sample(None, 0, 4096, 4096, 4096) == -1
    assert all(lib.ur5_policy_work_bytes(*bad) == 0 for bad in ((-1, 5, 0, 0), (5, 0, 0, 0), (5, 6, 4, 0), (5, 6, -1, 0), (5, 6, 0, -2)))
    assert lib.ur5_policy_work_bytes(5, 6, 0, -1) == 0 < lib.ur5_policy_work_bytes(5, 60000, 0, -1) < lib.ur5_policy_work_bytes(5, 60000, 0, 0)   # short rows: sampling and log-probabilities need none


def test_sizes_past_one_launch_are_refused():
    """A launch holds less than 2^32 threads, and a row (a pair) takes a workgroup of 256 at least."""
    lib = native.load()
    assert lib.ur5_policy_work_bytes(16_000_000, 6, 0, 0) > 0
    for rows, pairs in (((1 << 24) - 1, 0), (1 << 24, 0), (1, 1 << 24)):
        assert lib.ur5_policy_work_bytes(rows, 6, 0, pairs) == 0
    big = _good_rows()
    big.rows = 1 << 24
    assert lib.ur5_policy_logp(C.byref(big), 4096, 4096, None) == -1 and b"too many" in lib.ur5_last_error()


def test_no_gpu_is_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is visible here")
    lib = native.load()
    assert lib.ur5_policy_logp(C.byref(_good_rows()), 4096, 4096, 4096) in (-3, -4) and lib.ur5_last_error()
    z, a = torch.zeros(2, 5), torch.zeros(2, dtype=torch.long)
    for call in (lambda: policy.sample_actions(z, 1, a, 0), lambda: policy.action_log_probs(z, a), lambda: policy.clipped_policy_loss(z, a, z[:, 0], z[:, 0]),
                 lambda: policy.preference_loss(z, a, z[:, 0], torch.tensor([0, 1, 2]))):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()


# ------------------------------------------------------------------ plain implementations in 64 bits
def _inputs(shape, dtype, kind, seed=0):
    """logits, mask, allowed [N, A]: kinds of masks that leave rows empty, whole, or with one action."""
    g = torch.Generator().manual_seed(seed)
    n, r, h, w = shape
    z = (2 * torch.randn(shape, generator=g)).to(dtype)
    mask = None
    if kind in ("random", "poison"):
        mask = torch.rand((n, h, w), generator=g) < 0.6
        mask[0] = False                                        # a scene that sees no table
    elif kind == "shared":
        mask = torch.rand((1, h, w), generator=g) < 0.5
        mask[0, -1, -1] = True
    elif kind == "last":
        mask = torch.zeros((n, h, w), dtype=torch.bool)
        mask[:, -1, -1] = True
    elif kind == "lowest":                                     # additive masks of the type's lowest value, and of -inf
        z = torch.where(torch.rand(shape, generator=g) < 0.3, torch.finfo(dtype).min, z)
        z = torch.where(torch.rand(shape, generator=g) < 0.2, torch.tensor(-math.inf, dtype=dtype), z)
        z[0] = torch.finfo(dtype).min
    ok = torch.ones((n, r, h, w), dtype=torch.bool) if mask is None else mask[:, None].expand(n if mask.shape[0] == n else 1, r, h, w).expand(n, r, h, w)
    if kind == "poison":                                       # places that are not allowed hold anything
        junk = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max], dtype=dtype)[torch.randint(0, 4, shape, generator=g)]
        z = torch.where(ok, z, junk)
    ok = ok.reshape(n, -1) & ~(z.reshape(n, -1) == -math.inf)
    return z.cuda(), None if mask is None else mask.cuda(), ok.cuda()


class Plain:
    """Row statistics in 64 bits."""

    def __init__(self, z, ok):
        self.z = torch.where(ok, z.reshape(z.shape[0], -1).double(), -math.inf)
        self.ok, self.some = ok, ok.any(1)
        top = self.z.amax(1, keepdim=True)
        top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
        e = torch.exp(self.z - top)
        s = e.sum(1, keepdim=True)
        self.p = e / torch.where(s > 0, s, 1.0)
        self.logp = torch.where(ok, (self.z - top) - torch.log(torch.where(s > 0, s, 1.0)), 0.0)   # (the maximum may be the type's lowest: 64 bits do not hold it plus a logarithm)
        self.entropy = -(self.p * self.logp).sum(1)
        self.reach = (self.p * self.logp.abs()).sum(1)          # what the entropy's sum is made of


def _actions(ok, seed=1):
    """Allowed actions where there are some, and rows that do not count: -1, behind the row, not allowed."""
    g = torch.Generator().manual_seed(seed)
    n = ok.shape[0]
    score = torch.rand(ok.shape, generator=g).cuda() * ok
    a = torch.where(ok.any(1), score.argmax(1), -1)
    if n >= 4:
        a[1], a[2] = -1, ok.shape[1] + 5
        barred = (~ok[3]).nonzero()
        if len(barred):
            a[3] = barred[0, 0]
    counts = (a >= 0) & (a < ok.shape[1])
    counts &= ok.gather(1, a.clamp(0, ok.shape[1] - 1)[:, None])[:, 0]
    return a, counts


def _at(x, a):
    return x.gather(1, a.clamp(0, x.shape[1] - 1)[:, None])[:, 0]


def _close(got, want, tol, what):
    got, want = got.double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=want.device) + want.abs() * half_step(torch.float32)
    # results are float32: what lies beyond its range (a sum over an episode of logits of the type's lowest value, -3.4e38 each) rounds to an infinity of its sign, and no other
    beyond = want.abs() > torch.finfo(torch.float32).max
    off = torch.where(beyond, torch.where(got == want.sign() * math.inf, 0.0, math.inf), (got - want).abs() - tol)
    assert not torch.isnan(got).any() and (off <= 0).all(), f"{what}: off by {float((got - want).abs().max()):.3g}, {float(off.max()):.3g} over what it may be"


MASKS = ["none", "random", "shared", "last", "lowest", "poison"]


# ------------------------------------------------------------------ log-probabilities and sampling
@pytest.mark.gpu
@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_log_probabilities(shape, dtype, kind):
    z, mask, ok = _inputs(shape, dtype, kind)
    a, counts = _actions(ok)
    logp, entropy = policy.action_log_probs(z, a, mask)
    P = Plain(z, ok)
    inside = (a >= 0) & (a < ok.shape[1])
    assert (logp[~inside] == 0).all() and (logp[inside & ~counts] == -math.inf).all()
    _close(logp[counts], _at(P.logp, a)[counts], SUM, "logp")
    _close(entropy, torch.where(P.some, P.entropy, 0.0), SUM * (1 + P.reach), "entropy")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_sampled_actions_are_the_noisy_argmax(shape, dtype, kind):
    z, mask, ok = _inputs(shape, dtype, kind, seed=3)
    n, count = ok.shape
    gids = torch.arange(n).cuda() * 7 + (1 << 40)
    action, logp = policy.sample_actions(z, 20, gids, 5, mask, stream=9)
    u = sharding.scene_uniform(20, gids, 5, 9, count, dtype=torch.float64).clamp(min=2.0 ** -54)
    P = Plain(z, ok)
    want = torch.where(P.some, (P.z - torch.log(-torch.log(u))).argmax(1), -1)
    assert torch.equal(action, want)
    _close(logp, torch.where(P.some, _at(P.logp, action), 0.0), SUM, "logp")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,large", [(torch.float32, 1e8), (torch.float32, -3e5), (torch.bfloat16, 1e8), (torch.float16, 6e4)])
def test_sampling_of_large_logits(dtype, large):
    """Logits whose spacing is coarser than the noise: many actions stay in the running to the end, and 64 bits decide between them."""
    z, mask, ok = _inputs((3, 2, 70, 97), dtype, "random", seed=31)
    z = (z.double() + large).to(dtype)
    gids = torch.arange(3).cuda() + 5
    action, logp = policy.sample_actions(z, 4, gids, 2, mask)
    u = sharding.scene_uniform(4, gids, 2, policy.SAMPLE_STREAM, ok.shape[1], dtype=torch.float64).clamp(min=2.0 ** -54)
    P = Plain(z, ok)
    assert torch.equal(action, torch.where(P.some, (P.z - torch.log(-torch.log(u))).argmax(1), -1))
    _close(logp, torch.where(P.some, _at(P.logp, action), 0.0), SUM, "logp")


@pytest.mark.gpu
def test_a_scene_draws_the_same_however_the_scenes_are_split():
    z, mask, ok = _inputs((9, 6, 40, 40), torch.float32, "random", seed=4)
    gids = torch.randperm(9, generator=torch.Generator().manual_seed(1)).cuda() + 100
    whole, logp = policy.sample_actions(z, 3, gids, 0, mask)
    for lo, hi in ((0, 4), (4, 9)):
        part, lp = policy.sample_actions(z[lo:hi], 3, gids[lo:hi], 0, mask[lo:hi])
        assert torch.equal(part, whole[lo:hi]) and torch.equal(lp, logp[lo:hi])
    other, _ = policy.sample_actions(z, 3, gids, 1, mask)
    assert not torch.equal(other, whole)


@pytest.mark.gpu
def test_sampled_frequencies_follow_the_softmax():
    """40 000 draws of one row of 11 actions, 2 of them barred: Pearson's statistic of 8 degrees of freedom is below 26.1 (its 0.999 quantile) for these keys."""
    row = torch.tensor([0.3, -1.0, 2.0, 0.0, 1.1, -2.0, 0.7, 0.2, -0.5, 3.0, -3.0])
    mask = torch.ones(1, 11, dtype=torch.bool)
    mask[0, 2] = mask[0, 9] = False
    n = 40000
    action, _ = policy.sample_actions(row.expand(n, 11).contiguous().cuda(), 11, torch.arange(n).cuda(), 2, mask.cuda())
    p = torch.softmax(row.double().masked_fill(~mask[0], -math.inf), 0)
    seen = torch.bincount(action.cpu(), minlength=11).double()
    assert seen[2] == seen[9] == 0
    live = mask[0]
    assert float(((seen - n * p)[live] ** 2 / (n * p[live])).sum()) < 26.1


# ------------------------------------------------------------------ clipped policy loss
NUMBERS = [dict(clip=0.2), dict(clip=(0.1, 0.3), kl_coef=0.05), dict(clip=0.2, kl_coef=0.5, entropy_coef=0.01), dict(clip=0.0, entropy_coef=-0.02)]


def _plain_clip(z, ok, a, counts, old, adv, ref, clip=0.2, kl_coef=0.0, entropy_coef=0.0):
    """Loss, terms and gradient by the formulas, and per element what the gradient's sum is made of."""
    low, high = clip if isinstance(clip, tuple) else (clip, clip)
    P = Plain(z, ok)
    n = max(1, int(counts.sum()))
    at = torch.where(counts, _at(P.logp, a), 0.0)
    ratio = torch.exp(at - old.double())
    free, held = ratio * adv, ratio.clamp(1 - low, 1 + high) * adv
    kl, apart = torch.zeros_like(at), torch.zeros_like(P.p)
    if ref is not None:
        Q = Plain(ref, ok)
        apart = torch.where(ok, P.logp - Q.logp, 0.0)
        kl = (P.p * apart).sum(1)
    row = torch.where(counts, -torch.minimum(free, held) + kl_coef * kl - entropy_coef * P.entropy, 0.0)
    take = torch.where(counts & (free <= held), -adv * ratio, 0.0)
    terms = [(-take)[:, None].expand_as(P.p), kl_coef * (apart - kl[:, None]), entropy_coef * (P.logp + P.entropy[:, None])]
    one = torch.zeros_like(P.p).scatter_(1, a.clamp(0, P.p.shape[1] - 1)[:, None], take[:, None])
    grad = torch.where(counts[:, None], P.p * sum(terms) + one, 0.0) / n
    made_of = torch.where(counts[:, None], P.p * (sum(t.abs() for t in terms) + kl_coef * 4 + abs(entropy_coef) * 20) + one.abs(), 0.0) / n
    return dict(loss=row.sum() / n, logp=at, kl=torch.where(counts, kl, 0.0), entropy=torch.where(counts, P.entropy, 0.0), grad=grad, made_of=made_of,
                slack=float((ratio * adv).abs().max()) if len(at) else 0.0, reach=P.reach)


def _clip_case(shape, dtype, kind, with_ref, seed=0):
    z, mask, ok = _inputs(shape, dtype, kind, seed)
    a, counts = _actions(ok)
    g = torch.Generator().manual_seed(seed + 9)
    P = Plain(z, ok)
    old = (_at(P.logp, a).clamp(min=-50) + 0.3 * torch.randn(shape[0], generator=g).cuda()).float()
    adv = torch.randn(shape[0], generator=g).cuda()
    ref = None
    if with_ref:
        ref = (z.float() + 0.5 * torch.randn(shape, generator=g).cuda()).to(dtype)
        if kind == "lowest":
            ref = torch.where(z.float() < -1e4, z, ref)
    return z, mask, ok, a, counts, old, adv, ref


def _check_clip(got, grad, want, dtype, numbers, scale=1.0):
    w = 4 * numbers.get("kl_coef", 0.0) + abs(numbers.get("entropy_coef", 0.0)) * 20
    # the ratio is exp of a difference that is SUM off; the entropy's and the KL's parts weigh SUM by what they are made of (|log p| below 20, |z - q| below 4)
    _close(got.loss, want["loss"], SUM * (2 * want["slack"] + w) + 1e-6, "loss")
    _close(got.logp, want["logp"], SUM, "logp")
    _close(got.kl, want["kl"], SUM * 4, "kl")
    _close(got.entropy, want["entropy"], SUM * (1 + want["reach"]), "entropy")
    assert grad.dtype == dtype
    # an element is a product of a probability (2 SUM off) with a sum (SUM off) and a factor, rounded to its type: half a step, or half of the smallest step
    tol = 5 * SUM * want["made_of"] * scale + want["grad"].abs() * scale * half_step(dtype) * (1 + 1e-3) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (grad.reshape(want["grad"].shape).double() - want["grad"] * scale).abs() - tol
    assert (off <= 0).all(), f"grad: {float(off.max()):.3g} over what it may be off"


@pytest.mark.gpu
@pytest.mark.parametrize("numbers", NUMBERS)
@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_clipped_policy_loss_and_gradient(shape, dtype, kind, numbers):
    z, mask, ok, a, counts, old, adv, ref = _clip_case(shape, dtype, kind, "kl_coef" in numbers)
    want = _plain_clip(z, ok, a, counts, old, adv, ref, **numbers)
    scale = 64.0 if dtype == torch.float16 else 1.0
    got, grad = policy.clipped_policy_grad(z, a, old, adv, mask, ref, grad_scale=scale, **numbers)
    _check_clip(got, grad, want, dtype, numbers, scale)
    assert grad.shape == z.shape and (grad.reshape(len(a), -1)[~counts] == 0).all() and (grad.reshape(len(a), -1)[~ok] == 0).all()
    # the differentiable form: same terms to the bit, and the same gradient times the upstream one
    leaf = z.clone().requires_grad_()
    terms = policy.clipped_policy_loss(leaf, a, old, adv, mask, ref, **numbers)
    for x, y in zip(terms, got):
        assert torch.equal(x.detach(), y)
    (terms.loss * scale).backward()
    assert torch.equal(leaf.grad, grad)


@pytest.mark.gpu
def test_gradients_match_differences():
    """Central differences of the 64-bit losses along random directions: their own error is below 1e-7 at this step."""
    shape, numbers = (6, 2, 5, 7), dict(clip=0.2, kl_coef=0.3, entropy_coef=0.05)
    z, mask, ok, a, counts, old, adv, ref = _clip_case(shape, torch.float32, "random", True, seed=5)
    _, grad = policy.clipped_policy_grad(z, a, old, adv, mask, ref, **numbers)
    offsets, rl = torch.tensor([0, 2, 3, 3, 5]).cuda(), old
    _, pgrad = policy.preference_grad(z, a, rl, offsets, mask, beta=0.7, label_smoothing=0.1)
    g = torch.Generator().manual_seed(2)
    for _ in range(4):
        v = torch.randn(shape, generator=g).cuda().double()
        h = 1e-4
        f = lambda x: _plain_clip(x, ok, a, counts, old, adv, ref, **numbers)["loss"]  # noqa: E731
        assert abs(float((f(z + h * v) - f(z - h * v)) / (2 * h) - (grad.double() * v).sum())) < 1e-4
        f = lambda x: _plain_prefer(x, ok, a, counts, rl, offsets, 0.7, 0.1)["loss"]  # noqa: E731
        assert abs(float((f(z + h * v) - f(z - h * v)) / (2 * h) - (pgrad.double() * v).sum())) < 1e-4


@pytest.mark.gpu
def test_nan_and_infinity_in_allowed_places_show():
    z = torch.zeros(3, 40).cuda()
    z[0, 5], z[1, 7] = math.nan, math.inf
    a, one = torch.tensor([5, 1, 2]).cuda(), torch.ones(3).cuda()
    logp, entropy = policy.action_log_probs(z, a)
    assert torch.isnan(logp[:2]).all() and torch.isnan(entropy[:2]).all() and abs(float(logp[2]) + math.log(40)) < 1e-5
    terms, grad = policy.clipped_policy_grad(z, a, -one, one)
    assert torch.isnan(terms.loss) and torch.isnan(grad[0]).any() and torch.isnan(grad[1]).any() and torch.isfinite(grad[2]).all()
    action, _ = policy.sample_actions(z, 1, torch.arange(3).cuda(), 0)
    assert ((action >= -1) & (action < 40)).all()
    ref = z.clone().nan_to_num_()
    ref[2, 3] = -math.inf                                       # the reference rules out what the policy may do
    terms, _ = policy.clipped_policy_grad(torch.zeros(3, 40).cuda(), a, -one, one, ref_logits=ref, kl_coef=0.1)
    assert float(terms.kl[2]) == math.inf


# ------------------------------------------------------------------ preference loss
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_a_reference_that_rules_actions_out(dtype):
    """Its KL is infinite where the policy may take such an action: reported, and without weight in neither the loss nor the gradient. An action whose probability is 0 in 32 bits
    adds nothing, whatever the reference says of it."""
    shape, kind = (7, 2, 6, 11), "random"
    z, mask, ok, a, counts, old, adv, ref = _clip_case(shape, dtype, kind, True, seed=21)
    numbers = dict(clip=0.2, entropy_coef=0.1)
    hard = ref.clone()
    hard[..., ::3] = -math.inf
    terms, grad = policy.clipped_policy_grad(z, a, old, adv, mask, hard, **numbers)
    assert (terms.kl[counts] == math.inf).any()
    _check_clip(terms._replace(kl=torch.zeros_like(terms.kl)), grad, _plain_clip(z, ok, a, counts, old, adv, None, **numbers), dtype, numbers)
    leaf = z.clone().requires_grad_()
    loss = policy.clipped_policy_loss(leaf, a, old, adv, mask, hard, **numbers).loss
    loss.backward()
    assert torch.equal(loss.detach(), terms.loss) and torch.equal(leaf.grad, grad)
    far = z.clone()
    far[..., ::3] = -32768                                          # (its exp is 0 in 64 bits, too)
    a = torch.where((a % 11) % 3 == 0, -1, a)
    numbers = dict(clip=0.2, kl_coef=0.3)
    want = policy.clipped_policy_grad(far, a, old, adv, mask, far, **numbers), policy.clipped_policy_grad(far, a, old, adv, mask, torch.where(far == -32768, -math.inf, far), **numbers)
    for x, y in zip((*want[0][0], want[0][1]), (*want[1][0], want[1][1])):
        assert torch.isfinite(x).all() and torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(24, 1, 9, 11), (25, 1, 9, 11), (12, 3, 200, 200), (13, 6, 200, 200), (9, 6, 200, 200)])
def test_both_sides_of_the_rule_for_few_rows(shape, dtype):
    """Few rows are ended by the gradient itself, more by a launch of their own: same definition, and the same bits as the form that takes the gradient later."""
    z, mask, ok, a, counts, old, adv, ref = _clip_case(shape, dtype, "random", True, seed=shape[0])
    numbers, scale = dict(clip=0.2, kl_coef=0.5, entropy_coef=0.01), 64.0 if dtype == torch.float16 else 1.0
    got, grad = policy.clipped_policy_grad(z, a, old, adv, mask, ref, grad_scale=scale, **numbers)
    _check_clip(got, grad, _plain_clip(z, ok, a, counts, old, adv, ref, **numbers), dtype, numbers, scale)
    leaf = z.clone().requires_grad_()
    terms = policy.clipped_policy_loss(leaf, a, old, adv, mask, ref, **numbers)
    (terms.loss * scale).backward()
    assert all(torch.equal(x.detach(), y) for x, y in zip(terms, got)) and torch.equal(leaf.grad, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(6, 3000, 1, 1), (5, 700, 1, 2), (4, 3001, 1, 9), (3, 90, 3, 11), (30, 500, 2, 8)])
def test_small_masks_of_many_maps(shape, dtype):
    """Fewer pixels than a workgroup has threads, shared by many maps: every place that is not allowed still gets its zero."""
    z, mask, ok, a, counts, old, adv, ref = _clip_case(shape, dtype, "random", True, seed=shape[1])
    numbers, scale = dict(clip=0.2, kl_coef=0.5, entropy_coef=0.01), 64.0 if dtype == torch.float16 else 1.0
    for held in (mask, mask[1:2]):                                  # (the second: one mask for all rows)
        here = ok if held is mask else (held[:, None].expand(shape) & torch.isfinite(z)).reshape(shape[0], -1)
        counts = (a >= 0) & (a < here.shape[1]) & _at(here, a)
        torch.full((shape[0] * here.shape[1],), math.nan, dtype=dtype, device="cuda")                        # what the gradient's memory held before
        got, grad = policy.clipped_policy_grad(z, a, old, adv, held, ref, grad_scale=scale, **numbers)
        _check_clip(got, grad, _plain_clip(z, here, a, counts, old, adv, ref, **numbers), dtype, numbers, scale)
        assert (grad.reshape(here.shape)[~here | ~counts[:, None]] == 0).all()


@pytest.mark.gpu
def test_many_short_rows():
    """More rows than one workgroup counts, in parts that end inside it."""
    for n, shape, kind in ((257, (2, 1, 3), "random"), (70_001, (1, 1, 5), "none"), (20_000, (2, 2, 2), "random")):
        z, mask, ok, a, counts, old, adv, ref = _clip_case((n,) + shape, torch.float32, kind, True, seed=n)
        numbers = dict(clip=0.2, kl_coef=0.5, entropy_coef=0.01)
        got, grad = policy.clipped_policy_grad(z, a, old, adv, mask, ref, **numbers)
        _check_clip(got, grad, _plain_clip(z, ok, a, counts, old, adv, ref, **numbers), torch.float32, numbers)


def _plain_prefer(z, ok, a, counts, ref_logp, offsets, beta, eps):
    P = Plain(z, ok)
    ratio = torch.where(counts, _at(P.logp, a) - ref_logp.double(), 0.0)
    ends = offsets.clamp(0, len(a)).tolist()
    sums = torch.stack([ratio[lo:hi].sum() for lo, hi in zip(ends[:-1], ends[1:])]).view(-1, 2)
    margin = beta * (sums[:, 0] - sums[:, 1])
    soft = torch.nn.functional.softplus
    loss = ((1 - eps) * soft(-margin) + eps * soft(margin)).mean()
    pull = -beta * ((1 - eps) * torch.sigmoid(-margin) - eps * torch.sigmoid(margin)) / len(margin)
    weight = torch.zeros(len(a), dtype=torch.float64, device=z.device)
    for i, w in enumerate(pull):
        weight[ends[2 * i]:ends[2 * i + 1]] = w
        weight[ends[2 * i + 1]:ends[2 * i + 2]] = -w
    weight = torch.where(counts, weight, 0.0)
    one = torch.zeros_like(P.p).scatter_(1, a.clamp(0, P.p.shape[1] - 1)[:, None], weight[:, None])
    return dict(loss=loss, margin=margin, grad=one - P.p * weight[:, None], made_of=((one != 0) + P.p) * beta / len(margin))


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [0.0, 0.1])
@pytest.mark.parametrize("kind", MASKS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,offsets", [((1, 1, 1, 1), [0, 0, 1]), ((4, 2, 5, 9), [0, 4, 4]), ((5, 6, 40, 40), [1, 2, 4, 4, 4]), ((67, 3, 9, 9), [0, 30, 65, 65, 66, 66, 66]), ((3, 1, 33, 67), [0, 1, 3]),
                                           ((70, 1, 5, 9), [3, 40, 69]), ((150, 2, 40, 40), [0, 20, 110, 110, 150]), ((4200, 1, 1, 7), list(range(0, 4201, 15)))],
                         ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else f"{len(v) // 2}pairs")
def test_preference_loss_and_gradient(shape, offsets, dtype, kind, eps):
    z, mask, ok = _inputs(shape, dtype, kind, seed=6)
    a, counts = _actions(ok)
    rl = (_at(Plain(z, ok).logp, a).clamp(min=-50) + torch.randn(shape[0], generator=torch.Generator().manual_seed(3)).cuda()).float()
    off = torch.tensor(offsets).cuda()
    want = _plain_prefer(z, ok, a, counts, rl, off, 0.4, eps)
    scale = 64.0 if dtype == torch.float16 else 1.0
    got, grad = policy.preference_grad(z, a, rl, off, mask, beta=0.4, label_smoothing=eps, grad_scale=scale)
    # every row's log-probability may be SUM off; and 64 bits hold a sum of n terms, in whatever order, to n 2^-53 of the sum of their sizes, here and in the plain form: that is below
    # 1e-12, but for actions of the type's lowest logit, 3.4e38, which cancel between episodes
    sizes = torch.where(counts, (_at(Plain(z, ok).logp, a) - rl.double()).abs(), 0.0)
    pair = ((torch.searchsorted(off, torch.arange(shape[0]).cuda(), right=True) - 1) // 2).clamp(0, len(offsets) // 2 - 1)
    per = 0.4 * (SUM * shape[0] + shape[0] * 2.0 ** -52 * torch.zeros(len(offsets) // 2, dtype=torch.float64, device="cuda").index_add_(0, pair, sizes))
    _close(got.margin, want["margin"], per, "margin")
    _close(got.loss, want["loss"], per.mean(), "loss")
    per = per[pair][:, None]
    # the weight (at most beta / pairs) follows the margin with a slope of at most beta / 4 pairs, the probability is 2 SUM off
    tol = (5 * SUM + per) * want["made_of"] * scale + want["grad"].abs() * scale * half_step(dtype) * (1 + 1e-3) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert ((grad.reshape(want["grad"].shape).double() - want["grad"] * scale).abs() <= tol).all()
    rows = torch.arange(shape[0]).cuda()
    assert (grad.reshape(shape[0], -1)[(rows < offsets[0]) | (rows >= offsets[-1]) | ~counts] == 0).all()
    leaf = z.clone().requires_grad_()
    terms = policy.preference_loss(leaf, a, rl, off, mask, beta=0.4, label_smoothing=eps)
    (terms.loss * scale).backward()
    assert torch.equal(terms.loss.detach(), got.loss) and torch.equal(terms.margin, got.margin) and torch.equal(leaf.grad, grad)


@pytest.mark.gpu
def test_preference_offsets_outside_the_rows_stay_inside():
    z = torch.randn(4, 50).cuda()
    a, rl = torch.tensor([1, 2, 3, 4]).cuda(), torch.zeros(4).cuda()
    terms, grad = policy.preference_grad(z, a, rl, torch.tensor([-3, 2, 900]).cuda())
    want, wgrad = policy.preference_grad(z, a, rl, torch.tensor([0, 2, 4]).cuda())
    assert torch.equal(terms.loss, want.loss) and torch.equal(grad, wgrad)


# ------------------------------------------------------------------ layouts, sizes, streams, graphs
def _all_calls(z, mask, a, old, adv, ref, gids, offsets):
    out = list(policy.sample_actions(z, 4, gids, 1, mask)) + list(policy.action_log_probs(z, a, mask))
    terms, grad = policy.clipped_policy_grad(z, a, old, adv, mask, ref, kl_coef=0.1, entropy_coef=0.01)
    out += list(terms) + [grad]
    terms, grad = policy.preference_grad(z, a, old, offsets, mask)
    return out + list(terms) + [grad]


def _call_inputs(shape=(5, 3, 20, 23), dtype=torch.float32, seed=8):
    z, mask, ok, a, counts, old, adv, ref = _clip_case(shape, dtype, "random", True, seed)
    return [z, mask, a, old, adv, ref, torch.arange(shape[0]).cuda(), torch.tensor([0, 2, shape[0]]).cuda()]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [5, 31])
@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_misaligned_rows_give_the_same_bits(dtype, rows):
    args = _call_inputs((rows, 3, 20, 23), dtype=dtype)
    want = _all_calls(*args)
    n, width = args[0].shape[0], args[0][0].numel()

    def inside(t, before, gap):                                  # rows `gap` elements apart in a larger buffer, starting at an odd element
        flat = t.reshape(n, -1)
        buf = torch.full((before + n * (flat.shape[1] + gap),), True if t.dtype == torch.bool else math.nan, dtype=t.dtype, device="cuda")
        view = buf[before:].as_strided((n, flat.shape[1]), (flat.shape[1] + gap, 1))
        view.copy_(flat)
        return view
    for before, gap in ((1, 0), (3, 1), (0, 5)):
        moved = list(args)
        moved[0], moved[1], moved[5] = inside(args[0], before, gap), inside(args[1], before, gap), inside(args[5], before, gap + 2)
        got = _all_calls(*moved)
        for x, y in zip(got, want):
            assert torch.equal(x.reshape(y.shape), y)
    across = list(args)                                          # rows that are not contiguous are copied
    across[0] = args[0].permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    across[1] = args[1].transpose(1, 2).contiguous().transpose(1, 2)
    for x, y in zip(_all_calls(*across), want):
        assert torch.equal(x, y)
    assert width % 8 != 0


@pytest.mark.gpu
def test_empty_batches():
    z, i, f = torch.empty(0, 2, 3, 4).cuda(), torch.empty(0, dtype=torch.long).cuda(), torch.empty(0).cuda()
    action, logp = policy.sample_actions(z, 1, i, 0)
    assert action.shape == logp.shape == (0,) and policy.action_log_probs(z, i)[0].shape == (0,)
    terms, grad = policy.clipped_policy_grad(z, i, f, f)
    assert float(terms.loss) == 0 and grad.shape == z.shape
    terms, grad = policy.preference_grad(z, i, f, torch.tensor([0, 0, 0]).cuda())
    assert abs(float(terms.loss) - math.log(2)) < 1e-6 and grad.shape == z.shape
    z = torch.randn(3, 8).cuda()                                 # nothing counts
    terms, grad = policy.clipped_policy_grad(z, torch.full((3,), -1).cuda(), torch.zeros(3).cuda(), torch.ones(3).cuda(), kl_coef=1.0, ref_logits=z)
    assert float(terms.loss) == 0 and (grad == 0).all()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Rows whose elements lie more than 2^32 bytes and 2^31 elements into the buffer: the same row at both ends gives the same results."""
    n, a = 2200, 1000003
    z = torch.empty((n, a), dtype=torch.float16, device="cuda")
    row = torch.randn(a, generator=torch.Generator().manual_seed(1)).half().cuda()
    z.copy_(row.expand(n, a))
    act = torch.full((n,), 12345).cuda()
    gids = torch.full((n,), 77).cuda()
    drawn, lp = policy.sample_actions(z, 1, gids, 0)
    assert n * a > 1 << 31 and (drawn == drawn[0]).all() and (lp == lp[0]).all()
    logp, entropy = policy.action_log_probs(z, act)
    assert (logp == logp[0]).all() and (entropy == entropy[0]).all()
    _, grad = policy.clipped_policy_grad(z, act, logp, torch.ones(n).cuda(), grad_scale=1024.0 * n)
    assert torch.equal(grad[-1], grad[0]) and torch.equal(grad[n // 2], grad[0]) and float(grad[0, 12345]) < -1000


@pytest.mark.gpu
def test_refusals_of_tensors():
    z, a, f = torch.zeros(3, 6, 4, 5).cuda(), torch.zeros(3, dtype=torch.long).cuda(), torch.zeros(3).cuda()
    off = torch.tensor([0, 1, 2]).cuda()
    bad = [lambda: policy.action_log_probs(z.double(), a), lambda: policy.action_log_probs(z[0, 0, 0], a), lambda: policy.action_log_probs(z, a[:2]),
           lambda: policy.action_log_probs(z, a.float()), lambda: policy.action_log_probs(z, a.cpu()), lambda: policy.action_log_probs(z, a, torch.ones(3, 7, dtype=torch.bool).cuda()),
           lambda: policy.action_log_probs(z, a, torch.ones(2, 4, 5, dtype=torch.bool).cuda()), lambda: policy.action_log_probs(z, a, torch.ones(3, 4, 5).cuda()),
           lambda: policy.action_log_probs(z, a, torch.ones(3, 4, 5, dtype=torch.bool)), lambda: policy.action_log_probs(z[:, :0], a), lambda: policy.action_log_probs([1], a),
           lambda: policy.sample_actions(z, 1, a[:1], 0), lambda: policy.clipped_policy_loss(z, a, f, f, kl_coef=0.1), lambda: policy.clipped_policy_loss(z, a, f, a),
           lambda: policy.clipped_policy_loss(z, a, f, f, ref_logits=z.half()), lambda: policy.clipped_policy_loss(z, a, f, f, ref_logits=z[:, :3]),
           lambda: policy.preference_loss(z, a, f, off[:2]), lambda: policy.preference_loss(z, a, f, off[:1]), lambda: policy.preference_loss(z, a, f, [0, 1, 2])]
    for k, call in enumerate(bad):
        with pytest.raises((ValueError, TypeError)):
            call()
            raise AssertionError(k)
    for call in (lambda: policy.clipped_policy_loss(z, a, f, f, clip=-1), lambda: policy.clipped_policy_loss(z, a, f, f, clip=(2.0, 0.1)), lambda: policy.preference_loss(z, a, f, off, beta=0),
                 lambda: policy.preference_loss(z, a, f, off, label_smoothing=0.7)):
        with pytest.raises(RuntimeError, match="ur5_policy_"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,others", [(12, 7), (37, 60)])
def test_side_streams_and_two_calls_at_once(rows, others):
    args, other = _call_inputs((rows, 6, 40, 40)), _call_inputs((others, 6, 40, 40), seed=15)
    want, want2 = _all_calls(*args), _all_calls(*other)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)                            # inputs of this stream are late
        late = [x.clone() for x in args]
        got = _all_calls(*late)
    with torch.cuda.stream(t):
        got2 = _all_calls(*other)
    torch.cuda.synchronize()
    for x, y in zip(got + got2, want + want2):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("first,second", [((5, 3, 20, 23), (9, 6, 40, 40)), ((300, 1, 20, 23), (40, 6, 40, 40))])
def test_captured_graphs_replay(first, second):
    """Two graphs of the same calls on other sizes, replayed in turn with new inputs and eager work in between; every replay equals the eager result."""
    sets = [(_call_inputs(first, seed=s), _call_inputs(second, seed=s + 50)) for s in (21, 22, 23)]
    held = [[x.clone() for x in part] for part in sets[0]]
    for part in held:
        _all_calls(*part)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for part in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_all_calls(*part))
        graphs.append(g)
    for parts in sets + sets[::-1]:
        for mine, new in zip(held, parts):
            for x, y in zip(mine, new):
                x.copy_(y)
        for g in graphs:
            g.replay()
        want = [_all_calls(*part) for part in parts]
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            for x, y in zip(out, w):
                assert torch.equal(x, y)


@pytest.mark.gpu
def test_backward_in_a_graph_and_twice():
    z, mask, a, old, adv, ref, gids, offsets = _call_inputs()
    leaf = z.clone().requires_grad_()
    loss = policy.clipped_policy_loss(leaf, a, old, adv, mask, ref, kl_coef=0.1).loss + policy.preference_loss(leaf, a, old, offsets, mask).loss
    first, = torch.autograd.grad(loss, leaf, retain_graph=True)
    again, = torch.autograd.grad(loss, leaf)
    assert torch.equal(first, again)
    del loss                                                     # (no eager graph of the leaf lives while the capture runs)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step = lambda: torch.autograd.grad(policy.clipped_policy_loss(leaf, a, old, adv, mask, ref, kl_coef=0.1).loss + policy.preference_loss(leaf, a, old, offsets, mask).loss, leaf)[0]  # noqa: E731
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        captured.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, first)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(40, 6, 60, 61), (8, 6, 60, 61)])
def test_results_do_not_change_from_run_to_run(shape):
    args = _call_inputs(shape)
    want = _all_calls(*args)
    for _ in range(5):
        for x, y in zip(_all_calls(*args), want):
            assert torch.equal(x, y)
