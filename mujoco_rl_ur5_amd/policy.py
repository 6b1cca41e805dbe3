"""Operators of a grasp POLICY over the agent's action set: sampling, log-probabilities, a clipped policy loss and a preference loss, as HIP kernels
(include/ur5learn.h, csrc/ur5_policy.h).

The reference learns a Q map per wrist rotation (Grasping_Agent_multidiscrete.py:388-446); its ``POLICY_RESNET`` (Modules.py:304-305; here ``qnet.POLICY_RESNET`` and
``qnet.MULTIDISCRETE_POLICY_RESNET``) ends in LOGITS over the same actions. An action is the flat index rotation * H * W + pixel of ``[R, H, W]`` maps -- 240 000 of them for
200 x 200 observations and 6 rotations -- and the pixels that lie on the table are a mask that all rotations share.

Common arguments. ``logits``: float32 / float16 / bfloat16, ``[N, R, H, W]``, ``[N, H, W]`` or ``[N, A]``, on the GPU; rows may be strided, a row that is not contiguous is copied.
``mask``: bool or uint8 ``[N, H, W]``, ``[N, M]`` or with N = 1 for one mask shared by all rows; M divides A and action j is allowed where ``mask[j % M]`` is. Logits of actions that
are not allowed may hold anything. -inf is a logit of probability 0; NaN or +inf in an allowed place make the row's results NaN. A row COUNTS if its action is in [0, A) and
allowed with a logit above -inf; rows that do not count (action -1: padding, a scene that sees no table) add nothing to a loss and get a zero gradient.

Everything is queued on the current stream of the logits' device and can be captured into a graph; there is no host synchronisation and no CPU fallback.
"""
from __future__ import annotations

import ctypes as C
from collections import namedtuple

import torch

from . import native, sharding

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
SAMPLE_STREAM = 6                     # random stream of the sampled actions (sharding.scene_uniform); the agent's exploration, depth noise and jitter hold 1, 4 and 5

PolicyLoss = namedtuple("PolicyLoss", "loss logp kl entropy")
PreferenceLoss = namedtuple("PreferenceLoss", "loss margin")


def _flat(t, what):
    """[N, ...] as [N, A] with neighbouring elements, without a copy where the rows allow it."""
    n = t.shape[0]
    width = 1
    for d in t.shape[1:]:
        width *= d
    if width == 0:
        raise ValueError(f"{what} has no actions: {tuple(t.shape)}")
    if t.is_contiguous():
        return t.view(n, width)
    t = t.reshape(n, width)
    return t if t.stride(1) == 1 and (n <= 1 or t.stride(0) >= width) or width == 1 and (n <= 1 or t.stride(0) >= 1) else t.contiguous()


def _gpu(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{what} is on {t.device}: the policy operators run on the GPU, there is no CPU fallback")


def _vector(t, n, dtype, device, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    if t.shape != (n,) or t.device != device:
        raise ValueError(f"{what} must be a [{n}] tensor on {device}, not {tuple(t.shape)} on {t.device}")
    if t.dtype.is_floating_point != dtype.is_floating_point or t.dtype == torch.bool:
        raise TypeError(f"{what} must hold {dtype}, not {t.dtype}")
    return t.detach().to(dtype).contiguous()


def _logits(logits, what="logits"):
    _gpu(logits, what)
    if logits.dtype not in DTYPES:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, not {logits.dtype}")
    if logits.dim() < 2:
        raise ValueError(f"{what} must be [N, ...], not {tuple(logits.shape)}")
    return _flat(logits.detach(), what)


def _mask(mask, z):
    if mask is None:
        return None
    _gpu(mask, "mask")
    if mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"mask must be bool or uint8, not {mask.dtype}")
    if mask.device != z.device or mask.dim() < 2 or mask.shape[0] not in (1, z.shape[0]):
        raise ValueError(f"mask must be [{z.shape[0]} or 1, ...] on {z.device}, not {tuple(mask.shape)} on {mask.device}")
    m = _flat(mask, "mask")
    if z.shape[1] % m.shape[1]:
        raise ValueError(f"a mask of {m.shape[1]} pixels does not divide {z.shape[1]} actions")
    return m


def _reference(ref, z, shape):
    if ref is None:
        return None
    q = _logits(ref, "ref_logits")
    if ref.shape != shape or q.dtype != z.dtype or q.device != z.device:
        raise ValueError(f"ref_logits must be {tuple(shape)} {z.dtype} on {z.device} like the logits, not {tuple(ref.shape)} {q.dtype} on {q.device}")
    return q


def _work(lib, z, mask, pairs=0):
    return torch.empty(lib.ur5_policy_work_bytes(z.shape[0], z.shape[1], mask.shape[1] if mask is not None else 0, pairs), dtype=torch.uint8, device=z.device)


def _rows(z, mask, ref, work):
    """The C view of checked tensors (kept alive by the caller)."""
    n, a = z.shape
    return native.Rows(z.data_ptr(), ref.data_ptr() if ref is not None else None, mask.data_ptr() if mask is not None else None,
                       z.stride(0), ref.stride(0) if ref is not None else 0, mask.stride(0) if mask is not None and mask.shape[0] > 1 else 0,
                       n, a, mask.shape[1] if mask is not None else 0, DTYPES[z.dtype], z.device.index, torch.cuda.current_stream(z.device).cuda_stream,
                       work.data_ptr(), work.numel())


def sample_actions(logits, seed, gids, round_index, mask=None, stream=SAMPLE_STREAM):
    """One draw per row from the softmax over its allowed actions: (action int64 [N], log-probability float32 [N]). The randomness is
    ``sharding.scene_uniform(seed, gids, round_index, stream, A, dtype=float64)``, evaluated where it is needed: a pure function of the GLOBAL scene ids ``gids`` (int64 [N]), so a
    scene draws the same action however the scenes are sharded or chunked. A row that allows nothing gives (-1, 0)."""
    z = _logits(logits)
    m, g = _mask(mask, z), _vector(gids, z.shape[0], torch.int64, z.device, "gids")
    lib = native.load()
    action = torch.empty(z.shape[0], dtype=torch.int64, device=z.device)
    logp = torch.empty(z.shape[0], dtype=torch.float32, device=z.device)
    r = _rows(z, m, None, _w := _work(lib, z, m))
    native.check(lib, lib.ur5_policy_sample(C.byref(r), sharding.scene_key_offset(seed, round_index, stream), g.data_ptr(), action.data_ptr(), logp.data_ptr()), "ur5_policy_sample")
    return action, logp


def action_log_probs(logits, action, mask=None):
    """(log-probability of ``action`` (int64 [N]), entropy of the row), float32 [N] each, without a gradient: what a loss needs of the behaviour and reference policies.
    An action outside [0, A) has log-probability 0, one that is not allowed -inf; a row that allows nothing has entropy 0."""
    z = _logits(logits)
    m, a = _mask(mask, z), _vector(action, z.shape[0], torch.int64, z.device, "action")
    lib = native.load()
    out = torch.empty((2, z.shape[0]), dtype=torch.float32, device=z.device)
    logp, entropy = out[0], out[1]
    r = _rows(z, m, None, _w := _work(lib, z, m))
    native.check(lib, lib.ur5_policy_logp(C.byref(r), a.data_ptr(), logp.data_ptr(), entropy.data_ptr()), "ur5_policy_logp")
    return logp, entropy


# ------------------------------------------------------------------ clipped policy loss
def _clip_inputs(logits, action, old_logp, advantage, mask, ref_logits, clip, kl_coef, entropy_coef):
    z = _logits(logits)
    n = z.shape[0]
    low, high = (float(clip[0]), float(clip[1])) if isinstance(clip, (tuple, list)) else (float(clip), float(clip))
    if kl_coef and ref_logits is None:
        raise ValueError("kl_coef needs ref_logits")
    tensors = (z, _vector(action, n, torch.int64, z.device, "action"), _vector(old_logp, n, torch.float32, z.device, "old_logp"),
               _vector(advantage, n, torch.float32, z.device, "advantage"), _mask(mask, z), _reference(ref_logits, z, logits.shape))
    return tensors, (low, high, float(kl_coef), float(entropy_coef))


def _clip_struct(tensors, numbers, scale=1.0, upstream=None):
    _, action, old, adv, _, _ = tensors
    return native.Clip(action.data_ptr(), old.data_ptr(), adv.data_ptr(), *numbers, scale, upstream)


def _clip_outputs(z):
    out = torch.empty((3, z.shape[0]), dtype=torch.float32, device=z.device)
    return torch.empty((), dtype=torch.float32, device=z.device), out[0], out[1], out[2]


class _ClippedPolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tensors, numbers):
        z, _, _, _, mask, ref = tensors
        lib = native.load()
        work = _work(lib, z, mask)
        terms = _clip_outputs(z)
        r, c = _rows(z, mask, ref, work), _clip_struct(tensors, numbers)
        native.check(lib, lib.ur5_policy_clip_loss(C.byref(r), C.byref(c), *(t.data_ptr() for t in terms)), "ur5_policy_clip_loss")
        ctx.save_for_backward(*tensors, work)                  # (the logits as [N, A]: checkpoint8.saved_activations keeps two-dimensional tensors as they are)
        ctx.numbers, ctx.shape = numbers, logits.shape
        ctx.mark_non_differentiable(*terms[1:])
        return terms

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream, *_):
        *tensors, work = ctx.saved_tensors
        z, _, _, _, mask, ref = tensors
        lib = native.load()
        grad = torch.empty(z.shape, dtype=z.dtype, device=z.device)
        upstream = upstream.float().contiguous()
        r, c = _rows(z, mask, ref, work), _clip_struct(tensors, ctx.numbers, 1.0, upstream.data_ptr())
        native.check(lib, lib.ur5_policy_clip_grad(C.byref(r), C.byref(c), grad.data_ptr()), "ur5_policy_clip_grad")
        return grad.view(ctx.shape), None, None


def clipped_policy_loss(logits, action, old_logp, advantage, mask=None, ref_logits=None, clip=0.2, kl_coef=0.0, entropy_coef=0.0):
    """``PolicyLoss(loss, logp, kl, entropy)``; ``loss`` (float32 scalar) is differentiable with respect to ``logits``: the mean over the rows that count of

        -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef KL(row || ref row) - entropy_coef H(row),      r = exp(logp - old_logp)

    action int64 [N] (-1: the row does not count), old_logp / advantage A float [N] (constants); ``ref_logits`` like the logits: the KL is exact, over all allowed actions (+inf where
    the reference gives probability 0 to an action of positive probability). ``clip``: one number or (low, high). logp, kl, entropy: float32 [N], no gradient, 0 in rows that do not
    count (kl is 0 without ref_logits)."""
    tensors, numbers = _clip_inputs(logits, action, old_logp, advantage, mask, ref_logits, clip, kl_coef, entropy_coef)
    return PolicyLoss(*_ClippedPolicyLoss.apply(logits, tensors, numbers))


def clipped_policy_grad(logits, action, old_logp, advantage, mask=None, ref_logits=None, clip=0.2, kl_coef=0.0, entropy_coef=0.0, grad_scale=1.0):
    """(``PolicyLoss``, its gradient times ``grad_scale`` with respect to the logits, in their shape and type) in three launches, without an autograd graph: for
    ``logits.backward(grad)``. float16 logits want a ``grad_scale``: the entries are about p / N."""
    tensors, numbers = _clip_inputs(logits, action, old_logp, advantage, mask, ref_logits, clip, kl_coef, entropy_coef)
    z = tensors[0]
    lib = native.load()
    terms = _clip_outputs(z)
    grad = torch.empty(logits.shape, dtype=z.dtype, device=z.device)
    r, c = _rows(z, tensors[4], tensors[5], _w := _work(lib, z, tensors[4])), _clip_struct(tensors, numbers, float(grad_scale))
    native.check(lib, lib.ur5_policy_clip_loss_grad(C.byref(r), C.byref(c), *(t.data_ptr() for t in terms), grad.data_ptr()), "ur5_policy_clip_loss_grad")
    return PolicyLoss(*terms), grad


# ------------------------------------------------------------------ preference loss
def _prefer_inputs(logits, action, ref_logp, offsets, mask, beta, label_smoothing):
    z = _logits(logits)
    n = z.shape[0]
    if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 3 or offsets.shape[0] % 2 == 0:
        raise ValueError("offsets must be [2 pairs + 1] row numbers of the episodes' ends, with at least one pair")
    tensors = (z, _vector(action, n, torch.int64, z.device, "action"), _vector(ref_logp, n, torch.float32, z.device, "ref_logp"),
               _vector(offsets, offsets.shape[0], torch.int64, z.device, "offsets"), _mask(mask, z))
    return tensors, (float(beta), float(label_smoothing))


def _prefer_struct(tensors, numbers, scale=1.0, upstream=None):
    _, action, ref_logp, offsets, _ = tensors
    return native.Prefer(action.data_ptr(), ref_logp.data_ptr(), offsets.data_ptr(), offsets.shape[0] // 2, *numbers, scale, upstream)


def _prefer_forward(lib, tensors, numbers, work):
    z, _, _, offsets, mask = tensors
    loss = torch.empty((), dtype=torch.float32, device=z.device)
    margin = torch.empty(offsets.shape[0] // 2, dtype=torch.float32, device=z.device)
    r, p = _rows(z, mask, None, work), _prefer_struct(tensors, numbers)
    native.check(lib, lib.ur5_policy_prefer_loss(C.byref(r), C.byref(p), loss.data_ptr(), margin.data_ptr()), "ur5_policy_prefer_loss")
    return loss, margin


def _prefer_backward(lib, tensors, numbers, work, scale, upstream):
    z, _, _, _, mask = tensors
    grad = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    r, p = _rows(z, mask, None, work), _prefer_struct(tensors, numbers, scale, upstream)
    native.check(lib, lib.ur5_policy_prefer_grad(C.byref(r), C.byref(p), grad.data_ptr()), "ur5_policy_prefer_grad")
    return grad


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tensors, numbers):
        lib = native.load()
        work = _work(lib, tensors[0], tensors[4], tensors[3].shape[0] // 2)
        loss, margin = _prefer_forward(lib, tensors, numbers, work)
        ctx.save_for_backward(*tensors, work)
        ctx.numbers, ctx.shape = numbers, logits.shape
        ctx.mark_non_differentiable(margin)
        return loss, margin

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream, _):
        *tensors, work = ctx.saved_tensors
        upstream = upstream.float().contiguous()
        return _prefer_backward(native.load(), tensors, ctx.numbers, work, 1.0, upstream.data_ptr()).view(ctx.shape), None, None


def preference_loss(logits, action, ref_logp, offsets, mask=None, beta=0.1, label_smoothing=0.0):
    """``PreferenceLoss(loss, margin)`` over pairs of episodes; ``loss`` (float32 scalar) is differentiable with respect to ``logits``. Row t is one step: its logits, the action
    taken (int64; -1: the row does not count) and the reference policy's log-probability of it. Episode k holds the rows offsets[k] .. offsets[k + 1] - 1 (``offsets``: ascending int64
    [2 P + 1] on the device; an episode may be empty) and episode 2 i is preferred to 2 i + 1:

        margin_i = beta (sum over episode 2 i of (logp - ref_logp) - the same over episode 2 i + 1),    loss = mean_i (1 - eps) softplus(-margin_i) + eps softplus(margin_i)

    with eps = ``label_smoothing``. Rows of no episode get a zero gradient."""
    tensors, numbers = _prefer_inputs(logits, action, ref_logp, offsets, mask, beta, label_smoothing)
    return PreferenceLoss(*_PreferenceLoss.apply(logits, tensors, numbers))


def preference_grad(logits, action, ref_logp, offsets, mask=None, beta=0.1, label_smoothing=0.0, grad_scale=1.0):
    """(``PreferenceLoss``, its gradient times ``grad_scale`` with respect to the logits) without an autograd graph: for ``logits.backward(grad)``."""
    tensors, numbers = _prefer_inputs(logits, action, ref_logp, offsets, mask, beta, label_smoothing)
    z, pairs = tensors[0], offsets.shape[0] // 2
    lib = native.load()
    loss = torch.empty((), dtype=torch.float32, device=z.device)
    margin = torch.empty(pairs, dtype=torch.float32, device=z.device)
    grad = torch.empty(logits.shape, dtype=z.dtype, device=z.device)
    r, p = _rows(z, tensors[4], None, _w := _work(lib, z, tensors[4], pairs)), _prefer_struct(tensors, numbers, float(grad_scale))
    native.check(lib, lib.ur5_policy_prefer_loss_grad(C.byref(r), C.byref(p), loss.data_ptr(), margin.data_ptr(), grad.data_ptr()), "ur5_policy_prefer_loss_grad")
    return PreferenceLoss(loss, margin), grad
