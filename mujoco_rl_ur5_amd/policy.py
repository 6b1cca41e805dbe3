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

import struct
from collections import namedtuple

import torch

from . import native, sharding

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
SAMPLE_STREAM = 6                     # random stream of the sampled actions (sharding.scene_uniform); the agent's exploration, depth noise and jitter hold 1, 4 and 5

PolicyLoss = namedtuple("PolicyLoss", "loss logp kl entropy")
PreferenceLoss = namedtuple("PreferenceLoss", "loss margin")

# A call on a small batch takes as long as its Python: argument structs are packed bytes (native.Rows, Clip and Prefer spell them out), tensors that need no copy are not
# touched, and the current stream is asked for by its handle.
_ROWS, _CLIP, _PREFER = struct.Struct("@PPPqqqqqqiiPPq"), struct.Struct("@PPPfffffP"), struct.Struct("@PPPqddfP")
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_handle = None


def _library():
    global _handle
    if _handle is None:
        _handle = native.load()
    return _handle


def _check(rc, what):
    if rc:
        native.check(_library(), rc, what)


def _gpu(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    if not t.is_cuda:
        raise ValueError(f"{what} is on {t.device}: the policy operators run on the GPU, there is no CPU fallback")


class _Flat:
    """Rows of a tensor [N, ...]: n rows of `width` neighbouring elements, `stride` apart. `tensor` keeps the memory (a copy where the rows are not contiguous)."""
    __slots__ = ("tensor", "n", "width", "stride")

    def __init__(self, t, what):
        self.n = n = t.shape[0]
        if n:
            self.width = width = t.numel() // n
        else:
            self.width = width = 1
            for d in t.shape[1:]:
                width *= d
            self.width = width
        if width == 0:
            raise ValueError(f"{what} has no actions: {tuple(t.shape)}")
        self.stride = width
        if not t.is_contiguous():
            t = t.reshape(n, width)
            if (width > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < width):
                t = t.contiguous()
            self.stride = t.stride(0) if n > 1 else width
        self.tensor = t

    def matrix(self):
        """The rows as a two-dimensional tensor without a history."""
        t = self.tensor.detach()
        return t if t.dim() == 2 else t.view(self.n, self.width)


def _vector(t, n, dtype, index, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    if t.dim() != 1 or t.shape[0] != n or not t.is_cuda or t.get_device() != index:
        raise ValueError(f"{what} must be a [{n}] tensor on cuda:{index}, not {tuple(t.shape)} on {t.device}")
    if t.dtype is dtype and t.is_contiguous():
        return t
    if t.dtype.is_floating_point != dtype.is_floating_point or t.dtype == torch.bool:
        raise TypeError(f"{what} must hold {dtype}, not {t.dtype}")
    return t.detach().to(dtype).contiguous()


def _logits(logits, what="logits"):
    _gpu(logits, what)
    if logits.dtype not in DTYPES:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, not {logits.dtype}")
    if logits.dim() < 2:
        raise ValueError(f"{what} must be [N, ...], not {tuple(logits.shape)}")
    return _Flat(logits, what)


def _mask(mask, z):
    if mask is None:
        return None
    _gpu(mask, "mask")
    if mask.dtype is not torch.bool and mask.dtype is not torch.uint8:
        raise TypeError(f"mask must be bool or uint8, not {mask.dtype}")
    if mask.get_device() != z.tensor.get_device() or mask.dim() < 2 or mask.shape[0] not in (1, z.n):
        raise ValueError(f"mask must be [{z.n} or 1, ...] on {z.tensor.device}, not {tuple(mask.shape)} on {mask.device}")
    m = _Flat(mask, "mask")
    if z.width % m.width:
        raise ValueError(f"a mask of {m.width} pixels does not divide {z.width} actions")
    return m


def _reference(ref, z, shape):
    if ref is None:
        return None
    q = _logits(ref, "ref_logits")
    if ref.shape != shape or ref.dtype != z.tensor.dtype or ref.get_device() != z.tensor.get_device():
        raise ValueError(f"ref_logits must be {tuple(shape)} {z.tensor.dtype} on {z.tensor.device} like the logits, not {tuple(ref.shape)} {ref.dtype} on {ref.device}")
    return q


def _work(z, mask, pairs=0):
    """The workspace, None where none is needed. pairs = -1: of sampling and log-probabilities."""
    size = _library().ur5_policy_work_bytes(z.n, z.width, 0 if mask is None else mask.width, pairs)
    return torch.empty(size, dtype=torch.uint8, device=z.tensor.device) if size else None


def _rows(z, mask, ref, work):
    """ur5_rows of checked tensors (kept alive by the caller)."""
    t = z.tensor
    index = t.get_device()
    return _ROWS.pack(t.data_ptr(), 0 if ref is None else ref.tensor.data_ptr(), 0 if mask is None else mask.tensor.data_ptr(), z.stride, 0 if ref is None else ref.stride,
                      0 if mask is None or mask.n == 1 else mask.stride, z.n, z.width, 0 if mask is None else mask.width, DTYPES[t.dtype], index, _raw_stream(index),
                      0 if work is None else work.data_ptr(), 0 if work is None else work.numel())


def sample_actions(logits, seed, gids, round_index, mask=None, stream=SAMPLE_STREAM):
    """One draw per row from the softmax over its allowed actions: (action int64 [N], log-probability float32 [N]). The randomness is
    ``sharding.scene_uniform(seed, gids, round_index, stream, A, dtype=float64)``, evaluated where it is needed: a pure function of the GLOBAL scene ids ``gids`` (int64 [N]), so a
    scene draws the same action however the scenes are sharded or chunked. A row that allows nothing gives (-1, 0)."""
    z = _logits(logits)
    t = z.tensor
    m, g = _mask(mask, z), _vector(gids, z.n, torch.int64, t.get_device(), "gids")
    action = torch.empty(z.n, dtype=torch.int64, device=t.device)
    logp = torch.empty(z.n, dtype=torch.float32, device=t.device)
    work = _work(z, m, -1)
    _check(_library().ur5_policy_sample(_rows(z, m, None, work), sharding.scene_key_offset(seed, round_index, stream), g.data_ptr(), action.data_ptr(), logp.data_ptr()),
           "ur5_policy_sample")
    return action, logp


def action_log_probs(logits, action, mask=None):
    """(log-probability of ``action`` (int64 [N]), entropy of the row), float32 [N] each, without a gradient: what a loss needs of the behaviour and reference policies.
    An action outside [0, A) has log-probability 0, one that is not allowed -inf; a row that allows nothing has entropy 0."""
    z = _logits(logits)
    t = z.tensor
    m, a = _mask(mask, z), _vector(action, z.n, torch.int64, t.get_device(), "action")
    logp = torch.empty(z.n, dtype=torch.float32, device=t.device)
    entropy = torch.empty(z.n, dtype=torch.float32, device=t.device)
    work = _work(z, m, -1)
    _check(_library().ur5_policy_logp(_rows(z, m, None, work), a.data_ptr(), logp.data_ptr(), entropy.data_ptr()), "ur5_policy_logp")
    return logp, entropy


def _gradient_of(logits):
    """Room for a dense gradient (empty_like costs the host half of what a shape does)."""
    return torch.empty_like(logits) if logits.is_contiguous() else torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


# ------------------------------------------------------------------ clipped policy loss
class _Clip:
    """Checked arguments of a clipped loss."""
    __slots__ = ("z", "action", "old", "advantage", "mask", "ref", "numbers")

    def __init__(self, logits, action, old_logp, advantage, mask, ref_logits, clip, kl_coef, entropy_coef):
        self.z = z = _logits(logits)
        n, index = z.n, z.tensor.get_device()
        low, high = (float(clip[0]), float(clip[1])) if isinstance(clip, (tuple, list)) else (float(clip), float(clip))
        if kl_coef and ref_logits is None:
            raise ValueError("kl_coef needs ref_logits")
        self.action = _vector(action, n, torch.int64, index, "action")
        self.old = _vector(old_logp, n, torch.float32, index, "old_logp")
        self.advantage = _vector(advantage, n, torch.float32, index, "advantage")
        self.mask, self.ref = _mask(mask, z), _reference(ref_logits, z, logits.shape)
        self.numbers = (low, high, float(kl_coef), float(entropy_coef))

    def pack(self, scale=1.0, upstream=0):
        return _CLIP.pack(self.action.data_ptr(), self.old.data_ptr(), self.advantage.data_ptr(), *self.numbers, scale, upstream)

    def outputs(self):
        device = self.z.tensor.device
        return (torch.empty((), dtype=torch.float32, device=device),) + torch.empty((3, self.z.n), dtype=torch.float32, device=device).unbind()


def _saved(ctx, z, mask, ref, *others):
    """Keeps what a backward pass reads. Rows go in as matrices: checkpoint8.saved_activations keeps two-dimensional tensors as they are."""
    ctx.save_for_backward(z.matrix(), mask and mask.matrix(), ref and ref.matrix(), *others)


def _restored(ctx):
    """(z, mask, ref, others) as they were."""
    z, mask, ref, *others = ctx.saved_tensors
    return _Flat(z, "logits"), None if mask is None else _Flat(mask, "mask"), None if ref is None else _Flat(ref, "ref_logits"), others


class _ClippedPolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, c):
        work = _work(c.z, c.mask)
        loss, logp, kl, entropy = c.outputs()
        _check(_library().ur5_policy_clip_loss(_rows(c.z, c.mask, c.ref, work), c.pack(), loss.data_ptr(), logp.data_ptr(), kl.data_ptr(), entropy.data_ptr()), "ur5_policy_clip_loss")
        _saved(ctx, c.z, c.mask, c.ref, c.action, c.old, c.advantage, work)
        ctx.numbers, ctx.shape = c.numbers, logits.shape
        ctx.mark_non_differentiable(logp, kl, entropy)
        return loss, logp, kl, entropy

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream, *_):
        z, mask, ref, (action, old, advantage, work) = _restored(ctx)
        grad = torch.empty(ctx.shape, dtype=z.tensor.dtype, device=z.tensor.device)
        upstream = upstream.float().contiguous()
        c = _CLIP.pack(action.data_ptr(), old.data_ptr(), advantage.data_ptr(), *ctx.numbers, 1.0, upstream.data_ptr())
        _check(_library().ur5_policy_clip_grad(_rows(z, mask, ref, work), c, grad.data_ptr()), "ur5_policy_clip_grad")
        return grad, None


def clipped_policy_loss(logits, action, old_logp, advantage, mask=None, ref_logits=None, clip=0.2, kl_coef=0.0, entropy_coef=0.0):
    """``PolicyLoss(loss, logp, kl, entropy)``; ``loss`` (float32 scalar) is differentiable with respect to ``logits``: the mean over the rows that count of

        -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef KL(row || ref row) - entropy_coef H(row),      r = exp(logp - old_logp)

    action int64 [N] (-1: the row does not count), old_logp / advantage A float [N] (constants); ``ref_logits`` like the logits: the KL is exact, over all allowed actions (+inf where
    the reference gives probability 0 to an action whose own is above 0 in 32 bits; without a kl_coef it is only reported). ``clip``: one number or (low, high). logp, kl, entropy: float32 [N], no gradient, 0 in rows that do not
    count (kl is 0 without ref_logits)."""
    return PolicyLoss(*_ClippedPolicyLoss.apply(logits, _Clip(logits, action, old_logp, advantage, mask, ref_logits, clip, kl_coef, entropy_coef)))


def clipped_policy_grad(logits, action, old_logp, advantage, mask=None, ref_logits=None, clip=0.2, kl_coef=0.0, entropy_coef=0.0, grad_scale=1.0):
    """(``PolicyLoss``, its gradient times ``grad_scale`` with respect to the logits, in their shape and type) in two or three launches, without an autograd graph: for
    ``logits.backward(grad)``. float16 logits want a ``grad_scale``: the entries are about p / N."""
    c = _Clip(logits, action, old_logp, advantage, mask, ref_logits, clip, kl_coef, entropy_coef)
    loss, logp, kl, entropy = c.outputs()
    grad = _gradient_of(logits)
    work = _work(c.z, c.mask)
    _check(_library().ur5_policy_clip_loss_grad(_rows(c.z, c.mask, c.ref, work), c.pack(float(grad_scale)), loss.data_ptr(), logp.data_ptr(), kl.data_ptr(), entropy.data_ptr(),
                                                grad.data_ptr()), "ur5_policy_clip_loss_grad")
    return PolicyLoss(loss, logp, kl, entropy), grad


# ------------------------------------------------------------------ preference loss
class _Prefer:
    """Checked arguments of a preference loss."""
    __slots__ = ("z", "action", "ref_logp", "offsets", "mask", "pairs", "numbers")

    def __init__(self, logits, action, ref_logp, offsets, mask, beta, label_smoothing):
        self.z = z = _logits(logits)
        n, index = z.n, z.tensor.get_device()
        if not isinstance(offsets, torch.Tensor) or offsets.dim() != 1 or offsets.shape[0] < 3 or offsets.shape[0] % 2 == 0:
            raise ValueError("offsets must be [2 pairs + 1] row numbers of the episodes' ends, with at least one pair")
        self.action = _vector(action, n, torch.int64, index, "action")
        self.ref_logp = _vector(ref_logp, n, torch.float32, index, "ref_logp")
        self.offsets = _vector(offsets, offsets.shape[0], torch.int64, index, "offsets")
        self.mask, self.pairs, self.numbers = _mask(mask, z), offsets.shape[0] // 2, (float(beta), float(label_smoothing))

    def pack(self, scale=1.0):
        return _PREFER.pack(self.action.data_ptr(), self.ref_logp.data_ptr(), self.offsets.data_ptr(), self.pairs, *self.numbers, scale, 0)

    def outputs(self):
        device = self.z.tensor.device
        return torch.empty((), dtype=torch.float32, device=device), torch.empty(self.pairs, dtype=torch.float32, device=device)


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, p):
        work = _work(p.z, p.mask, p.pairs)
        loss, margin = p.outputs()
        _check(_library().ur5_policy_prefer_loss(_rows(p.z, p.mask, None, work), p.pack(), loss.data_ptr(), margin.data_ptr()), "ur5_policy_prefer_loss")
        _saved(ctx, p.z, p.mask, None, p.action, p.ref_logp, p.offsets, work)
        ctx.numbers, ctx.shape = p.numbers, logits.shape
        ctx.mark_non_differentiable(margin)
        return loss, margin

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, upstream, _):
        z, mask, _, (action, ref_logp, offsets, work) = _restored(ctx)
        grad = torch.empty(ctx.shape, dtype=z.tensor.dtype, device=z.tensor.device)
        upstream = upstream.float().contiguous()
        p = _PREFER.pack(action.data_ptr(), ref_logp.data_ptr(), offsets.data_ptr(), offsets.shape[0] // 2, *ctx.numbers, 1.0, upstream.data_ptr())
        _check(_library().ur5_policy_prefer_grad(_rows(z, mask, None, work), p, grad.data_ptr()), "ur5_policy_prefer_grad")
        return grad, None


def preference_loss(logits, action, ref_logp, offsets, mask=None, beta=0.1, label_smoothing=0.0):
    """``PreferenceLoss(loss, margin)`` over pairs of episodes; ``loss`` (float32 scalar) is differentiable with respect to ``logits``. Row t is one step: its logits, the action
    taken (int64; -1: the row does not count) and the reference policy's log-probability of it. Episode k holds the rows offsets[k] .. offsets[k + 1] - 1 (``offsets``: ascending int64
    [2 P + 1] on the device; an episode may be empty) and episode 2 i is preferred to 2 i + 1:

        margin_i = beta (sum over episode 2 i of (logp - ref_logp) - the same over episode 2 i + 1),    loss = mean_i (1 - eps) softplus(-margin_i) + eps softplus(margin_i)

    with eps = ``label_smoothing``. Rows of no episode get a zero gradient. A ref_logp of -inf (an action that the reference rules out) makes its pair's margin infinite; loss and
    gradient are their limits."""
    return PreferenceLoss(*_PreferenceLoss.apply(logits, _Prefer(logits, action, ref_logp, offsets, mask, beta, label_smoothing)))


def preference_grad(logits, action, ref_logp, offsets, mask=None, beta=0.1, label_smoothing=0.0, grad_scale=1.0):
    """(``PreferenceLoss``, its gradient times ``grad_scale`` with respect to the logits) without an autograd graph: for ``logits.backward(grad)``."""
    p = _Prefer(logits, action, ref_logp, offsets, mask, beta, label_smoothing)
    loss, margin = p.outputs()
    grad = _gradient_of(logits)
    work = _work(p.z, p.mask, p.pairs)
    _check(_library().ur5_policy_prefer_loss_grad(_rows(p.z, p.mask, None, work), p.pack(float(grad_scale)), loss.data_ptr(), margin.data_ptr(), grad.data_ptr()),
           "ur5_policy_prefer_loss_grad")
    return PreferenceLoss(loss, margin), grad
