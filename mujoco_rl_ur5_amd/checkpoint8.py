"""Activation checkpoints in 8 bits: what a layer's backward pass needs of its input, kept as int8 codes with one float32 scale per 64 neighbouring values (1.06 bytes per value
instead of 4), as HIP kernels (include/ur5learn.h, csrc/ur5_act8.h).

``pack`` / ``PackedActivation.unpack`` are the checkpoint itself; ``PackedActivation.weight_grad`` is a pointwise convolution's weight gradient that reads the codes as they are;
``pointwise_conv`` is such a layer; ``saved_activations`` keeps the inputs of a network's layers this way between forward and backward pass (``agent.Learner(activations="int8")``). The
forward pass is unchanged; the layers' gradients see inputs that are off by at most half a step, 1/254 of the largest of their 64 neighbours.

Tensors are float32 / float16 / bfloat16 on the GPU; work is queued on the current stream of their device; there is no CPU fallback.
"""
from __future__ import annotations

import contextlib
import threading

import torch
import torch.nn.functional as F
from torch.overrides import TorchFunctionMode

from .policy import DTYPES, _check, _gpu, _library, _raw_stream

GROUP = 64
_active = threading.local()


def _float_gpu(t, what):
    _gpu(t, what)
    if t.dtype not in DTYPES:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, not {t.dtype}")


def _layout(shape):
    """(planes, values of a plane, groups of a plane) of a tensor: groups never reach over a plane's end. [N, C, ...] has N C planes, a matrix its rows, a vector is one plane. A tensor
    without values has no groups."""
    planes = shape[0] * shape[1] if len(shape) > 2 else shape[0] if len(shape) == 2 else 1
    count = shape.numel()
    size = count // planes if planes else 0
    return planes, size, -(-size // GROUP)


def _smaller(t):
    """Whether a checkpoint of ``t`` takes less memory: a plane of a few values still takes a whole group, and an expanded tensor holds less than its shape says."""
    planes, _, groups = _layout(t.shape)
    return planes * groups * (GROUP + 4) < min(t.numel() * t.element_size(), t.untyped_storage().nbytes())


class PackedActivation:
    """A checkpoint: ``codes`` int8 [planes, groups, 64], ``scales`` float32 [planes, groups], and the ``shape`` and ``dtype`` that ``unpack`` restores. Codes and, behind them, scales lie
    in one tensor of bytes, ``data``: on a small activation a call takes as long as its allocations."""
    __slots__ = ("data", "shape", "dtype", "planes", "size", "groups")

    def __init__(self, data, shape, dtype):
        self.data, self.shape, self.dtype = data, shape, dtype
        self.planes, self.size, self.groups = _layout(shape)

    @property
    def codes(self):
        return self.data[:self.planes * self.groups * GROUP].view(torch.int8).view(self.planes, self.groups, GROUP)

    @property
    def scales(self):
        return self.data[self.planes * self.groups * GROUP:].view(torch.float32).view(self.planes, self.groups)

    def _pointers(self):
        at = self.data.data_ptr()
        return at, at + self.planes * self.groups * GROUP

    def unpack(self):
        x = self.data.new_empty(self.shape, dtype=self.dtype)
        if self.planes * self.groups:
            index = x.get_device()
            _check(_library().ur5_act8_unpack(*self._pointers(), self.planes, self.size, x.data_ptr(), DTYPES[self.dtype], index, _raw_stream(index)), "ur5_act8_unpack")
        return x

    def weight_grad(self, dy, bias=True):
        """For a pointwise convolution y[n, o] = sum_c w[o, c] x[n, c] + b[o] of the packed x [N, C, ...]: (dw float32 [O, C], db float32 [O]) from dy [N, O, ...] -- sums over images
        and pixels, the same every time; an infinity in dy gives NaN. bias=False: (dw, None)."""
        _float_gpu(dy, "dy")
        shape = self.shape
        if len(shape) < 3 or shape[1] == 0 or dy.dim() != len(shape) or dy.shape[0] != shape[0] or dy.shape[2:] != shape[2:] or dy.get_device() != self.data.get_device():
            raise ValueError(f"dy must be [N, O, ...] like the packed {tuple(shape)} on {self.data.device}, not {tuple(dy.shape)} on {dy.device}")
        n, cin, cout = shape[0], shape[1], dy.shape[1]
        dw = torch.empty((cout, cin), dtype=torch.float32, device=dy.device)
        db = torch.empty(cout, dtype=torch.float32, device=dy.device) if bias else None
        if dy.numel() == 0:
            return dw.zero_(), db.zero_() if bias else None
        dy = dy.detach().contiguous()
        size, index, lib = self.size, dy.get_device(), _library()
        work = torch.empty(max(1, lib.ur5_act8_wgrad_work_bytes(n, cin, cout, size)), dtype=torch.uint8, device=dy.device)
        _check(lib.ur5_act8_wgrad(*self._pointers(), dy.data_ptr(), DTYPES[dy.dtype], n, cin, cout, size, dw.data_ptr(), db.data_ptr() if bias else None,
                                  work.data_ptr(), work.numel(), index, _raw_stream(index)), "ur5_act8_wgrad")
        return dw, db


def pack(x):
    """``PackedActivation`` of a tensor of any shape (at least one dimension): per group of 64 neighbouring values of a plane, scale = largest magnitude / 127 and code = the nearest
    integer to value / scale. A group that holds an infinity or a NaN is restored as NaN throughout, one below 1e-30 as zeros."""
    _float_gpu(x, "x")
    shape = x.shape
    if not shape:
        raise ValueError("a scalar has no activations to pack")
    planes, size, groups = _layout(shape)
    data = torch.empty(planes * groups * (GROUP + 4), dtype=torch.uint8, device=x.device)
    if planes * groups:
        src, index, at = x.contiguous(), x.get_device(), data.data_ptr()
        _check(_library().ur5_act8_pack(src.data_ptr(), DTYPES[x.dtype], planes, size, at, at + planes * groups * GROUP, index, _raw_stream(index)), "ur5_act8_pack")
    return PackedActivation(data, shape, x.dtype)


class _PointwiseConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        n, c = x.shape[:2]
        w = weight.reshape(weight.shape[0], c)
        y = torch.matmul(w, x.flatten(2).contiguous())
        if bias is not None:
            y = y + bias.view(1, -1, 1)
        ctx.packed = _smaller(x)                                                             # (else its backward pass packs it)
        ctx.save_for_backward(pack(x).data if ctx.packed else x, weight)
        ctx.shape, ctx.dtype, ctx.bias_dtype = x.shape, x.dtype, None if bias is None else bias.dtype
        return y.view(n, w.shape[0], *x.shape[2:])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        kept, weight = ctx.saved_tensors
        dx = dw = db = None
        cin, cout = ctx.shape[1], weight.shape[0]
        if ctx.needs_input_grad[0]:
            w = weight.reshape(cout, cin).t().contiguous().to(dy.dtype)                      # (under autocast the output, and so dy, has fewer bits than the input)
            dx = torch.matmul(w, dy.flatten(2).contiguous()).view(ctx.shape).to(ctx.dtype)
        if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
            kept = PackedActivation(kept, ctx.shape, ctx.dtype) if ctx.packed else pack(kept)
            dw, db = kept.weight_grad(dy, bias=ctx.bias_dtype is not None)
            dw = dw.view(weight.shape).to(weight.dtype)
            db = None if db is None else db.to(ctx.bias_dtype)
        return dx, dw, db


def pointwise_conv(x, weight, bias=None):
    """1 x 1 convolution [N, C, ...] -> [N, O, ...] (weight [O, C] or [O, C, 1, 1]) whose input is kept in 8 bits for the weight gradient. Same result and input gradient as the
    plain layer. Under autocast, which decides the product's type, input and weight may differ in theirs; gradients come in the types of what they belong to."""
    _float_gpu(x, "x")
    if x.dim() < 3 or weight.numel() != weight.shape[0] * x.shape[1] or weight.device != x.device or weight.dtype not in DTYPES or (weight.dtype != x.dtype and not torch.is_autocast_enabled("cuda")):
        raise ValueError(f"weight {tuple(weight.shape)} {weight.dtype} does not fit x {tuple(x.shape)} {x.dtype}")
    if bias is not None and (not isinstance(bias, torch.Tensor) or bias.shape != weight.shape[:1] or bias.device != x.device or bias.dtype not in DTYPES):
        raise ValueError(f"bias must be a [{weight.shape[0]}] tensor of float32, float16 or bfloat16 on {x.device}")
    return _PointwiseConv.apply(x, weight, bias)


def _format(t):
    """The memory format in which the values of ``t`` lie next to each other."""
    return torch.channels_last if t.dim() == 4 and not t.is_contiguous() and t.is_contiguous(memory_format=torch.channels_last) else torch.contiguous_format


class _Relu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        ctx.format = _format(x)
        x = x.contiguous(memory_format=ctx.format)
        y, count, index = torch.empty_like(x), x.numel(), x.get_device()
        bits = torch.empty(-(-count // 512) * 8, dtype=torch.int64, device=x.device)
        _check(_library().ur5_act8_relu(x.data_ptr(), DTYPES[x.dtype], count, y.data_ptr(), bits.data_ptr(), index, _raw_stream(index)), "ur5_act8_relu")
        ctx.save_for_backward(bits)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dy = dy.contiguous(memory_format=ctx.format)
        dx, index = torch.empty_like(dy), dy.get_device()
        _check(_library().ur5_act8_relu_grad(dy.data_ptr(), DTYPES[dy.dtype], ctx.saved_tensors[0].data_ptr(), dy.numel(), dx.data_ptr(), index, _raw_stream(index)), "ur5_act8_relu_grad")
        return dx


def relu(x):
    """ReLU that keeps which values are positive (a bit each) for its backward pass, not the values: a checkpoint rounds the smallest positive ones to zero, about 1 % of them, and
    without their gradient a layer's would be off by 10 % where its other values' rounding costs 0.3 %. Same result and gradient as the plain layer, NaN included."""
    _float_gpu(x, "x")
    return _Relu.apply(x)


def active():
    """Whether this thread is inside ``saved_activations``."""
    return getattr(_active, "depth", 0) > 0


def active_for(x):
    """Whether this thread is inside ``saved_activations`` and x is of the tensors that it is for."""
    return active() and x.is_cuda and x.dtype in DTYPES


def _is_parameter(t):
    """A parameter, a view of one, or its copy in another type (what autocast hands to a layer)."""
    source = t if t._base is None else t._base
    if isinstance(source, torch.nn.Parameter) or (source.is_leaf and source.requires_grad):
        return True
    made = source.grad_fn
    return made is not None and made.name() == "ToCopyBackward0" and made.next_functions[0][0].name() == "torch::autograd::AccumulateGrad"


# The layers whose inputs are packed: products and convolutions are linear in what their backward pass reads, normalisations read their input against its own mean and spread, pooling
# asks for its shape alone. What other functions save stays as it is: autograd keeps a sigmoid's OUTPUT and multiplies by q (1 - q), an exp's or a softmax's likewise, and a log divides by
# its input. Half a step is an unbounded share of those (0.0005 next to a 0.2 has code 0: no gradient at all). Of a layer, its input alone: not a normalisation's reciprocal spreads.
_PRODUCTS = frozenset([torch.matmul, torch.mm, torch.bmm, torch.addmm, torch.baddbmm, torch.einsum] + [getattr(torch.Tensor, name) for name in "matmul __matmul__ __rmatmul__ mm bmm addmm baddbmm".split()])
_LAYERS = frozenset(getattr(module, name) for module, names in (
    (F, "conv1d conv2d conv3d conv_transpose1d conv_transpose2d conv_transpose3d linear batch_norm instance_norm group_norm layer_norm max_pool1d max_pool2d max_pool3d avg_pool1d avg_pool2d "
        "avg_pool3d adaptive_avg_pool1d adaptive_avg_pool2d adaptive_avg_pool3d adaptive_max_pool1d adaptive_max_pool2d adaptive_max_pool3d max_pool1d_with_indices max_pool2d_with_indices "
        "max_pool3d_with_indices adaptive_max_pool1d_with_indices adaptive_max_pool2d_with_indices adaptive_max_pool3d_with_indices"),
    (torch, "batch_norm instance_norm group_norm layer_norm max_pool1d max_pool2d max_pool3d")) for name in names.split())


class _Functions(TorchFunctionMode):
    """Notes for the hooks below how many values the inputs of the layer or product that is running have. (A composite function, such as an attention module's, is seen as one: what runs
    inside it is not.) The number, not the tensor: autocast and a layer's own reshaping hand autograd another one."""

    def __torch_function__(self, func, types, args=(), kwargs=None):
        kwargs = kwargs or {}
        inputs = (args[0] if args else kwargs.get("input"),) if func in _LAYERS else (*args, *kwargs.values()) if func in _PRODUCTS else ()
        before, _active.inputs = getattr(_active, "inputs", ()), [t.numel() for t in inputs if isinstance(t, torch.Tensor)]
        try:
            return func(*args, **kwargs)
        finally:
            _active.inputs = before


class saved_activations:
    """Context manager for a forward pass: the inputs of convolutions, matrix products, normalisations and poolings that autograd saves inside it -- floating-point GPU tensors of three or more
    dimensions and at least ``min_values`` values -- are kept as 8-bit checkpoints, where those are smaller, and restored when their backward runs. What other functions save (a sigmoid's,
    softmax's or plain ReLU's output, a logarithm's argument) is kept as it is, and so are a layer's weights and parameters (leaves that want a gradient, frozen nn.Parameters), views of them and
    autocast's copies of the former; a factor of a product that is computed from parameters is an activation here. In it, ``qnet``'s pointwise convolutions keep theirs for ``weight_grad`` and its ReLUs which values are positive (``relu``).

    A normalisation sees its input half a step off: where a group's values lie close together and far from 0, that is more of their spread than of themselves. What is kept must not be
    changed in place before the backward pass; unlike without the context, that is not noticed."""

    def __init__(self, min_values=4096):
        self.min_values = int(min_values)
        self._entered = []

    def _pack(self, t):
        if not (t.is_cuda and t.dtype in DTYPES and t.dim() >= 3 and t.numel() >= self.min_values and t.numel() in getattr(_active, "inputs", ())):
            return t
        return pack(t) if _smaller(t) and not _is_parameter(t) else t

    @staticmethod
    def _unpack(t):
        return t.unpack() if isinstance(t, PackedActivation) else t

    def __enter__(self):
        inside = contextlib.ExitStack()
        inside.enter_context(torch.autograd.graph.saved_tensors_hooks(self._pack, self._unpack))
        inside.enter_context(_Functions())
        self._entered.append(inside)
        _active.depth = getattr(_active, "depth", 0) + 1
        return self

    def __exit__(self, *exc):
        _active.depth -= 1
        return self._entered.pop().__exit__(*exc)
