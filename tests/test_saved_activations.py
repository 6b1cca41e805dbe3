"""What checkpoint8.saved_activations keeps in 8 bits and what it leaves alone, inside networks: saved outputs, functions with a pole, mixed and other types, module hooks."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from mujoco_rl_ur5_amd import checkpoint8, qnet


# ------------------------------------------------------------------ functions that are not linear in what they save
CURVED = [torch.sigmoid, torch.tanh, torch.exp, lambda x: x.exp().sqrt(), lambda x: x.exp().rsqrt(), lambda x: x.exp().reciprocal(), lambda x: x.exp().log(), lambda x: 1 / x.exp(),
          lambda x: x.exp() ** 0.25, lambda x: x.softmax(-1), lambda x: F.log_softmax(x, -1), lambda x: torch.sigmoid(x).log(), torch.relu, lambda x: torch.asin(x.sigmoid())]


@pytest.mark.gpu
@pytest.mark.parametrize("number", range(len(CURVED)))
def test_functions_that_are_not_linear_keep_what_they_save(number):
    """Half a step of a value is an unbounded share of q (1 - q), 1 / x or exp: the gradient is the plain one, bit for bit."""
    f = CURVED[number]
    x = (3 * torch.randn(4, 16, 130, generator=torch.Generator().manual_seed(number))).cuda().requires_grad_()
    up = torch.randn(x.shape, generator=torch.Generator().manual_seed(90)).cuda()
    want, = torch.autograd.grad(f(x * 1.0), x, up)
    with checkpoint8.saved_activations():
        y = f(x * 1.0)
    got, = torch.autograd.grad(y, x, up)
    assert torch.isfinite(want).all() and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [-6.0, -4.0, 0.0, 4.0, 6.0])
def test_q_maps_near_their_ends(shift):
    """The learner's expression -- sigmoid, gather, binary cross entropy -- on maps near 0 and near 1, where the samples that are most wrong have all of the gradient."""
    g = torch.Generator().manual_seed(4)
    z = (2 * torch.randn(12, 6, 40, 40, generator=g) + shift).cuda().requires_grad_()
    action, reward = torch.randint(0, 9600, (12, 1), generator=g).cuda(), torch.randint(0, 2, (12, 1), generator=g).float().cuda()
    def loss():
        return F.binary_cross_entropy(torch.sigmoid(z * 1.0).reshape(12, -1).gather(1, action), reward)
    want, = torch.autograd.grad(loss(), z)
    with checkpoint8.saved_activations():
        held = loss()
    got, = torch.autograd.grad(held, z)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [-6.0, 6.0])
def test_a_network_whose_maps_lie_near_their_ends(shift):
    """The whole Q network: the last bias' gradient is the sum of dL/dz, which no packed value enters; the others see their layers' inputs half a step off."""
    torch.manual_seed(0)
    net = qnet.MULTIDISCRETE_RESNET(6).cuda().train()
    with torch.no_grad():
        net[1].C1.bias += shift
    g = torch.Generator().manual_seed(5)
    x, action, reward = torch.rand(8, 4, 40, 40, generator=g).cuda(), torch.randint(0, 9600, (8, 1), generator=g).cuda(), torch.tensor([0.0, 1] * 4).view(8, 1).cuda()
    grads = []
    for packed in (False, True):
        net.zero_grad(set_to_none=True)
        if packed:
            with checkpoint8.saved_activations():
                q = net(x)
        else:
            q = net(x)
        F.binary_cross_entropy(q.reshape(8, -1).gather(1, action), reward).backward()
        grads.append({n: p.grad.clone() for n, p in net.named_parameters()})
    most = max(float(v.norm()) for v in grads[0].values())
    assert torch.allclose(grads[0]["1.C1.bias"], grads[1]["1.C1.bias"], rtol=1e-3, atol=1e-5)
    for name, a in grads[0].items():
        if float(a.norm()) > 1e-3 * most:
            assert float((a - grads[1][name]).norm() / a.norm()) < 0.15, name


LAYERS = {"conv2d": lambda x: F.conv2d(x, torch.ones(3, 16, 3, 3, device=x.device, requires_grad=True)), "matmul": lambda x: x.flatten(0, 1) @ torch.ones(64, 20, 5, device=x.device, requires_grad=True),
          "batch_norm": lambda x: nn.BatchNorm2d(16).to(x.device)(x),
          "group_norm": lambda x: nn.GroupNorm(4, 16).to(x.device)(x), "layer_norm": lambda x: F.layer_norm(x, (20,)), "max_pool2d": lambda x: nn.MaxPool2d(2)(x), "max_pool2d_indices": lambda x: nn.MaxPool2d(2, return_indices=True)(x)[0],
          "conv_transpose2d": lambda x: nn.ConvTranspose2d(16, 3, 2).to(x.device)(x)}


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(LAYERS))
def test_layers_still_pack_their_inputs(name, monkeypatch):
    x = torch.randn(4, 16, 20, 20, device="cuda").requires_grad_()
    seen, pack = [], checkpoint8.pack
    monkeypatch.setattr(checkpoint8, "pack", lambda t: seen.append(tuple(t.shape)) or pack(t))
    with checkpoint8.saved_activations():
        y = LAYERS[name](x * 1.0)
    assert seen and all(torch.Size(s).numel() == x.numel() for s in seen)
    torch.autograd.grad(y.sum(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("layer", ["layer_norm", "conv2d"])
def test_only_a_layers_input_is_packed(layer, monkeypatch):
    """Not the reciprocal spreads that a normalisation saves, whose own groups may differ by any factor, and not a weight that is computed."""
    g = torch.Generator().manual_seed(8)
    x = (torch.randn(16, 12, 64, 64, generator=g) * torch.exp(3 * torch.randn(16, 12, 64, 1, generator=g))).cuda().requires_grad_()
    gain = torch.rand(64, 12, 3, 3, device="cuda").requires_grad_()
    f = {"layer_norm": lambda h: F.layer_norm(h, (64,)), "conv2d": lambda h: F.conv2d(h, gain * 2.0)}[layer]
    seen, pack = [], checkpoint8.pack
    monkeypatch.setattr(checkpoint8, "pack", lambda t: seen.append(tuple(t.shape)) or pack(t))
    with checkpoint8.saved_activations():
        y = f(x * 1.0)
    assert seen == [tuple(x.shape)]
    up = torch.randn(y.shape, generator=g).cuda()
    got, = torch.autograd.grad(y, x, up)
    # the definition's gradient is the plain one of the restored input (a convolution's does not depend on it)
    back = pack(x.detach()).unpack().double().requires_grad_()
    z = back if layer == "layer_norm" else x.detach().double().requires_grad_()
    m = x.detach().double()
    if layer == "layer_norm":                                    # mean and spread are the exact input's
        mean, rstd = m.mean(-1, keepdim=True), (m.var(-1, keepdim=True, unbiased=False) + 1e-5).rsqrt()
        h, u = (z.detach() - mean) * rstd, up.double()
        want = rstd * (u - u.mean(-1, keepdim=True) - h * (u * h).mean(-1, keepdim=True))
    else:
        want = torch.nn.grad.conv2d_input(x.shape, (gain * 2.0).detach().double(), up.double())
    # up to 576 products of either sign added in 32 bits: 576 x 2^-24 = 3.4e-5 of their sizes, whose sum the largest entries come near
    assert float((got.double() - want).abs().amax()) <= 1e-4 * float(want.abs().amax())
    if layer == "layer_norm":                                    # row by row: their gradients differ in size as their spreads do
        off = (got.double() - want).abs().amax(-1) / want.abs().amax(-1)
        assert float(off.max()) < 1e-4


def test_the_context_knows_which_function_saves():
    """On the host: what it would be allowed to pack, function by function, also after an exception inside one."""
    context, seen = checkpoint8.saved_activations(), []
    context._pack = lambda t: seen.append(t.numel() in checkpoint8._active.inputs) or t
    x = torch.randn(2, 4, 20, 20).requires_grad_()
    for f, layer in ((nn.Conv2d(4, 5, 3, bias=False), True), (nn.BatchNorm2d(4), True), (nn.MaxPool2d(2), True), (lambda t: t.flatten(0, 1) @ torch.ones(8, 20, 3, requires_grad=True), True),
                     (torch.sigmoid, False), (lambda t: t.softmax(-1), False), (torch.exp, False), (lambda t: t * t, False), (lambda t: 1 / t, False)):
        del seen[:]
        with context:
            f(x)
        assert seen and any(seen) == layer
    del seen[:]
    with context:
        with pytest.raises(RuntimeError):
            nn.functional.conv2d(x, torch.ones(3, 5, 1, 1))
        del seen[:]                                              # (a convolution saves its input before it looks at the weight)
        with context:
            torch.exp(x)
        torch.exp(x)
    assert len(seen) == 2 and not any(seen) and not checkpoint8.active()


# ------------------------------------------------------------------ types
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per_image", [False, True])
def test_the_policy_network_under_autocast(dtype, per_image):
    """Inside the network a 16-bit activation meets fp32 weights. Same output as without checkpoints, and gradients near those."""
    import contextlib
    torch.manual_seed(1)
    net = qnet.MULTIDISCRETE_POLICY_RESNET(6).cuda().train()
    x = torch.rand(3, 4, 40, 40, device="cuda")
    up = torch.randn(3, 6, 40, 40, device="cuda")
    out = []
    for context in (contextlib.nullcontext(), checkpoint8.saved_activations()):
        net.zero_grad(set_to_none=True)
        with context, torch.autocast("cuda", dtype=dtype), (qnet.per_sample_statistics() if per_image else contextlib.nullcontext()):
            y = net(x)
        (y.float() * up).sum().backward()
        out.append((y.detach().float(), y.dtype, {n: p.grad.clone() for n, p in net.named_parameters()}))
    (y, t, grads), (y8, t8, grads8) = out
    # both runs round every layer to the same 16-bit type; where the library adds in another order a rounding may fall the other way, a step of the type per layer
    assert t == t8 and float((y - y8).norm() / y.norm()) < 8 * torch.finfo(dtype).eps
    most = max(float(v.norm()) for v in grads.values())
    for name, a in grads.items():
        assert grads8[name].dtype == a.dtype == torch.float32
        if float(a.norm()) > 1e-2 * most:
            assert float((a - grads8[name]).norm() / a.norm()) < 0.2, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("types", ["xh", "wh", "xw", "none"])
def test_pointwise_conv_of_mixed_types_under_autocast(dtype, types):
    g = torch.Generator().manual_seed(5)
    x, w, b = torch.randn(3, 20, 9, 14, generator=g).cuda(), torch.randn(11, 20, generator=g).cuda(), torch.randn(11, generator=g).cuda()
    x = (x.to(dtype) if "x" in types else x).requires_grad_()
    w = (w.to(dtype) if "w" in types else w).requires_grad_()
    b = b.requires_grad_()
    up = torch.randn(3, 11, 9, 14, generator=g).cuda()
    with torch.autocast("cuda", dtype=dtype):
        y = checkpoint8.pointwise_conv(x, w, b)
    grads = torch.autograd.grad(y, (x, w, b), up.to(y.dtype))
    assert [t.dtype for t in grads] == [x.dtype, w.dtype, b.dtype]
    want = torch.autograd.grad(F.conv2d(x.double(), w.double()[..., None, None], b.double()), (x, w, b), up.double())
    for a, e in zip(grads, want):                               # inputs half a checkpoint's step off, products rounded to the type: a few per cent of the largest entry is far over both
        assert float((a.double() - e.double()).abs().max()) < 0.03 * float(e.abs().max())
    if x.dtype != w.dtype:
        with pytest.raises(ValueError, match="does not fit"):   # without autocast nothing decides the product's type: refused, as the plain layer refuses it
            checkpoint8.pointwise_conv(x, w, b)


@pytest.mark.gpu
def test_a_network_of_another_type_is_left_alone():
    torch.manual_seed(2)
    block = qnet.BasicBlock(4, 6).cuda().double().train()
    x = torch.randn(2, 4, 30, 30, device="cuda", dtype=torch.double).requires_grad_()
    want = torch.autograd.grad(block(x).sum(), [x, *block.parameters()])
    with checkpoint8.saved_activations():
        y = block(x)
    got = torch.autograd.grad(y.sum(), [x, *block.parameters()])
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-9, atol=1e-9)


@pytest.mark.gpu
def test_pointwise_conv_refuses_a_bias_that_does_not_fit():
    x, w = torch.randn(2, 5, 3, 4).cuda(), torch.randn(7, 5).cuda()
    for bias in (torch.zeros(1).cuda(), torch.zeros(5).cuda(), torch.zeros(7), torch.zeros(7, 1).cuda(), torch.zeros(7, dtype=torch.double).cuda(), torch.zeros(7, dtype=torch.long).cuda(), 0.5):
        with pytest.raises(ValueError, match="bias"):
            checkpoint8.pointwise_conv(x, w, bias)


# ------------------------------------------------------------------ modules
@pytest.mark.gpu
def test_module_hooks_run_inside_the_context():
    torch.manual_seed(3)
    block = qnet.BasicBlock(8, 8).cuda().train()
    x = torch.randn(2, 8, 30, 30, device="cuda")
    calls = []
    block.relu.register_forward_hook(lambda m, i, o: calls.append(tuple(o.shape)))
    block(x)
    plain = list(calls)
    with checkpoint8.saved_activations():
        block(x)
    assert len(plain) == 2 and calls[2:] == plain
