"""Calls that something between the caller and the kernels would have to see: tracers, proxies, forward-mode
derivatives and function transforms.  The operators go past torch's dispatcher, so such a call is refused
rather than answered without them.  The refusals come before any other check, so host tensors show them."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from rfdetr_training_throughput_b200.linear import linear
from rfdetr_training_throughput_b200.norm import layer_norm
from rfdetr_training_throughput_b200.optim import adamw_step, dequantize_moments

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
WEIGHT = torch.randn(8, 8, generator=torch.Generator().manual_seed(1)).bfloat16()


def product(x):
    return linear(x, WEIGHT.to(x.device), activation="relu")


def square(x):
    return layer_norm(x) * 2


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("call", [product, square])
@pytest.mark.parametrize("grad", [False, True])
def test_traced_calls_are_refused(call, device, grad):
    x = torch.randn(4, 8).bfloat16().to(device).requires_grad_(grad)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(call)(x)


@pytest.mark.parametrize("device", DEVICES)
def test_traced_steps_are_refused(device):
    def step(p):
        q, m, v = p * 1, p * 0, p * 0
        adamw_step([q], [p], [m], [v], 1)
        return q

    def decoded(p):
        return dequantize_moments(p.to(torch.int8), p.to(torch.uint8), p[:1], p[:1])

    for call in (step, decoded):
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (torch.ones(7, device=device),), check_trace=False)
        with pytest.raises(RuntimeError, match="traced"):
            make_fx(call)(torch.ones(7, device=device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(device, which, grad):
    shapes = dict(x=(4, 8), weight=(8, 8), bias=(8,), residual=(4, 8))
    tensors = {k: torch.randn(s).bfloat16().to(device).requires_grad_(grad) for k, s in shapes.items()}
    with forward_ad.dual_level():
        tensors[which] = forward_ad.make_dual(tensors[which], torch.ones_like(tensors[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear(tensors["x"], tensors["weight"], tensors["bias"], residual=tensors["residual"])
        if which != "residual":
            with pytest.raises(RuntimeError, match="forward-mode"):
                layer_norm(tensors["x"], tensors["weight"][0], tensors["bias"])


@pytest.mark.gpu
@pytest.mark.parametrize("call", [product, square])
def test_tangents_of_a_gradient_are_refused(call):
    """Forward over reverse: the tangent comes in behind the operator, with the gradient of its output."""
    x = torch.randn(4, 8, device="cuda").bfloat16().requires_grad_(True)
    with forward_ad.dual_level():
        out = call(x)
        dy = forward_ad.make_dual(torch.ones_like(out), torch.ones_like(out))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(out, x, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("call", [product, square])
def test_other_tensors_inside_a_dual_level(call):
    """A dual level by itself refuses nothing."""
    x = torch.randn(4, 8, device="cuda").bfloat16()
    want = call(x)
    with forward_ad.dual_level():
        assert torch.equal(call(x), want)


@pytest.mark.gpu
@pytest.mark.parametrize("call", [product, square])
def test_function_transforms_are_refused(call):
    """vmap, jvp and grad of torch.func wrap what they pass in: no storage, no kernel."""
    x = torch.randn(2, 4, 8, device="cuda").bfloat16()
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(x)
    with pytest.raises(RuntimeError):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: call(t).float().sum())(x)
