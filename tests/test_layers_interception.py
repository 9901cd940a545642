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
