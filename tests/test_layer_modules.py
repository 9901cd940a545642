"""What the patches of the layer operators leave to torch: arguments by torch's names, modules that do more
than their weight says, and calls that a tracer, a compiler or a transform has to see."""

import sys
import types

import pytest
import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.nn.utils import parametrize

from rfdetr_training_throughput_b200 import linear as products
from rfdetr_training_throughput_b200 import patches
from rfdetr_training_throughput_b200.linear import project

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.fixture()
def norms(monkeypatch):
    """torch.nn.LayerNorm with the patch applied, torch's own forward back after the test."""
    monkeypatch.setattr(torch.nn.LayerNorm, "forward", torch.nn.LayerNorm.forward)
    patches.apply_patches("fused_layer_norm")


def norm_layer(device, dtype=torch.float32):
    torch.manual_seed(3)
    layer = torch.nn.LayerNorm(16).to(device, dtype)
    with torch.no_grad():
        layer.weight.uniform_(0.5, 1.5)
        layer.bias.uniform_(-1, 1)
    return layer, torch.randn(5, 16, device=device, dtype=dtype)


def own(layer, x):
    return F.layer_norm(x, layer.normalized_shape, layer.weight, layer.bias, layer.eps)


def near(got, want):
    """Two float32 layer norms of 16 values: 100 roundings of values of order 4."""
    return bool(((got - want).abs() <= 400 * 2.0 ** -24).all())


@pytest.mark.parametrize("device", DEVICES)
def test_layer_norm_by_torch_s_argument_name(norms, device):
    layer, x = norm_layer(device)
    assert near(layer(input=x), own(layer, x))


@pytest.mark.parametrize("device", DEVICES)
def test_layer_norm_traced(norms, device):
    """A trace holds torch's layer norm: it computes, also on other inputs."""
    layer, x = norm_layer(device)
    other = x * 2 + 1
    graph = torch.jit.trace(layer, (x,))
    assert "layer_norm" in str(graph.graph) and torch.equal(graph(other), own(layer, other))
    fx = make_fx(layer)(x)
    assert near(fx(other), own(layer, other))
    exported = torch.export.export(layer, (x,)).module()
    assert near(exported(other), own(layer, other))


@pytest.mark.parametrize("device", DEVICES)
def test_layer_norm_compiled(norms, device):
    layer, x = norm_layer(device)
    assert near(torch.compile(layer, backend="eager", fullgraph=True)(x), own(layer, x))
    torch._dynamo.reset()


@pytest.mark.parametrize("device", DEVICES)
def test_layer_norm_scripted(norms, device):
    """A scripted module holds torch's layer norm."""
    class Block(torch.nn.Module):
        def __init__(self, norm):
            super().__init__()
            self.norm = norm

        def forward(self, x):
            return self.norm(x) * 2

    layer, x = norm_layer(device)
    assert near(torch.jit.script(Block(layer))(x) / 2, own(layer, x))


@pytest.mark.parametrize("device", DEVICES)
def test_layer_norm_under_transforms(norms, device):
    """vmap, jvp, forward-mode and a second derivative by functorch, as torch's module has them."""
    layer, x = norm_layer(device)
    t = torch.ones_like(x).cumsum(0)
    want, tangent = torch.func.jvp(lambda v: own(layer, v), (x,), (t,))
    got = torch.func.jvp(layer, (x,), (t,))
    assert near(got[0], want) and near(got[1], tangent)
    with forward_ad.dual_level():
        out = forward_ad.unpack_dual(layer(forward_ad.make_dual(x, t)))
    assert near(out.primal, want) and near(out.tangent, tangent)
    assert near(torch.func.vmap(layer)(x[:, None]), want[:, None])
    grad = torch.func.grad(lambda v: own(layer, v).square().sum())(x)
    assert near(torch.func.grad(lambda v: layer(v).square().sum())(x) / 16, grad / 16)


# ------------------------------------------------------------------ projections

class Twice(torch.nn.Linear):
    """A subclass whose forward adds a term of its own, as adapters do."""

    def forward(self, x):
        return super().forward(x) + 1


class Halved(torch.nn.Module):
    def forward(self, w):
        return w / 2


def plain(device):
    torch.manual_seed(4)
    return torch.nn.Linear(16, 8).to(device, torch.bfloat16)


def hooked(kind):
    def make(device):
        layer = plain(device)
        getattr(layer, f"register_{kind}")(HOOKS[kind])
        return layer
    return make


HOOKS = {"forward_hook": lambda m, a, out: out + 1, "forward_pre_hook": lambda m, a: (a[0] * 2,),
         "full_backward_hook": lambda m, gi, go: tuple(None if g is None else g * 3 for g in gi),
         "full_backward_pre_hook": lambda m, go: tuple(g * 3 for g in go)}


def subclass(device):
    torch.manual_seed(4)
    return Twice(16, 8).to(device, torch.bfloat16)


def parametrized(device):
    layer = plain(device)
    parametrize.register_parametrization(layer, "weight", Halved())
    return layer


def rebound(device):
    layer = plain(device)
    layer.forward = lambda x: F.linear(x, layer.weight, layer.bias) - 1
    return layer


def wrapper(device):
    class Adapter(torch.nn.Module):
        def __init__(self, base):
            super().__init__()
            self.base = base

        weight = property(lambda self: self.base.weight)
        bias = property(lambda self: self.base.bias)

        def forward(self, x):
            return self.base(x) + x[..., :8]

    return Adapter(plain(device))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("make", [*(pytest.param(hooked(k), id=k) for k in HOOKS), subclass, parametrized, rebound,
                                  wrapper])
def test_layers_that_do_more_are_called(make, device):
    layer = make(device)
    x = torch.randn(5, 16, device=device).bfloat16().requires_grad_(True)
    want, got = layer(x), project(layer, x)
    assert torch.equal(got, want)
    (a,) = torch.autograd.grad(want.float().sum(), x)
    (b,) = torch.autograd.grad(got.float().sum(), x)
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_global_hooks_are_called():
    layer, x = plain("cuda"), torch.randn(5, 16, device="cuda").bfloat16()
    hook = torch.nn.modules.module.register_module_forward_hook(lambda m, a, out: out * 2)
    try:
        assert torch.equal(project(layer, x), layer(x))
    finally:
        hook.remove()


@pytest.mark.gpu
def test_a_plain_layer_runs_on_the_kernels(monkeypatch):
    """... and a float64 input under autocast, which torch's autocast leaves alone, on torch."""
    calls = []
    kernel = products.linear
    monkeypatch.setattr(products, "linear", lambda *a, **k: calls.append(1) or kernel(*a, **k))
    layer = torch.nn.Linear(16, 8).cuda()
    x = torch.randn(5, 16, device="cuda")
    project(plain("cuda"), x.bfloat16())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        project(layer, x)
    assert len(calls) == 2
    with torch.autocast("cuda", dtype=torch.bfloat16):
        wide = layer.double()
        assert project(wide, x.double()).dtype == torch.float64
    assert len(calls) == 2


class Projecting(torch.nn.Module):
    def __init__(self, layer):
        super().__init__()
        self.layer = layer

    def forward(self, x):
        return project(self.layer, x)


@pytest.mark.parametrize("device", DEVICES)
def test_traced_projection(device):
    layer, x = plain(device), torch.randn(5, 16, device=device).bfloat16()
    graph = torch.jit.trace(Projecting(layer), (x,))
    assert torch.equal(graph(x * 2), layer(x * 2))
    out, tangent = torch.func.jvp(Projecting(layer), (x,), (torch.ones_like(x),))
    assert torch.equal(out, layer(x)) and tangent.shape == out.shape


@pytest.mark.parametrize("device", DEVICES)
def test_traced_attention_keeps_the_original(device, monkeypatch):
    name = "rfdetr.models.ops.modules.ms_deform_attn"
    parts = name.split(".")
    for i in range(1, len(parts) + 1):
        monkeypatch.setitem(sys.modules, ".".join(parts[:i]), types.ModuleType(".".join(parts[:i])))
    cls = type("MSDeformAttn", (), {"forward": lambda self, x: x * 3, "_export": False})
    sys.modules[name].MSDeformAttn = cls
    patches.apply_patches("fused_msda_linear")
    attn, x = cls(), torch.ones(2, device=device)
    # the check would call the stand-in untraced, with arguments that the module does not take
    assert torch.equal(torch.jit.trace(attn.forward, (x,), check_trace=False)(x * 2), x * 6)
