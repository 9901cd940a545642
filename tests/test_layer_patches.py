"""The patches that install the layer operators: what they rebind, what keeps torch's path, and (on the
GPU) that a module computes through them what it computed before."""

import sys
import types

import pytest
import torch

from rfdetr_training_throughput_b200 import msda, optim, patches
from rfdetr_training_throughput_b200.linear import project


@pytest.fixture()
def restored(monkeypatch):
    """torch's own names come back after the test."""
    monkeypatch.setattr(torch.nn.LayerNorm, "forward", torch.nn.LayerNorm.forward)
    monkeypatch.setattr(torch.optim, "AdamW", torch.optim.AdamW)
    name = "rfdetr.models.ops.modules.ms_deform_attn"
    parts = name.split(".")
    for i in range(1, len(parts) + 1):
        monkeypatch.setitem(sys.modules, ".".join(parts[:i]), types.ModuleType(".".join(parts[:i])))
    sys.modules[name].MSDeformAttn = type("MSDeformAttn", (), {"forward": lambda self, *a, **k: "upstream",
                                                               "_export": False})
    return sys.modules[name]


def test_rebinding(restored):
    done = patches.apply_patches("fused_msda_linear,fused_layer_norm,fused_adamw")
    assert len(done) == 3 and all(":" in d for d in done)
    assert torch.optim.AdamW is optim.AdamW
    # host tensors, several normalised dimensions and other types keep torch's layer norm
    x = torch.randn(4, 6)
    assert torch.equal(torch.nn.LayerNorm(6)(x), torch.nn.functional.layer_norm(x, (6,)))
    wide = torch.nn.LayerNorm((4, 6))(x)
    assert torch.equal(wide, torch.nn.functional.layer_norm(x, (4, 6)))
    attn = restored.MSDeformAttn()
    attn._export = True
    assert attn.forward(1) == "upstream"


def test_host_projection_is_the_layer():
    layer, x = torch.nn.Linear(6, 5), torch.randn(3, 6)
    assert torch.equal(project(layer, x), layer(x))


class Module(torch.nn.Module):
    """The projections of a deformable attention module (d_model 64, 4 heads, 2 levels, 4 points)."""

    def __init__(self, d_model=64, heads=4, levels=2, points=4):
        super().__init__()
        self.d_model, self.n_heads, self.n_levels, self.n_points = d_model, heads, levels, points
        self.sampling_offsets = torch.nn.Linear(d_model, heads * levels * points * 2)
        self.attention_weights = torch.nn.Linear(d_model, heads * levels * points)
        self.value_proj = torch.nn.Linear(d_model, d_model)
        self.output_proj = torch.nn.Linear(d_model, d_model)


@pytest.mark.gpu
def test_attention_module_with_projected_layers(restored):
    """Under a bf16 autocast, with and without the library's products: the same four projections rounded
    to bf16 (each product may round to the neighbouring value: 2^-8 of it), a softmax, sums of samples
    and the output projection; 2 % of the output's norm is above what such roundings make.  Without
    autocast the products stay torch's: equal."""
    torch.manual_seed(0)
    dev = torch.device("cuda", 0)
    mod = Module().to(dev)
    shapes = torch.tensor([(12, 12), (6, 6)], device=dev)
    start = torch.tensor([0, 144], device=dev)
    query, flat = torch.randn(2, 30, 64, device=dev), torch.randn(2, 180, 64, device=dev)
    points = torch.rand(2, 30, 2, 2, device=dev)
    mask = torch.zeros(2, 180, dtype=torch.bool, device=dev)
    mask[1, 170:] = True
    args = (mod, query, points, flat, shapes, start, mask)
    assert torch.equal(msda.module_forward(*args), msda.module_forward(*args, project=project))
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a, b = msda.module_forward(*args), msda.module_forward(*args, project=project)
    assert a.dtype == b.dtype == torch.bfloat16
    assert float((a.double() - b.double()).norm() / a.double().norm()) < 0.02
    b.float().sum().backward()
    assert all(bool(p.grad.isfinite().all()) and bool(p.grad.any()) for p in mod.parameters())


@pytest.mark.gpu
def test_layer_norm_module(restored):
    dev = torch.device("cuda", 0)
    x = torch.randn(5, 7, 48, device=dev) * 3 + 1
    layer = torch.nn.LayerNorm(48).to(dev)
    with torch.no_grad():
        layer.weight.uniform_(0.5, 1.5)
        layer.bias.uniform_(-1, 1)
    before = layer(x)
    half = torch.nn.LayerNorm(48, elementwise_affine=False)(x.half())
    with torch.autocast("cuda", dtype=torch.bfloat16):
        auto = layer(x.bfloat16())
    patches.apply_patches("fused_layer_norm")
    # both in float32: 200 roundings of what enters a row are above either one's error
    bound = 200 * 2.0 ** -24 * (1.5 * (before.abs() + x.abs().mean(-1, keepdim=True)) + 1)
    assert bool(((layer(x) - before).abs() <= bound).all())
    assert float((torch.nn.LayerNorm(48, elementwise_affine=False)(x.half()) - half).abs().max()) <= 2.0 ** -8
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = layer(x.bfloat16())
    assert got.dtype == auto.dtype == torch.float32
    assert bool(((got - auto).abs() <= bound).all())
    with pytest.raises(RuntimeError):
        layer(torch.randn(3, 47, device=dev))  # torch's own error for a wrong shape


@pytest.mark.gpu
def test_adamw_by_torch_s_name(restored):
    """A model's parameters after five steps, by torch's AdamW in 64 bits and by the patched name."""
    def model(dtype):
        torch.manual_seed(1)
        return torch.nn.Linear(12, 7).to("cuda", dtype)

    ref, ours = model(torch.float64), model(torch.float32)
    a = torch.optim.AdamW(ref.parameters(), lr=1e-2, weight_decay=0.1)
    patches.apply_patches("fused_adamw")
    b = torch.optim.AdamW(ours.parameters(), lr=1e-2, weight_decay=0.1)
    assert isinstance(b, optim.AdamW)
    for t in range(5):
        for p, q in zip(ref.parameters(), ours.parameters()):
            g = torch.randn(p.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(t))
            p.grad, q.grad = g.double(), g.clone()
        a.step()
        b.step()
    for p, q in zip(ref.parameters(), ours.parameters()):
        # five steps' roundings: some 20 units each of parameters and updates of order 1
        assert float((p - q.double()).abs().max().detach()) <= 100 * 2.0 ** -24
