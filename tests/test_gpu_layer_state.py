"""What the layer operators hold between a forward and its backward, what counts as written, and when their
fault mark can be read."""

import pytest
import torch

from rfdetr_training_throughput_b200.linear import check_faults, linear
from rfdetr_training_throughput_b200.optim import adamw_step, quantize_moments

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def operands(rows=64, inner=48, outer=40):
    g = torch.Generator(device="cuda").manual_seed(0)

    def normal(*shape):
        return torch.randn(*shape, device=DEV, generator=g).bfloat16()

    return dict(x=normal(rows, inner), weight=normal(outer, inner), bias=normal(outer), residual=normal(rows, outer),
                dy=normal(rows, outer))


@pytest.mark.parametrize("inner", [48, 45])  # 45: operands that have to be copied
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("wanted", [("x",), ("weight",), ("bias",), ("residual",), ("x", "bias"),
                                    ("weight", "residual")])
def test_only_what_the_gradients_need_is_kept(wanted, act, inner):
    """Operands that no wanted gradient reads may change before the backward: the bits stay those of an
    unchanged one.  Those that one reads may not."""
    d = operands(inner=inner)
    needed = {"weight"} if "x" in wanted else {"x"} if "weight" in wanted else set()

    def grads(change):
        t = {k: d[k].clone() for k in ("x", "weight", "bias", "residual")}
        for k in wanted:
            t[k].requires_grad_(True)
        out = linear(t["x"], t["weight"], t["bias"], activation=act, residual=t["residual"])
        with torch.no_grad():
            for k in change:
                t[k].add_(1)
        return torch.autograd.grad(out, [t[k] for k in wanted], d["dy"])

    free = [k for k in ("x", "weight", "bias", "residual") if k not in needed]
    for a, b in zip(grads([]), grads(free)):
        assert torch.equal(a, b)
    for k in needed:
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            grads([k])


@pytest.mark.parametrize("leaf", ["x", "weight", "residual"])
def test_memory_between_forward_and_backward(leaf):
    """An operand that no wanted gradient reads is freed with its last reference."""
    rows, inner, outer = (64, 512, 65536) if leaf == "weight" else (65536, 512, 64)
    sizes = dict(x=(rows, inner), weight=(outer, inner), residual=(rows, outer))
    leaves = {k: torch.zeros(s, device=DEV, dtype=torch.bfloat16, requires_grad=k == leaf) for k, s in sizes.items()}
    passing = {k: t * 1 for k, t in leaves.items()}
    out = linear(passing["x"], passing["weight"], activation="gelu", residual=passing["residual"])
    passing.clear()
    before = torch.cuda.memory_allocated()
    del out
    freed = before - torch.cuda.memory_allocated()
    # the output; the pre-activation and the one operand that the gradient reads, where it reads any
    values = rows * outer
    if leaf != "residual":
        values += rows * outer + (outer * inner if leaf == "x" else rows * inner)
    assert freed <= 2 * values + 4096


def test_faults_are_read_after_everything():
    """check_faults waits for streams that do not synchronise with the default one."""
    side = torch.cuda.Stream()
    x = torch.zeros(128, 64, device=DEV, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # some 100 ms
        linear(x, x)
        done.record()
    check_faults()
    assert done.query()


@pytest.mark.parametrize("which", ["param", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"])
def test_written_tensors_count_as_changed(which):
    """A graph that saved something the step writes says so instead of using the new values."""
    p, g, m, v = (torch.rand(600, device=DEV) for _ in range(4))
    eight = "scale" in which
    cm, cv, sm, sv = quantize_moments(m, v)
    saved = dict(param=p, exp_avg=m, exp_avg_sq=v, exp_avg_scale=sm, exp_avg_sq_scale=sv)[which]
    w = torch.ones_like(saved, requires_grad=True)
    loss = (w * saved).sum()
    if eight:
        adamw_step([p], [g], [cm], [cv], 1, scales=([sm], [sv]))
    else:
        adamw_step([p], [g], [m], [v], 1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_inference_tensors_are_not_written_outside_inference_mode():
    """... as torch's in-place operations: refused before anything is written."""
    with torch.inference_mode():
        p = torch.rand(600, device=DEV)
    g, m, v = (torch.rand(600, device=DEV) for _ in range(3))
    before = [t.clone() for t in (p, m, v)]
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        adamw_step([p], [g], [m], [v], 1)
    assert all(torch.equal(a, b) for a, b in zip((p, m, v), before))
    with torch.inference_mode():
        adamw_step([p], [g], [m], [v], 1)
    assert not torch.equal(p, before[0])


def test_device_scalars_apart_from_what_is_written():
    """A scalar inside a written tensor would be read by some blocks before and by some after its update."""
    p, g, m, v = (torch.rand(5000, device=DEV) for _ in range(4))
    one = torch.ones(1, device=DEV)
    for bad in (p[10:11], m[-1:], v[:1]):
        with pytest.raises(ValueError, match="share memory"):
            adamw_step([p], [g], [m], [v], 1, grad_scale=bad)
        with pytest.raises(ValueError, match="share memory"):
            adamw_step([p], [g], [m], [v], 1, lr=bad)
    step = torch.ones(1, dtype=torch.int64, device=DEV)
    with pytest.raises(ValueError, match="share memory"):
        adamw_step([step.view(torch.float32)], [one.repeat(2)], [torch.zeros(2, device=DEV)],
                   [torch.zeros(2, device=DEV)], step)
    adamw_step([p], [g], [m], [v], 1, grad_scale=g[:1], lr=one)  # a gradient's element is only read
