"""AdamW's bookkeeping: which parameters share a step counter, when counters and states move, and what a
capture may hold.  The host tests put the step itself in plain torch in the place of the kernel."""

import copy

import pytest
import torch

from rfdetr_training_throughput_b200 import optim
from rfdetr_training_throughput_b200.optim import AdamW

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def plain_step(params, grads, exp_avg, exp_avg_sq, step, *, scales=None, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2, grad_scale=None):
    t, (b1, b2) = int(step), betas
    if any(p.dtype != g.dtype for p, g in zip(params, grads)):
        raise ValueError("grads must be of the params' type")
    for p, g, m, v in zip(params, grads, exp_avg, exp_avg_sq):
        m.mul_(b1).add_(g.float(), alpha=1 - b1)
        v.mul_(b2).addcmul_(g.float(), g.float(), value=1 - b2)
        p.copy_(p.float() * (1 - lr * weight_decay) - lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps))


@pytest.fixture(autouse=True)
def host_step(request, monkeypatch):
    if request.node.callspec.params.get("device") == "cpu":
        monkeypatch.setattr(optim, "adamw_step", plain_step)


def parameters(device, types, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(40 + 3 * i, generator=g).to(device, t)) for i, t in enumerate(types)]


def set_grads(params, t, skip=()):
    for i, p in enumerate(params):
        g = torch.randn(p.shape, generator=torch.Generator().manual_seed(100 * t + i))
        p.grad = None if i in skip else g.to(p.device, p.dtype)


def counts(opt, params):
    return [int(opt.state[p]["step"]) if opt.state.get(p) else 0 for p in params]


def check_alike(a, pa, b, pb):
    """Parameters, moments and counts of two optimisers, bit for bit."""
    for p, q in zip(pa, pb):
        assert torch.equal(p, q)
        assert bool(a.state.get(p)) == bool(b.state.get(q))
        for k, x in a.state.get(p, {}).items():
            y = b.state[q][k]
            assert int(x) == int(y) if k == "step" else torch.equal(x, y), k


MIXED = [torch.float32, torch.bfloat16, torch.float32, torch.float16]


@pytest.mark.parametrize("device", DEVICES)
def test_capturable_group_of_mixed_types(device):
    """One counter advances once a step whatever the types; the same bits as with host counters."""
    ours, ref = parameters(device, MIXED), parameters(device, MIXED)
    a, b = AdamW(ours, lr=1e-2, capturable=True), AdamW(ref, lr=1e-2)
    for t in range(3):
        set_grads(ours, t)
        set_grads(ref, t)
        a.step()
        b.step()
        assert counts(a, ours) == [t + 1] * 4
    check_alike(a, ours, b, ref)
    # through a state dict, in both directions
    again = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    c = AdamW(again, lr=1e-2, capturable=True)
    c.load_state_dict(copy.deepcopy(a.state_dict()))
    for t in range(3, 5):
        set_grads(again, t)
        set_grads(ref, t)
        c.step()
        b.step()
    check_alike(c, again, b, ref)


@pytest.mark.parametrize("device", DEVICES)
def test_capturable_after_a_change_of_type(device):
    """Parameters that shared a counter and no longer have one type."""
    ours, ref = parameters(device, [torch.float32] * 3), parameters(device, [torch.float32] * 3)
    a, b = AdamW(ours, lr=1e-2, capturable=True), AdamW(ref, lr=1e-2)
    for t in range(4):
        if t == 2:
            for p in (ours[1], ref[1]):
                p.grad = None
                p.data = p.data.bfloat16()
        set_grads(ours, t)
        set_grads(ref, t)
        a.step()
        b.step()
    assert counts(a, ours) == [4] * 3
    check_alike(a, ours, b, ref)


@pytest.mark.parametrize("device", DEVICES)
def test_capturable_with_absent_gradients(device):
    """A parameter without a gradient is passed over and its count stands, as with torch's AdamW."""
    ours, ref = parameters(device, MIXED), parameters(device, MIXED)
    a, b = AdamW(ours, lr=1e-2, capturable=True), AdamW(ref, lr=1e-2)
    absent = [(), (0,), (0, 1), (), (2,), (0, 1, 2, 3), ()]
    for t, skip in enumerate(absent):
        set_grads(ours, t, skip)
        set_grads(ref, t, skip)
        a.step()
        b.step()
    assert counts(a, ours) == [sum(i not in s for s in absent) for i in range(4)]
    check_alike(a, ours, b, ref)


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("device", DEVICES)
def test_a_refused_step_leaves_everything(device, capturable, monkeypatch):
    """A step that is refused moves no counter and makes no state, whether it is the first or a later one."""
    params = parameters(device, [torch.float32] * 2)
    opt = AdamW(params, lr=1e-2, capturable=capturable)
    step = optim.adamw_step

    def refuse(*args, **kwargs):
        raise ValueError("refused")

    set_grads(params, 0)
    for done in (0, 1):
        monkeypatch.setattr(optim, "adamw_step", refuse)
        for _ in range(2):
            with pytest.raises(ValueError, match="refused"):
                opt.step()
        assert counts(opt, params) == [done] * 2 and (done or not opt.state)
        monkeypatch.setattr(optim, "adamw_step", step)
        opt.step()
        assert counts(opt, params) == [done + 1] * 2
    ref = parameters(device, [torch.float32] * 2)
    other = AdamW(ref, lr=1e-2)
    set_grads(ref, 0)
    other.step()
    other.step()
    check_alike(opt, params, other, ref)


@pytest.mark.parametrize("device", DEVICES)
def test_a_refusal_among_buckets(device):
    """Two types, two launches: what was launched has counted, what was refused has not."""
    params = parameters(device, [torch.float32, torch.bfloat16])
    opt = AdamW(params, lr=1e-2)
    set_grads(params, 0)
    wrong = params[1].grad
    params[1].grad = None
    opt.step()
    params[1].grad = wrong.to_sparse()
    with pytest.raises(ValueError, match="sparse"):
        opt.step()
    assert counts(opt, params) == [1, 0]  # seen before anything is launched


@pytest.mark.parametrize("device", ["cpu"])
def test_no_new_counter_inside_a_capture(device, monkeypatch):
    """A replay would set it back every time."""
    params = parameters(device, [torch.float32] * 2)
    opt = AdamW(params, lr=1e-2, capturable=True)
    set_grads(params, 0)
    opt.step()
    monkeypatch.setattr(optim, "_capturing", lambda: True)
    opt.step()
    assert counts(opt, params) == [2, 2]
    set_grads(params, 1, skip=(0,))
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    # nor later: the graph would go on counting for the parameter that left its counter
    monkeypatch.setattr(optim, "_capturing", lambda: False)
    with pytest.raises(RuntimeError, match="captured"):
        opt.step()
    assert counts(opt, params) == [2, 2]


@pytest.mark.parametrize("device", ["cpu"])
def test_no_host_counter_inside_a_capture(device, monkeypatch):
    """It would stay at the captured step's number in every replay."""
    params = parameters(device, [torch.float32] * 2)
    opt = AdamW(params, lr=1e-2)
    set_grads(params, 0)
    opt.step()
    before = [p.detach().clone() for p in params]
    monkeypatch.setattr(optim, "_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="capturable"):
        opt.step()
    assert counts(opt, params) == [1, 1] and all(torch.equal(p, q) for p, q in zip(params, before))


@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda"])
def test_host_counter_in_a_real_capture(device):
    params = parameters(device, MIXED)
    opt = AdamW(params, lr=1e-2)
    set_grads(params, 0)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capturable"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    assert counts(opt, params) == [1] * 4


@pytest.mark.gpu
@pytest.mark.parametrize("device", ["cuda"])
def test_captured_with_absent_gradients(device):
    """Mixed types, and a parameter that stopped having gradients before the capture."""
    ours, ref = parameters(device, MIXED), parameters(device, MIXED)
    a, b = AdamW(ours, lr=1e-2, capturable=True), AdamW(ref, lr=1e-2)
    for t, skip in enumerate([(), (2,)]):
        set_grads(ours, t, skip)
        set_grads(ref, t, skip)
        a.step()
        b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    grads = [p.grad for p in ours]
    for t in range(2, 5):
        set_grads(ref, t, (2,))
        for g, q in zip(grads, ref):
            if g is not None:
                g.copy_(q.grad)
        graph.replay()
        b.step()
    torch.cuda.synchronize()
    check_alike(a, ours, b, ref)
