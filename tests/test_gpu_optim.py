"""adamw_step and AdamW against the formula: 32-bit moments in 64 bits, 8-bit ones bit for bit.

Tolerances (u = 2^-24): m and v are two products and a sum (v one product more), so each is off by at
most 4 u of the sum of its terms' magnitudes, the coefficients themselves by u.  The update is a
quotient of such values (a root, a product, a sum, a quotient, two products: 12 u), applied to a
parameter with two more roundings, and to half a step of the parameter's type."""

import math

import numpy as np
import pytest
import torch

from rfdetr_training_throughput_b200 import optim
from rfdetr_training_throughput_b200.optim import AdamW, adamw_step, dequantize_moments, quantize_moments

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
ARGS = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)
SIZES = [1, 2, 3, 4, 5, 255, 256, 257, 511, 512, 513, 4095, 4096, 4097, 9001, 0, 128 * 300]


def values(sizes, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, device=DEV, generator=g) * scale).to(dtype) for n in sizes]


def close(got, want, bound):
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.2f} bounds"


def check32(p0, g, m0, v0, t, got, grad_scale=1.0, lr=ARGS["lr"]):
    """One tensor's step in 64 bits, and the bounds above."""
    p, m, v = got
    dtype = p.dtype
    (b1, b2), eps, wd = ARGS["betas"], ARGS["eps"], ARGS["weight_decay"]
    p0, g, m0, v0 = (x.double() for x in (p0, g, m0, v0))
    g = g * grad_scale
    want_m, size_m = b1 * m0 + (1 - b1) * g, (b1 * m0).abs() + ((1 - b1) * g).abs()
    want_v = b2 * v0 + (1 - b2) * g * g
    close(m, want_m, 6 * U * size_m + 1e-45)
    close(v, want_v, 6 * U * want_v + 1e-44)
    rate = lr / (1 - b1 ** t)
    denom = (want_v / (1 - b2 ** t)).sqrt() + eps
    want = p0 * (1 - lr * wd) - rate * want_m / denom
    loose = 4 * U * p0.abs() + rate / denom * (14 * U * want_m.abs() + 6 * U * size_m)
    close(p, want, loose + torch.finfo(dtype).eps / 2 * (want.abs() + loose)
          + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("step", [1, 2, 1000])
def test_32_bits(dtype, step):
    p, g = values(SIZES, dtype, 1), values(SIZES, dtype, 2, 0.1)
    m, v = values(SIZES, torch.float32, 3, 0.05), [x.square() for x in values(SIZES, torch.float32, 4, 0.1)]
    before = [[x.clone() for x in one] for one in (p, g, m, v)]
    adamw_step(p, g, m, v, step, **ARGS)
    for i in range(len(SIZES)):
        assert torch.equal(g[i], before[1][i])
        check32(*(one[i] for one in before), step, (p[i], m[i], v[i]))


def test_unaligned_views_and_neighbours():
    """Tensors at odd places of one buffer; what lies between them stays."""
    sizes, gap = [5, 300, 1023, 4100], 3
    total = sum(sizes) + gap * (len(sizes) + 1)
    bufs = [values([total], torch.float32, k, 0.1)[0] for k in range(4)]
    bufs[3].square_()
    old = [b.clone() for b in bufs]
    starts, at = [], gap
    for n in sizes:
        starts.append(at)
        at += n + gap
    lists = [[b[s:s + n] for s, n in zip(starts, sizes)] for b in bufs]
    adamw_step(*lists, 7, **ARGS)
    inside = torch.zeros(total, dtype=torch.bool, device=DEV)
    for s, n in zip(starts, sizes):
        inside[s:s + n] = True
        check32(*(o[s:s + n] for o in old), 7, (bufs[0][s:s + n], bufs[2][s:s + n], bufs[3][s:s + n]))
    for b, o in zip(bufs, old):
        assert torch.equal(b[~inside], o[~inside])


@pytest.mark.parametrize("count", [60, 61, 508, 509, 1100])
def test_many_tensors(count):
    """The small table, the large one, and more than one launch."""
    sizes = [(i * 37) % 700 + (i % 5 == 0) * 5000 for i in range(count)]
    p, g = values(sizes, torch.float32, 1), values(sizes, torch.float32, 2, 0.1)
    m, v = values(sizes, torch.float32, 3, 0.05), [x.square() for x in values(sizes, torch.float32, 4, 0.1)]
    before = [torch.cat([x.clone() for x in one]) for one in (p, g, m, v)]
    adamw_step(p, g, m, v, 3, **ARGS)
    check32(*before, 3, (torch.cat(p), torch.cat(m), torch.cat(v)))


# ------------------------------------------------------------------ 8 bits

F = np.float32


def mix(h):
    h = (h * 0x9E3779B1) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x85C1E8B7) & 0xFFFFFFFF
    return h ^ (h >> 13)


def decode(cm, cv, sm, sv):
    n = cm.size
    a, b = cm.astype(F) * F(1 / 127), cv.astype(F) * F(1 / 255)
    b = b * b
    return np.repeat(sm, 256)[:n] * (a * np.abs(a)), np.repeat(sv, 256)[:n] * (b * b)


def step8(p, g, cm, cv, sm, sv, t, ordinal):
    """One tensor's step by the definition, in float32 operations of numpy (each rounded by itself)."""
    n = g.size
    b1, b2 = ARGS["betas"]
    m, v = decode(cm, cv, sm, sv)
    m = m * F(b1) + g * F(1 - b1)
    v = v * F(b2) + (g * g) * F(1 - b2)
    pad = -n % 256
    top = lambda x: np.abs(np.pad(x, (0, pad))).reshape(-1, 256).max(1)  # noqa: E731
    sm, sv = top(m), top(v)
    key = mix((ordinal * 0x632BE5AB + t * 0xC2B2AE35) & 0xFFFFFFFF)
    h = mix((np.arange(n, dtype=np.uint64) + np.uint64(key)) & np.uint64(0xFFFFFFFF))
    low, high = ((h & np.uint64(0xFFFF)).astype(F) * F(2.0 ** -16), (h >> np.uint64(16)).astype(F) * F(2.0 ** -16))
    with np.errstate(all="ignore"):
        x = np.sqrt(np.abs(m) / np.repeat(sm, 256)[:n]) * F(127) + low
        y = np.sqrt(np.sqrt(v / np.repeat(sv, 256)[:n])) * F(255) + high
    qm = np.minimum(np.floor(np.nan_to_num(x, nan=0.0)), 127)
    qv = np.minimum(np.floor(np.nan_to_num(y, nan=0.0)), 255)
    qv = np.where(v > 0, np.maximum(qv, 1), qv)
    return m, v, np.where(m < 0, -qm, qm).astype(np.int8), qv.astype(np.uint8), sm, sv


def eight(sizes, seed):
    m, v = values(sizes, torch.float32, seed, 0.05), [x.square() for x in values(sizes, torch.float32, seed + 1, 0.1)]
    packed = [quantize_moments(a, b) for a, b in zip(m, v)]
    return [list(x) for x in zip(*packed)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_8_bits_bit_for_bit(dtype):
    sizes = [n for n in SIZES if n]
    p = values(sizes, dtype, 1)
    cm, cv, sm, sv = eight(sizes, 3)
    for t in (1, 2, 3):
        g = values(sizes, dtype, 20 + t, 0.1)
        old = [[x.clone() for x in one] for one in (p, g, cm, cv, sm, sv)]
        adamw_step(p, g, cm, cv, t, scales=(sm, sv), **ARGS)
        for i in range(len(sizes)):
            host = [one[i].float().cpu().numpy() if one[i].is_floating_point() else one[i].cpu().numpy()
                    for one in old]
            m, v, qm, qv, nsm, nsv = step8(*host, t, i)
            assert np.array_equal(sm[i].cpu().numpy(), nsm) and np.array_equal(sv[i].cpu().numpy(), nsv)
            assert np.array_equal(cm[i].cpu().numpy(), qm) and np.array_equal(cv[i].cpu().numpy(), qv)
            # the parameter moves by the moments before they are rounded to codes
            want_m, want_v = decode(qm, qv, nsm, nsv)
            got_m, got_v = dequantize_moments(cm[i], cv[i], sm[i], sv[i])
            assert np.array_equal(got_m.cpu().numpy(), want_m) and np.array_equal(got_v.cpu().numpy(), want_v)
            before = decode(*host[2:])
            tensors = [torch.from_numpy(x.astype(np.float32)).to(DEV) for x in (*before, m, v)]
            check32(old[0][i], old[1][i], tensors[0], tensors[1], t, (p[i], tensors[2], tensors[3]))


def test_8_bits_zero_and_special_blocks():
    n = 256 * 4 + 10
    p = torch.zeros(n, device=DEV)
    g = torch.zeros(n, device=DEV)
    g[256:512] = 1e-30         # squares underflow to zero
    g[600] = float("nan")
    g[1030] = float("inf")     # the ragged last block
    g[800:] += 0.5
    cm, cv = torch.zeros(n, dtype=torch.int8, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV)
    sm, sv = torch.zeros(5, device=DEV), torch.zeros(5, device=DEV)
    adamw_step([p], [g], [cm], [cv], 1, scales=([sm], [sv]), **ARGS)
    m, v = dequantize_moments(cm, cv, sm, sv)
    assert not m[:256].any() and not v[:256].any() and not p[:256].any()
    assert bool(m[256:512].isfinite().all()) and bool(p[256:512].isfinite().all())
    assert bool(m[512:768].isnan().all()) and bool(v[512:768].isnan().all())  # its block is poisoned
    assert bool(m[768:1024].isfinite().all()) and bool(p[768:1024].isfinite().all())
    # m: 0 * inf and NaN codes (0) * inf; v: the scale is inf and a code of a nonzero v at least 1
    assert bool(m[1024:].isnan().any()) and not bool(m[1024:].isfinite().any())
    assert bool((v[1024:] == float("inf")).all())


def test_8_bit_rounding_is_unbiased_and_not_stuck():
    """A second moment whose target is 4 times its value rises along the exact average: after 1000 steps
    of b2 = 0.999 by 1 - 0.999^1000 = 63 % of the way.  One block of equal elements would share the scale;
    a large element holds it, so the others live at code 255 / sqrt(2) = 180 or so.  Codes are rounded one
    by one (independent between elements), each step adding at most a quarter code^2 of variance that the
    average over 248 elements divides: the mean of v stays within 5 % of the exact one."""
    n = 256
    g = torch.full((n,), 1e-3, device=DEV)
    g[:8] = 4e-3
    p = torch.zeros(n, device=DEV)
    v0 = (g * 0.5).square()
    v0[:8] = g[:8].square()
    cm, cv, sm, sv = quantize_moments(torch.zeros(n, device=DEV), v0)
    _, start = dequantize_moments(cm, cv, sm, sv)
    for t in range(1, 1001):
        adamw_step([p], [g], [cm], [cv], t, scales=([sm], [sv]), lr=0.0, betas=(0.9, 0.999), weight_decay=0.0)
    _, v = dequantize_moments(cm, cv, sm, sv)
    target = float(g[20]) ** 2
    want = target + (float(start[20]) - target) * 0.999 ** 1000
    assert abs(float(v[8:].mean()) / want - 1) < 0.05


# ------------------------------------------------------------------ device scalars, streams, graphs

def test_device_step_lr_and_grad_scale():
    p, g, m, v = (values([1000], torch.float32, k, 0.1) for k in range(4))
    v = [x.square() for x in v]
    old = [x[0].clone() for x in (p, g, m, v)]
    step = torch.tensor([5], dtype=torch.int64, device=DEV)
    lr = torch.tensor(ARGS["lr"], device=DEV)
    half = torch.tensor([0.5], device=DEV)
    adamw_step(p, g, m, v, step, grad_scale=half, **{**ARGS, "lr": lr})
    check32(*old, 5, (p[0], m[0], v[0]), grad_scale=0.5, lr=float(lr))


@pytest.mark.parametrize("bits", [32, 8])
def test_class_captured_and_replayed(bits):
    """A captured step whose counter lies on the device gives, replayed, the eager steps' bits."""
    def model(seed):
        return [torch.nn.Parameter(x.view(-1, 4)) for x in values([400, 64, 1200], torch.float32, seed)]

    grads = [[x.view(-1, 4) for x in values([400, 64, 1200], torch.float32, 50 + t, 0.1)] for t in range(5)]
    eager, replayed = model(1), model(1)
    a = AdamW(eager, capturable=True, moment_bits=bits, **ARGS)
    b = AdamW(replayed, capturable=True, moment_bits=bits, **ARGS)
    for p in replayed:
        p.grad = torch.zeros_like(p)
    for p, x in zip(replayed, grads[0]):
        p.grad.copy_(x)
    b.step()  # makes the state outside the capture
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.step()
    for t in range(1, 5):
        for p, x in zip(replayed, grads[t]):
            p.grad.copy_(x)
        graph.replay()
    for t in range(5):
        for p, x in zip(eager, grads[t]):
            p.grad = x.clone()
        a.step()
    torch.cuda.synchronize()
    for p, q in zip(eager, replayed):
        assert torch.equal(p, q)
        for k, x in a.state[p].items():
            assert torch.equal(x, b.state[q][k]), k


def test_class_follows_torch():
    """Two groups, a parameter whose gradient comes late, a channels-last weight: against torch's AdamW in
    64 bits, 20 steps.  A step's error is below 20 u of the update and 2 u of the parameter; 20 of them,
    with room for what they do to one another (the gradients do not depend on the parameters): 1000 u of
    a size of order 1."""
    def model(dtype):
        g = torch.Generator(device="cuda").manual_seed(4)
        ps = [torch.randn(s, device=DEV, generator=g).to(dtype) for s in ((33, 7), (5,), (8, 3, 3, 3), (300,))]
        ps[2] = ps[2].to(memory_format=torch.channels_last)
        return [torch.nn.Parameter(p) for p in ps]

    ours, ref = model(torch.float32), model(torch.float64)
    kw = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6)
    groups = lambda ps: [dict(params=ps[:2], weight_decay=0.1), dict(params=ps[2:], lr=3e-3)]  # noqa: E731
    a, b = AdamW(groups(ours), **kw), torch.optim.AdamW(groups(ref), **kw)
    gen = torch.Generator(device="cuda").manual_seed(5)
    for t in range(20):
        for i, (p, q) in enumerate(zip(ours, ref)):
            g = torch.randn(p.shape, device=DEV, generator=gen)
            p.grad, q.grad = (None, None) if i == 3 and t < 4 else (g.clone(), g.double())
        a.step()
        b.step()
    for p, q in zip(ours, ref):
        assert float((p.double() - q).abs().max()) <= 1000 * U * max(1.0, float(q.abs().max()))
    # the state carries over in both directions of precision
    c = AdamW(groups(model(torch.float32)), moment_bits=32, **kw)
    c.load_state_dict(b.state_dict())
    for group, mine in zip(c.param_groups, a.param_groups):
        for p, q in zip(group["params"], mine["params"]):
            assert c.state[p]["step"] == a.state[q]["step"]
            assert torch.allclose(c.state[p]["exp_avg_sq"], a.state[q]["exp_avg_sq"], rtol=1e-4, atol=0)
    flat = [torch.nn.Parameter(p.detach().contiguous().clone()) for p in model(torch.float32)]
    d = AdamW(groups(flat), moment_bits=8, **kw)
    d.load_state_dict(a.state_dict())
    e = AdamW(groups(flat), moment_bits=8, **kw)
    e.load_state_dict(d.state_dict())
    for p, q in zip(flat, ours):
        assert d.state[p]["exp_avg"].dtype == torch.int8 and e.state[p]["exp_avg_sq"].dtype == torch.uint8
        m, v = dequantize_moments(*(e.state[p][k] for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale",
                                                           "exp_avg_sq_scale")))
        top = a.state[q]["exp_avg"].abs().max()
        # nearest code: half a code of 127, |m| = s (c / 127)^2, is off by at most s / 127
        assert float((m - a.state[q]["exp_avg"]).abs().max()) <= float(top) * (1 / 127 + 1e-3)


def test_class_with_8_bits_trains_on():
    """Runs with gradients of a small model, sparse and absent ones refused or skipped."""
    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Linear(16, 32), torch.nn.ReLU(), torch.nn.Linear(32, 4)).to(DEV)
    unused = torch.nn.Parameter(torch.ones(3, device=DEV))
    opt = AdamW([*net.parameters(), unused], lr=1e-3, moment_bits=8)
    for _ in range(3):
        opt.zero_grad()
        net(torch.randn(8, 16, device=DEV)).square().mean().backward()
        opt.step()
    assert all(bool(p.isfinite().all()) for p in net.parameters()) and torch.equal(unused, torch.ones_like(unused))
    assert unused not in opt.state or not opt.state[unused]


def test_no_host_synchronisation():
    p, g, m, v = (values([5000, 77], torch.float32, k, 0.1) for k in range(4))
    v = [x.square() for x in v]
    scale = torch.tensor([0.5], device=DEV)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        adamw_step(p, g, m, v, 1, grad_scale=scale, **ARGS)
    finally:
        torch.cuda.set_sync_debug_mode("default")


def test_gpu_refusals():
    p, g, m, v = (values([64, 32], torch.float32, k, 0.1) for k in range(4))
    with pytest.raises(ValueError, match="twice"):
        adamw_step([p[0], p[0]], [g[0], g[0]], [m[0], m[0]], [v[0], v[0]], 1)
    with pytest.raises(ValueError, match="share memory"):
        adamw_step([p[0]], [g[0]], [p[0]], [v[0]], 1)
    with pytest.raises(ValueError, match="gradients"):
        adamw_step([p[0][:32]], [p[0][16:48]], [m[1]], [v[1]], 1)
    with pytest.raises(ValueError, match="grads"):
        adamw_step(p, [g[0], g[1].half()], m, v, 1)
    with pytest.raises(ValueError, match="exp_avg"):
        adamw_step(p, g, [m[0], m[1][:31]], v, 1)
    with pytest.raises(ValueError, match="exp_avg_sq"):
        adamw_step(p, g, m, [v[0], v[1].view(8, 4).t()], 1)
    with pytest.raises(ValueError, match="grads"):
        adamw_step(p, g[:1], m, v, 1)
    with pytest.raises(ValueError, match="scales"):
        adamw_step(p, g, [x.to(torch.int8) for x in m], [x.to(torch.uint8) for x in v], 1,
                   scales=([sm[:0] for sm in m], [sv[:0] for sv in v]))
    with pytest.raises(ValueError, match="step"):
        adamw_step(p, g, m, v, 0)
    with pytest.raises(ValueError, match="lr"):
        adamw_step(p, g, m, v, 1, lr=torch.ones(1, dtype=torch.float64, device=DEV))
    with pytest.raises(ValueError, match="betas"):
        adamw_step(p, g, m, v, 1, betas=(1.0, 0.9))
    adamw_step([], [], [], [], 1)
    assert optim.moment_scales(257) == 2 and math.isclose(ARGS["lr"], 3e-3)
