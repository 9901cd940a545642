"""linear against the formula in 64 bits.

Tolerances.  Products of two 16-bit values are exact in float32; a sum of K of them, in any order and
with truncating adders, is off by at most K 2^-23 of the sum of magnitudes S.  The bias, the activation
(slope at most 1.13; erff and expf a few units) and the residual add at most 16 * 2^-24 of the magnitudes
there; the store rounds by half a step, eps/2.  dP = dY act'(saved) is rounded to 16 bits (eps/2), and so
was `saved`: gelu'' is at most 0.8, so act' is off by 0.8 eps/2 |pre|; relu's border moves for a value
within its own error of 0, where dP is off by |dY|.  What is off in dP comes into the sums of the
backward products with the magnitudes of the other operand."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

from rfdetr_training_throughput_b200.linear import check_faults, linear
from rfdetr_training_throughput_b200.norm import layer_norm
from rfdetr_training_throughput_b200.optim import AdamW

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
ACTS = ["none", "relu", "gelu"]
TYPES = [torch.bfloat16, torch.float16]


def make(rows, inner, outer, dtype, residual=True, seed=0, bias_dtype=None):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device=DEV, generator=g) * scale

    return dict(x=normal(rows, inner).to(dtype), weight=normal(outer, inner, scale=inner ** -0.5).to(dtype),
                bias=normal(outer, scale=0.2).to(bias_dtype or dtype),
                residual=normal(rows, outer).to(dtype) if residual else None, dy=normal(rows, outer).to(dtype))


def act64(v, act):
    return v.clamp_min(0) if act == "relu" else v * torch.special.ndtr(v) if act == "gelu" else v


def grad64(v, act):
    if act == "relu":
        return (v > 0).double()
    if act == "gelu":
        return torch.special.ndtr(v) + v * torch.exp(-v * v / 2) / (2 * torch.pi) ** 0.5
    return torch.ones_like(v)


def reference(d, act, dtype):
    """Values in 64 bits and the bounds of the text above, per element."""
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x, w, b, dy = (d[k].double() for k in ("x", "weight", "bias", "dy"))
    r = None if d["residual"] is None else d["residual"].double()
    rows, (outer, inner) = x.shape[0], w.shape
    size = x.abs() @ w.abs().t()
    pre = x @ w.t() + b
    pre_off = inner * 2 * U * size + 4 * U * (size + b.abs())
    out = act64(pre, act)
    off = 1.13 * pre_off + 16 * U * (pre.abs() + (0 if r is None else r.abs()))
    if r is not None:
        out = out + r
    ref = dict(out=(out, off + half * (out.abs() + off) + tiny))
    slope = grad64(pre, act)
    dp = dy * slope
    slope_off = {"none": torch.zeros_like(pre), "relu": (pre.abs() <= pre_off + tiny).double(),
                 "gelu": 0.8 * (half * pre.abs() + pre_off) + 16 * U + tiny}[act]
    dp_sum_off = dy.abs() * slope_off + 4 * U * dp.abs()
    dp_off = dp_sum_off + half * (dp.abs() + dp_sum_off) + tiny if act != "none" else torch.zeros_like(dp)

    def product(a, a_off, c, depth):
        want, mags = a @ c, a.abs() @ c.abs()
        off = a_off @ c.abs() + depth * 2 * U * (mags + a_off @ c.abs())
        return want, off + half * (want.abs() + off) + tiny

    ref["x"] = product(dp, dp_off, w, outer)
    ref["weight"] = product(dp.t(), dp_off.t(), x, rows)
    bias_half = torch.finfo(d["bias"].dtype).eps / 2
    want, off = dp.sum(0), dp_sum_off.sum(0) + rows * U * dp.abs().sum(0)
    ref["bias"] = (want, off + bias_half * (want.abs() + off) + tiny)
    ref["residual"] = (dy, torch.zeros_like(dy))
    return ref


def close(name, got, ref):
    want, bound = ref
    assert got.shape == want.shape, name
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{name} off by {float((off / bound).max()):.2f} bounds"


def check(d, act, dtype, **views):
    names = [k for k in ("x", "weight", "bias", "residual") if d[k] is not None]
    leaves = {k: d[k].clone().requires_grad_(True) for k in names}
    out = linear(leaves["x"], leaves["weight"], leaves["bias"], activation=act, residual=leaves.get("residual"))
    assert out.dtype == dtype and out.is_contiguous()
    grads = dict(zip(names, torch.autograd.grad(out, list(leaves.values()), d["dy"])))
    with torch.no_grad():
        again = linear(d["x"], d["weight"], d["bias"], activation=act, residual=d["residual"])
    ref = reference(d, act, dtype)
    close("out", out.detach(), ref["out"])
    assert torch.equal(again, out)
    for k in names:
        assert grads[k].dtype == d[k].dtype
        close(f"grad {k}", grads[k], ref[k])


# one row, one column, one feature; the borders of a tile (128 rows, 64 deep, 64 to 256 columns) and of a
# 32 x 32 box; odd sizes (padded operands, element stores); deep and shallow products (splits)
SIZES = [(1, 1, 1), (1, 64, 64), (1, 4096, 300), (3, 8, 8), (5, 7, 9), (31, 63, 33), (32, 64, 32), (33, 65, 31),
         (127, 128, 91), (128, 64, 128), (129, 72, 136), (300, 256, 91), (300, 256, 4), (257, 40, 264), (64, 1000, 520),
         (1000, 8, 2048), (2049, 256, 256), (4100, 96, 200), (10, 2048, 2000)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,inner,outer", SIZES)
def test_matches_the_formula(rows, inner, outer, act, dtype):
    d = make(rows, inner, outer, dtype, residual=(rows + outer) % 2 == 0, seed=rows + inner)
    check(d, act, dtype)


@pytest.mark.parametrize("rows,inner,outer,act,residual,dtype",
                         [(31200, 256, 2048, "relu", False, torch.bfloat16),
                          (31200, 2048, 256, "none", True, torch.bfloat16),
                          (13608, 384, 1536, "gelu", False, torch.float16),
                          (2000, 2000, 2008, "gelu", True, torch.bfloat16),
                          (20000, 128, 64, "relu", True, torch.float16)])
def test_training_sizes(rows, inner, outer, act, residual, dtype):
    check(make(rows, inner, outer, dtype, residual=residual, seed=1, bias_dtype=torch.float32), act, dtype)
    check_faults()


def test_layouts():
    """Rows apart, bases off 16 bytes, more dimensions, columns apart, one row in many places."""
    dtype = torch.bfloat16
    d = make(24, 40, 56, dtype, seed=2)
    ref = reference(d, "relu", dtype)

    def place(t, pad, first):
        wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), device=DEV, dtype=dtype)
        wide[:, first:first + t.shape[1]] = t
        return wide[:, first:first + t.shape[1]]

    for pad, first in ((8, 0), (8, 8), (3, 1), (16, 3)):
        out = linear(place(d["x"], pad, first), place(d["weight"], pad, first), d["bias"], activation="relu",
                     residual=place(d["residual"], pad, first))
        close("out", out, ref["out"])
    out = linear(d["x"].view(2, 3, 4, 40), d["weight"].t().contiguous().t(), d["bias"][None].expand(3, 56)[1],
                 activation="relu", residual=d["residual"].view(2, 3, 4, 56))
    assert out.shape == (2, 3, 4, 56)
    close("out", out.view(24, 56), ref["out"])
    swapped = d["x"].view(4, 6, 40).transpose(0, 1).contiguous().transpose(0, 1)
    close("out", linear(swapped, d["weight"], d["bias"], activation="relu",
                        residual=d["residual"].view(4, 6, 56)).reshape(24, 56), ref["out"])
    # one row expanded, as x, as the residual and as the gradient
    e = {**d, "x": d["x"][:1].expand(24, 40), "residual": d["residual"][:1].expand(24, 56),
         "dy": d["dy"][:1].expand(24, 56)}
    row, res = d["x"][:1].clone().requires_grad_(True), d["residual"][:1].clone().requires_grad_(True)
    w = d["weight"].clone().requires_grad_(True)
    out = linear(row.expand(24, 40), w, d["bias"], residual=res.expand(24, 56))
    g = torch.autograd.grad(out, [w, row, res], e["dy"])
    far = reference(e, "none", dtype)
    close("out", out.detach(), far["out"])
    close("grad weight", g[0], far["weight"])
    # autograd adds the 24 rows' gradients in 16 bits (or more): each addition rounds by eps/2
    eps = torch.finfo(dtype).eps
    close("grad row", g[1], (far["x"][0].sum(0, keepdim=True),
                             far["x"][1].sum(0, keepdim=True) + 24 * eps * far["x"][0].abs().sum(0, keepdim=True)))
    close("grad residual", g[2], (24 * e["dy"][:1].double(), 24 * 24 * eps * e["dy"][:1].double().abs()))
    # a gradient with columns apart, no activation: dP cannot be read where it lies
    leaf = d["x"].clone().requires_grad_(True)
    none = reference(d, "none", dtype)
    (gx,) = torch.autograd.grad(linear(leaf, d["weight"], d["bias"], residual=d["residual"]), leaf,
                                d["dy"].t().contiguous().t())
    close("grad x", gx, none["x"])


def test_missing_parts():
    dtype = torch.float16
    d = make(70, 48, 40, dtype, residual=False, seed=3)
    zero = {**d, "bias": torch.zeros_like(d["bias"])}
    ref = reference(zero, "gelu", dtype)
    x, w = d["x"].clone().requires_grad_(True), d["weight"].clone().requires_grad_(True)
    out = linear(x, w, activation="gelu")
    close("out", out.detach(), ref["out"])
    (gw,) = torch.autograd.grad(out, [w], d["dy"], retain_graph=True)
    (gx,) = torch.autograd.grad(out, [x], d["dy"])
    close("grad weight", gw, ref["weight"])
    close("grad x", gx, ref["x"])
    bias = d["bias"].clone().requires_grad_(True)
    (gb,) = torch.autograd.grad(linear(d["x"], d["weight"], bias), [bias], d["dy"])
    close("grad bias", gb, reference(d, "none", dtype)["bias"])
    empty = torch.zeros((0, 48), device=DEV, dtype=dtype, requires_grad=True)
    out = linear(empty, w, bias, activation="relu", residual=torch.zeros((0, 40), device=DEV, dtype=dtype))
    gx, gw, gb = torch.autograd.grad(out, [empty, w, bias], torch.zeros((0, 40), device=DEV, dtype=dtype))
    assert out.shape == (0, 40) and gx.shape == (0, 48) and not gw.any() and not gb.any()


def test_a_vector_and_one_tensor_twice():
    d = make(1, 72, 40, torch.bfloat16, residual=False, seed=21)
    out = linear(d["x"][0], d["weight"], d["bias"], activation="gelu")
    assert out.shape == (40,)
    close("out", out[None], reference(d, "gelu", torch.bfloat16)["out"])
    w = make(48, 48, 48, torch.bfloat16, residual=False, seed=22)
    both = w["weight"].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(linear(both, both), [both], w["dy"])
    ref = reference({**w, "x": w["weight"], "bias": torch.zeros_like(w["bias"])}, "none", torch.bfloat16)
    want, bound = (a + b for a, b in zip(ref["x"], ref["weight"]))
    # autograd adds the two gradients in 16 bits
    close("grad", g, (want, bound + torch.finfo(torch.bfloat16).eps * (want.abs() + bound)))


def test_products_beyond_the_type_s_range():
    """fp16 values beyond 65504 before the activation: the output follows the rounding (infinite, or 0 on
    gelu's other side), and the gradient is that of a far value, 1 or 0."""
    x = torch.full((130, 64), 200.0, device=DEV, dtype=torch.float16, requires_grad=True)
    w = torch.full((64, 64), 20.0, device=DEV, dtype=torch.float16)
    w[1::2] *= -1
    for rows in (1, 130):
        part = x[:rows]
        out = linear(part, w, activation="gelu")
        assert bool((out[:, ::2] == float("inf")).all()) and not out[:, 1::2].any()
        (g,) = torch.autograd.grad(out, x, torch.full_like(out, 1 / 64))
        # dP = dy on the even columns: 32 of them times 20 / 64
        assert torch.equal(g[:rows], torch.full_like(g[:rows], 10.0))


def test_offsets_beyond_32_bits():
    """An output of 2.2e9 elements: the last rows and the first, forward and backward."""
    rows, inner, outer = 1_073_000, 16, 2056
    g = torch.Generator(device="cuda").manual_seed(23)
    x = torch.randn(rows, inner, device=DEV, generator=g).to(torch.bfloat16).requires_grad_(True)
    w = torch.randn(outer, inner, device=DEV, generator=g).to(torch.bfloat16)
    b = torch.randn(outer, device=DEV, generator=g).to(torch.bfloat16)
    out = linear(x, w, b, activation="relu")
    assert out.numel() > 2 ** 31
    dy = torch.zeros_like(out)
    ends = torch.cat([torch.arange(300), torch.arange(rows - 300, rows)]).to(DEV)
    d = dict(x=x.detach()[ends], weight=w, bias=b, residual=None,
             dy=torch.randn(600, outer, device=DEV, generator=g).to(torch.bfloat16))
    dy[ends] = d["dy"]
    gx, = torch.autograd.grad(out, [x], dy)
    ref = reference(d, "relu", torch.bfloat16)
    close("out", out.detach()[ends], ref["out"])
    close("grad x", gx[ends], ref["x"])
    assert not gx[300:-300].any()
    check_faults()


def test_a_changed_output_is_noticed():
    d = make(8, 16, 16, torch.bfloat16, residual=False, seed=24)
    x = d["x"].clone().requires_grad_(True)
    out = linear(x, d["weight"], activation="relu")
    out.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_special_values_stay_in_their_rows():
    d = make(200, 72, 136, torch.bfloat16, residual=False, seed=4)
    clean = linear(d["x"], d["weight"], d["bias"], activation="relu")
    x = d["x"].clone()
    x[3, 5], x[150, 0] = float("nan"), float("inf")
    out = linear(x, d["weight"], d["bias"], activation="relu")
    assert bool(out[3].isnan().all())
    bad = out[150]  # +-inf by the weight's sign; relu keeps +inf and cuts -inf
    assert bool(((bad == float("inf")) | (bad == 0)).all())
    keep = torch.ones(200, dtype=torch.bool, device=DEV)
    keep[[3, 150]] = False
    assert torch.equal(out[keep], clean[keep])


def test_gradients_against_differences():
    """Central differences of the 64-bit formula along a direction, h = 2^-12 (their error is of order h^2);
    the gradient itself is 16 bits: within 2 % of the sum of magnitudes."""
    d = make(6, 24, 16, torch.bfloat16, seed=5)
    for act in ("none", "gelu"):
        leaves = {k: d[k].clone().requires_grad_(True) for k in ("x", "weight", "bias", "residual")}
        out = linear(leaves["x"], leaves["weight"], leaves["bias"], activation=act, residual=leaves["residual"])
        out.backward(d["dy"])
        for k, leaf in leaves.items():
            direction = torch.randn(leaf.shape, device=DEV, generator=torch.Generator(device="cuda").manual_seed(6))

            def loss(sign):
                t = {n: d[n].double() + (sign * 2.0 ** -12 * direction if n == k else 0) for n in leaves}
                return float(((act64(t["x"] @ t["weight"].t() + t["bias"], act) + t["residual"])
                              * d["dy"].double()).sum())

            got = leaf.grad.double() * direction
            assert abs(float(got.sum()) - (loss(1) - loss(-1)) * 2.0 ** 11) <= 0.02 * float(got.abs().sum())


def test_second_derivative_and_changed_operands_raise():
    d = make(16, 16, 16, torch.bfloat16, seed=7)
    x = d["x"].clone().requires_grad_(True)
    (g,) = torch.autograd.grad(linear(x, d["weight"], activation="gelu"), x, d["dy"], create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()
    w = d["weight"].clone().requires_grad_(True)
    out = linear(x.view(2, 8, 16), w)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    out = layer_norm((x * 1.0).view(2, 8, 16))
    (g,) = torch.autograd.grad(out, x, torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        g.sum().backward()


def test_autocast_takes_its_type():
    d = make(40, 32, 24, torch.bfloat16, seed=8)
    full = {k: d[k].float() for k in ("x", "weight", "bias", "residual")}
    w = full["weight"].requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        out = linear(full["x"], w, full["bias"], activation="relu", residual=full["residual"])
    assert out.dtype == torch.bfloat16
    close("out", out.detach(), reference(d, "relu", torch.bfloat16)["out"])
    out.backward(d["dy"])
    assert w.grad.dtype == torch.float32
    close("grad weight", w.grad, reference(d, "relu", torch.bfloat16)["weight"])


def test_same_bits_on_streams_and_at_once():
    """Two calls at once on two streams, each with its own workspace, give what each gives alone."""
    sets = [make(4000, 256, 256, torch.bfloat16, seed=10 + i) for i in range(2)]

    def both(d):
        leaves = [d[k].clone().requires_grad_(True) for k in ("x", "weight", "bias")]
        out = linear(*leaves, activation="gelu", residual=d["residual"])
        return [out.detach(), *torch.autograd.grad(out, leaves, d["dy"])]

    alone = [both(d) for d in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(3):
        for s, d in zip(streams, sets):
            with torch.cuda.stream(s):
                got.append(both(d))
    torch.cuda.synchronize()
    for i, one in enumerate(got):
        for a, b in zip(one, alone[i % 2]):
            assert torch.equal(a, b)


def test_captured_and_replayed():
    d = make(700, 256, 128, torch.bfloat16, seed=12)
    leaves = [d[k].clone().requires_grad_(True) for k in ("x", "weight", "bias", "residual")]

    def both():
        out = linear(leaves[0], leaves[1], leaves[2], activation="relu", residual=leaves[3])
        return [out.detach(), *torch.autograd.grad(out, leaves, d["dy"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs, replayed one after the other: neither uses the other's workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = both()
        graphs.append((graph, captured))
    with torch.no_grad():
        leaves[0].copy_(make(700, 256, 128, torch.bfloat16, seed=13)["x"])
    for graph, _ in graphs:
        graph.replay()
    torch.cuda.synchronize()
    want = both()
    for _, captured in graphs:
        for a, b in zip(captured, want):
            assert torch.equal(a, b)


def test_refusals():
    d = make(16, 16, 8, torch.bfloat16, seed=14)
    x, w, b, r = (d[k] for k in ("x", "weight", "bias", "residual"))
    for bad in (lambda: linear(x.float(), w), lambda: linear(x, w.half()), lambda: linear(x.float(), w.float()),
                lambda: linear(x[:, :8], w), lambda: linear(x, w[0]), lambda: linear(x, w, b[:7]),
                lambda: linear(x, w, b.double()), lambda: linear(x, w, residual=r[:1]),
                lambda: linear(x, w, residual=r.float()), lambda: linear(x, w, activation="silu"),
                lambda: linear(x, w.cpu()), lambda: linear(x[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            bad()


def test_a_feed_forward_block_trains():
    """linear(relu) -> linear(+ residual) -> layer_norm -> loss, its gradients against autograd in 64 bits
    on the same bf16 weights, then a step of AdamW on all of them.  Each bf16 tensor on the way is off by
    2^-9 of its size (two products, a norm, and the same back): 2 % of a gradient's norm is above their sum."""
    torch.manual_seed(0)
    d, f, rows = 256, 512, 600
    shapes = dict(w1=(f, d), b1=(f,), w2=(d, f), b2=(d,), g=(d,), h=(d,))
    start = {k: torch.randn(s, device=DEV) * (s[-1] ** -0.5 if len(s) == 2 else 0.1) for k, s in shapes.items()}
    start["g"] = start["g"] + 1
    ps = {k: torch.nn.Parameter(v.to(torch.bfloat16)) for k, v in start.items()}
    x = torch.randn(2, rows // 2, d, device=DEV, dtype=torch.bfloat16)
    seed = torch.randn_like(x)

    def run(p, x, mm, norm):
        hidden = mm(x, p["w1"], p["b1"], "relu", None)
        return norm(mm(hidden, p["w2"], p["b2"], "none", x), p["g"], p["h"])

    out = run(ps, x, lambda a, w, b, act, r: linear(a, w, b, activation=act, residual=r), layer_norm)
    (out * seed).float().sum().backward()
    wide = {k: p.detach().double().requires_grad_(True) for k, p in ps.items()}

    def mm64(a, w, b, act, r):
        v = act64(a @ w.t() + b, act)
        return v if r is None else v + r

    ref = run(wide, x.double(), mm64, lambda v, g, h: torch.nn.functional.layer_norm(v, (d,), g, h))
    (ref * seed.double()).sum().backward()
    assert float((out.double() - ref).norm() / ref.norm()) < 0.02
    for k, p in ps.items():
        assert float((p.grad.double() - wide[k].grad).norm() / wide[k].grad.norm()) < 0.02, k
    before = {k: p.detach().clone() for k, p in ps.items()}
    for bits in (32, 8):
        AdamW(ps.values(), lr=1e-2, moment_bits=bits).step()
    for k, p in ps.items():
        assert bool(p.isfinite().all()) and not torch.equal(p, before[k])
    check_faults()


def test_relu_cuts_infinite_gradients():
    """Where relu cut, an infinite or undefined incoming gradient does not come through; where it kept a NaN
    the gradient passes, as torch's relu has it.  Rows of the identity's product, so that each element of
    dX is one of dP."""
    bad = [float("inf"), -float("inf"), float("nan"), 1.0]
    for outer, residual in ((64, False), (64, True), (51, False)):
        x = torch.zeros(8, outer, device=DEV, dtype=torch.bfloat16)
        x[:4] = -1
        x[4:] = 1
        x[7] = float("nan")
        bias = torch.zeros(outer, device=DEV, dtype=torch.bfloat16, requires_grad=True)
        leaf = x.clone().requires_grad_(True)
        res = torch.ones_like(x) if residual else None
        out = linear(leaf, torch.eye(outer, device=DEV, dtype=torch.bfloat16), bias, activation="relu", residual=res)
        dy = torch.ones_like(x)
        dy[:4, 0] = torch.tensor(bad, device=DEV, dtype=torch.bfloat16)
        out.backward(dy)
        want = torch.zeros_like(x)
        want[4:] = 1
        assert torch.equal(leaf.grad, want)
        assert torch.equal(bias.grad, torch.full_like(bias, 4.0))


# enough rows that dP and dX come from one kernel: columns of dX around 128, 256 and 384, slices of dP that
# end inside 64 columns, more slices than stages, CTAs with one, two and three tiles, a last tile of one row
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ["relu", "gelu"])
@pytest.mark.parametrize("rows,inner,outer", [(9473, 8, 8), (9600, 128, 72), (9729, 136, 1000), (18944, 256, 64),
                                              (19073, 264, 520), (20001, 384, 2048), (38017, 40, 200),
                                              (10000, 256, 4096), (10000, 384, 2056), (10000, 392, 96)])
def test_gradients_of_many_rows(rows, inner, outer, act, dtype):
    check(make(rows, inner, outer, dtype, residual=outer == 72, seed=31 + inner), act, dtype)
    check_faults()


def test_gradients_of_many_rows_in_parts():
    """dX alone, without a bias, from gradients whose rows lie apart; the same bits alone, together with the
    others, and on another stream at once."""
    dtype = torch.bfloat16
    rows, inner, outer = 12345, 256, 328
    d = make(rows, inner, outer, dtype, residual=False, seed=33)
    ref = reference(d, "gelu", dtype)
    wide = torch.full((rows, outer + 24), float("nan"), device=DEV, dtype=dtype)
    wide[:, 8:8 + outer] = d["dy"]
    leaves = [d[k].clone().requires_grad_(True) for k in ("x", "weight", "bias")]
    out = linear(*leaves, activation="gelu")
    whole = torch.autograd.grad(out, leaves, d["dy"], retain_graph=True)
    apart = torch.autograd.grad(out, leaves, wide[:, 8:8 + outer], retain_graph=True)
    (alone,) = torch.autograd.grad(out, leaves[:1], d["dy"], retain_graph=True)
    for name, a, b in zip(("x", "weight", "bias"), whole, apart):
        close(f"grad {name}", a, ref[name])
        assert torch.equal(a, b)
    assert torch.equal(alone, whole[0])
    x = d["x"].clone().requires_grad_(True)
    (frozen,) = torch.autograd.grad(linear(x, d["weight"], d["bias"], activation="gelu"), x, d["dy"])
    assert torch.equal(frozen, whole[0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for stream in streams:
        with torch.cuda.stream(stream):
            mine = [t.detach().clone().requires_grad_(True) for t in leaves]
            results.append(torch.autograd.grad(linear(*mine, activation="gelu"), mine, d["dy"]))
    torch.cuda.synchronize()
    for grads in results:
        for a, b in zip(grads, whole):
            assert torch.equal(a, b)
    check_faults()


def test_gradients_of_many_rows_with_special_values():
    """A NaN and infinities in the gradient stay in their rows of dX; the rows behind the last one are not
    read as values."""
    dtype = torch.float16
    d = make(9501, 256, 136, dtype, residual=False, seed=34)
    x = d["x"].clone().requires_grad_(True)
    out = linear(x, d["weight"], d["bias"], activation="relu")
    (clean,) = torch.autograd.grad(out, x, d["dy"], retain_graph=True)
    dy = d["dy"].clone()
    live, cut = (out[9500] > 0).nonzero()[0, 0], (out[9500] == 0).nonzero()[0, 0]
    dy[9500, live] = float("nan")
    dy[77, (out[77] == 0).nonzero()[0, 0]] = float("inf")
    dy[9500, cut] = float("inf")
    (g,) = torch.autograd.grad(out, x, dy)
    assert bool(g[9500].isnan().all())
    assert bool(g[77].isfinite().all())
    keep = torch.ones(9501, dtype=torch.bool, device=DEV)
    keep[[77, 9500]] = False
    assert torch.equal(g[keep], clean[keep])


@pytest.mark.parametrize("act,rows", [("none", 40), ("relu", 10000)])
def test_first_backward_of_a_process(act, rows):
    """Autograd's thread has made no CUDA call when the first backward of a process reaches the product."""
    code = ("import torch; from rfdetr_training_throughput_b200.linear import linear\n"
            f"x = torch.ones({rows}, 64, device='cuda', dtype=torch.bfloat16, requires_grad=True)\n"
            "w = torch.ones(32, 64, device='cuda', dtype=torch.bfloat16)\n"
            f"out = linear(x, w, activation='{act}')\n"
            "(g,) = torch.autograd.grad(out, x, torch.ones_like(out))\n"
            "assert bool((g == 32).all())\n")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=Path(__file__).resolve().parents[1])


def test_many_rows_captured_and_replayed():
    """The backward that takes dP and dX from one kernel, captured behind the kernel that makes its input."""
    d = make(10017, 256, 264, torch.bfloat16, residual=False, seed=35)
    leaves = [d[k].clone().requires_grad_(True) for k in ("x", "weight", "bias")]

    def both():
        out = linear(*leaves, activation="gelu")
        return [out.detach(), *torch.autograd.grad(out, leaves, d["dy"].neg())]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    with torch.no_grad():
        leaves[0].copy_(make(10017, 256, 264, torch.bfloat16, seed=36)["x"])
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(captured, both()):
        assert torch.equal(a, b)
    check_faults()


def test_copied_operands_serve_the_backward():
    """Operands that TMA cannot read are copied once, and a change of the originals is still noticed; a frozen
    weight's or input's gradient needs neither."""
    dtype = torch.bfloat16
    d = make(37, 45, 51, dtype, residual=False, seed=37)
    ref = reference(d, "gelu", dtype)
    wide = torch.zeros(45, 37, device=DEV, dtype=dtype)
    wide.copy_(d["x"].t())
    x = wide.t().requires_grad_(True)  # columns apart
    w = d["weight"].clone().requires_grad_(True)
    out = linear(x, w, d["bias"], activation="gelu")
    gx, gw = torch.autograd.grad(out, [x, w], d["dy"], retain_graph=True)
    close("grad x", gx, ref["x"])
    close("grad weight", gw, ref["weight"])
    again = torch.autograd.grad(out, [x, w], d["dy"], retain_graph=True)
    assert torch.equal(again[0], gx) and torch.equal(again[1], gw)
    (only_w,) = torch.autograd.grad(linear(x.detach(), w, d["bias"], activation="gelu"), w, d["dy"])
    (only_x,) = torch.autograd.grad(linear(x, w.detach(), d["bias"], activation="gelu"), x, d["dy"])
    assert torch.equal(only_w, gw) and torch.equal(only_x, gx)
    with torch.no_grad():
        w.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


@pytest.mark.parametrize("sizes", [(37, 45, 51), (64, 64, 64)])
def test_saved_tensor_hooks(sizes):
    """What the backward needs may be packed and come back elsewhere with other strides."""
    d = make(*sizes, torch.bfloat16, residual=False, seed=38)
    norm = torch.ones(sizes[2], device=DEV, dtype=torch.bfloat16)

    def grads():
        leaves = [d[k].clone().requires_grad_(True) for k in ("x", "weight", "bias")]
        out = layer_norm(linear(*leaves, activation="gelu"), norm)
        return torch.autograd.grad(out, leaves, d["dy"])

    def turned(t):
        return t.t().contiguous().t() if t.dim() == 2 else t.clone()

    want = grads()
    with torch.autograd.graph.save_on_cpu():
        off = grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, turned):
        other = grads()
    for a, b, c in zip(want, off, other):
        assert torch.equal(a, b) and torch.equal(a, c)
