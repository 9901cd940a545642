"""layer_norm against the formula in 64 bits.

Tolerances (u = 2^-24, a rounding of float32): a row sum passes at most 16 additions in a thread, 5 in
a warp and 16 over warps (wide rows: dim / 256 + 13), so a mean is off by at most K u mean|x| with
K = 40 + dim / 256, a deviation by (K + 1) u (|x| + mean|x|) and rstd by about 2 K u of itself.  With
A = mean|x| rstd and |unit| the output's error is below 4 K u (|w| (|unit| + A) + |b|), plus half a step
of the output's type.  A gradient of x has the same roundings on three terms; the sums over the rows add
one rounding a row (bounded by rows + 64)."""

import pytest
import torch

from rfdetr_training_throughput_b200.norm import layer_norm

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def step(dtype):
    return torch.finfo(dtype).eps / 2


def make(rows, dim, dtype, seed=0, shift=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, dim, device=DEV, generator=g) * 2 + torch.randn(rows, 1, device=DEV, generator=g) * shift
    w = 1 + 0.3 * torch.randn(dim, device=DEV, generator=g)
    b = 0.3 * torch.randn(dim, device=DEV, generator=g)
    dy = torch.randn(rows, dim, device=DEV, generator=g)
    return x.to(dtype), w, b, dy.to(dtype)


def reference(x, w, b, dy, eps):
    """Outputs in 64 bits and the magnitudes their bounds are made of."""
    x, w, b, dy = (t.double() for t in (x, w, b, dy))
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    unit = (x - mean) * rstd
    reach = unit.abs() + x.abs().mean(1, keepdim=True) * rstd  # |unit| + A
    t = dy * w
    m1, m2 = t.mean(1, keepdim=True), (t * unit).mean(1, keepdim=True)
    size = rstd * (t.abs() + t.abs().mean(1, keepdim=True) + reach * (t.abs() * reach).mean(1, keepdim=True))
    return dict(out=unit * w + b, dx=rstd * (t - m1 - unit * m2), dw=(dy * unit).sum(0), db=dy.sum(0),
                out_size=w.abs() * reach + b.abs(), dx_size=size, dw_size=(dy.abs() * reach).sum(0),
                db_size=dy.abs().sum(0))


def close(got, want, size, factor, dtype):
    """|got - want| within `factor` roundings of `size` and half a step of the type (fp16 subnormals: of
    its smallest step)."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = factor * U * size + step(dtype) * (want.abs() + factor * U * size) + tiny
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"off by {float((off / bound).max()):.2f} bounds"


# one element; short rows (teams of 8); the borders of each team's columns; odd sizes (element loads);
# rows longer than the registers hold
DIMS = [1, 2, 7, 8, 31, 32, 33, 64, 65, 128, 129, 256, 257, 384, 393, 512, 520, 1000, 1024, 1025, 2048, 2050, 2056,
        4096, 4100, 8192, 8191, 8193, 9000]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("dim", DIMS)
def test_matches_the_formula(dim, dtype):
    for rows in (1, 5, 300):
        x, w, b, dy = make(rows, dim, dtype, seed=dim * 7 + rows)
        eps = 1e-5
        w, b = w.to(dtype), b.to(dtype)
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        out = layer_norm(*leaves, eps)
        assert out.dtype == dtype and out.shape == x.shape
        out.backward(dy)
        ref = reference(x, w, b, dy, eps)
        k = 4 * (40 + dim / 256)
        close(out, ref["out"], ref["out_size"], k, dtype)
        # with one column, or rows that hardly vary, rstd is large: the bounds grow with it
        close(leaves[0].grad, ref["dx"], ref["dx_size"], 3 * k, dtype)
        close(leaves[1].grad, ref["dw"], ref["dw_size"], k + rows + 64, dtype)
        close(leaves[2].grad, ref["db"], ref["db_size"], rows + 64, dtype)


@pytest.mark.parametrize("rows,dim,dtype", [(31200, 256, torch.bfloat16), (5003, 1024, torch.float16),
                                            (70001, 40, torch.float32), (1201, 4096, torch.float32),
                                            (257, 10007, torch.bfloat16)])
def test_many_rows(rows, dim, dtype):
    x, w, b, dy = make(rows, dim, dtype, seed=1)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]  # float32 weights beside 16-bit rows
    out = layer_norm(*leaves)
    out.backward(dy)
    ref = reference(x, w, b, dy, 1e-5)
    k = 4 * (40 + dim / 256)
    close(out, ref["out"], ref["out_size"], k, dtype)
    close(leaves[0].grad, ref["dx"], ref["dx_size"], 3 * k, dtype)
    close(leaves[1].grad, ref["dw"], ref["dw_size"], k + rows + 64, torch.float32)
    close(leaves[2].grad, ref["db"], ref["db_size"], rows + 64, torch.float32)


def test_gradients_against_differences():
    """d(sum dy out) along a direction, by central differences of the 64-bit formula at h = 2^-12: their
    error is of the order h^2 = 6e-8 of the third derivative (order 1 here), the gradient's own that of
    float32; 1e-4 of the sum of magnitudes is above both."""
    x, w, b, dy = make(6, 48, torch.float32, seed=3)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    layer_norm(*leaves).backward(dy)
    h = 2.0 ** -12
    for leaf, base in zip(leaves, (x, w, b)):
        d = torch.randn(base.shape, device=DEV, generator=torch.Generator(device="cuda").manual_seed(9)).double()

        def loss(sign):
            moved = [t.double() + (sign * h * d if t is base else 0) for t in (x, w, b)]
            return (reference(*moved, dy, 1e-5)["out"] * dy.double()).sum()

        want = float((loss(1) - loss(-1)) / (2 * h))
        got = float((leaf.grad.double() * d).sum())
        assert abs(got - want) <= 1e-4 * float((leaf.grad.double() * d).abs().sum())


def test_layouts_and_missing_parameters():
    x, w, b, dy = make(24, 40, torch.float32, seed=5)
    ref = reference(x, w, b, dy, 1e-5)
    want = ref["out"]
    wide = torch.full((24, 57), float("nan"), device=DEV)
    wide[:, 3:43] = x
    for view in (wide[:, 3:43],                                       # rows apart, base off 16 bytes
                 x.t().contiguous().t(),                              # columns apart
                 x.view(2, 3, 4, 40),                                 # more dimensions
                 x.view(4, 6, 40).transpose(0, 1).contiguous().transpose(0, 1)):
        got = layer_norm(view, w, b).reshape(24, 40)
        close(got, want, ref["out_size"], 200, torch.float32)
    # a row in many places (stride 0), and its gradient summed over them
    one = x[:1].clone().requires_grad_(True)
    out = layer_norm(one.expand(24, 40), w, b)
    out.backward(dy)
    same = reference(x[:1].expand(24, 40), w, b, dy, 1e-5)
    close(out, same["out"], same["out_size"], 200, torch.float32)
    close(one.grad[0], same["dx"].sum(0), same["dx_size"].sum(0), 600 + 24, torch.float32)
    # gradients that are not contiguous: expanded, and columns apart
    leaf = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(layer_norm(leaf, w, b), leaf, dy[:, :1].expand(24, 40))
    spread = reference(x, w, b, dy[:, :1].expand(24, 40), 1e-5)
    close(g, spread["dx"], spread["dx_size"], 600, torch.float32)
    (g,) = torch.autograd.grad(layer_norm(leaf, w, b), leaf, dy.t().contiguous().t())
    close(g, ref["dx"], ref["dx_size"], 600, torch.float32)
    # no weight, no bias, neither; only some gradients wanted
    ones, zeros = torch.ones(40, device=DEV), torch.zeros(40, device=DEV)
    for ww, bb in ((None, b), (w, None), (None, None)):
        part = reference(x, ones if ww is None else ww, zeros if bb is None else bb, dy, 1e-5)
        leaf = x.clone().requires_grad_(True)
        out = layer_norm(leaf, ww, bb)
        out.backward(dy)
        close(out, part["out"], part["out_size"], 200, torch.float32)
        close(leaf.grad, part["dx"], part["dx_size"], 600, torch.float32)
    bias = b.clone().requires_grad_(True)
    layer_norm(x, w, bias).backward(dy)
    close(bias.grad, ref["db"], ref["db_size"], 24 + 64, torch.float32)


@pytest.mark.parametrize("rows,dim", [(2_100_000, 1032), (262_200, 8200)])
def test_offsets_beyond_32_bits(rows, dim):
    """2.2e9 elements, rows in registers and re-read: the last rows, forward and backward."""
    x = torch.zeros(rows, dim, device=DEV, dtype=torch.bfloat16)
    tail, w, b, dy_tail = make(40, dim, torch.bfloat16, seed=31)
    assert x.numel() > 2 ** 31
    x[-40:] = tail
    x.requires_grad_(True)
    out = layer_norm(x, w, b)
    dy = torch.zeros_like(out)
    dy[-40:] = dy_tail
    (g,) = torch.autograd.grad(out, [x], dy)
    ref = reference(tail, w, b, dy_tail, 1e-5)
    k = 4 * (40 + dim / 256)
    close(out[-40:].detach(), ref["out"], ref["out_size"], k, torch.bfloat16)
    close(g[-40:], ref["dx"], ref["dx_size"], 3 * k, torch.bfloat16)
    assert not g[:-40].any()


def test_empty_rows_and_special_values():
    w = torch.ones(16, device=DEV, requires_grad=True)
    x = torch.zeros((0, 16), device=DEV, requires_grad=True)
    out = layer_norm(x, w)
    out.sum().backward()
    assert out.shape == (0, 16) and x.grad.shape == (0, 16) and not w.grad.any()
    x, w, b, _ = make(9, 264, torch.float32, seed=6)
    clean = layer_norm(x, w, b)
    x[2, 5], x[4, 0], x[6] = float("nan"), float("inf"), 7.0
    got = layer_norm(x, w, b)
    assert got[2].isnan().all() and got[4].isnan().all()  # as inf - inf makes every deviation NaN
    assert torch.equal(got[6], b)  # a constant row: deviations 0
    keep = [0, 1, 3, 5, 7, 8]
    assert torch.equal(got[keep], clean[keep])


def test_same_bits_every_run_and_on_another_stream():
    x, w, b, dy = make(7001, 256, torch.bfloat16, seed=8)
    runs = []
    for stream in (None, torch.cuda.Stream(), torch.cuda.Stream()):
        with torch.cuda.stream(stream):
            if stream is not None:
                stream.wait_stream(torch.cuda.default_stream())
            leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
            out = layer_norm(*leaves)
            runs.append([out.detach(), *torch.autograd.grad(out, leaves, dy)])
    torch.cuda.synchronize()
    for other in runs[1:]:
        for a, c in zip(runs[0], other):
            assert torch.equal(a, c)


def test_captured_and_replayed():
    x, w, b, dy = make(300, 256, torch.float32, seed=10)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]

    def both():
        out = layer_norm(*leaves)
        return [out.detach(), *torch.autograd.grad(out, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    fresh = make(300, 256, torch.float32, seed=11)[0]
    with torch.no_grad():
        leaves[0].copy_(fresh)
    graph.replay()
    torch.cuda.synchronize()
    for a, c in zip(captured, both()):
        assert torch.equal(a, c)
