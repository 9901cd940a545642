"""Cases of the decoder-layer training operators: ``linear`` (matrix product with bias, activation
and residual, and its gradients), ``layer_norm`` (forward and backward) and ``adamw_step`` (one AdamW
step over many tensors, moments in 32 or in 8 bits).

``own`` false: the operators written with elementary torch operations.  ``own`` true: the calls a
user makes of the package.  ``exact`` gives the same outputs from the definitions in 64 bits.
"""

import itertools
import math

import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BETAS, EPS, DECAY, LR = (0.9, 0.999), 1e-8, 1e-4, 1e-4
BLOCK = 256  # elements that share one scale of the 8-bit moments


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # the class head on one image's queries: an odd number of outputs, latency counts
        _linear("class head", 300, 256, 91, "bfloat16", "none", False, False),
        # one row against a wide layer: bound by reading the weight once
        _linear("one row", 1, 4096, 4096, "float16", "gelu", False, False),
        # the decoder's feed-forward block in training: 8 images x 13 groups x 300 queries, d_model 256
        _linear("feed-forward up", 31200, 256, 2048, "bfloat16", "relu", False, True),
        _linear("feed-forward down", 31200, 2048, 256, "bfloat16", "none", True, True),
        # the feature map's tokens (8 images x 1701) through a smooth activation
        _linear("token mixer", 13608, 384, 1536, "float16", "gelu", False, True),
        # the largest product: a wide layer in training
        _linear("wide layer", 16384, 4096, 4096, "bfloat16", "gelu", True, True),
        # the decoder's norms in training, and a ragged one in float32; the widest batch; one image's queries
        _norm("decoder norm", 31200, 256, "bfloat16", True),
        _norm("ragged norm", 1701, 393, "float32", True),
        _norm("large norm", 65536, 1024, "float16", True),
        _norm("query norm", 300, 256, "float32", False),
        # six decoder layers' parameters, moments in 32 bits
        _adamw("decoder step", 6, 256, 2048, "float32", 32),
        # eight wide layers, moments in 8 bits
        _adamw("wide step", 8, 1024, 4096, "float32", 8),
    ]


def _linear(name, rows, inner, outer, dtype, act, residual, train):
    return {"name": name, "op": "linear", "rows": rows, "in": inner, "out": outer, "dtype": dtype, "act": act,
            "residual": residual, "train": train}


def _norm(name, rows, dim, dtype, train):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "train": train}


def _adamw(name, layers, width, hidden, dtype, bits):
    return {"name": name, "op": "adamw", "layers": layers, "width": width, "hidden": hidden, "dtype": dtype,
            "bits": bits}


def draw(rng):
    """One more case.  Sizes are log-uniform over the whole range, so most are odd."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("linear", "norm", "adamw"))
    if op == "linear":
        inner, outer, train = log(8, 4096), log(1, 4096), rng.random() < 0.6
        if rng.random() < 0.5:  # widths of real layers are mostly multiples of 8
            inner, outer = max(8, inner // 8 * 8), max(8, outer // 8 * 8)
        most = 16384 * 4096 * 4096 // (inner * outer)
        c = _linear("", min(log(1, 32768), most), inner, outer, rng.choice(("bfloat16", "float16")),
                    rng.choice(("none", "relu", "gelu")), rng.random() < 0.4, train)
    elif op == "norm":
        dim = log(8, 8192)
        c = _norm("", min(log(1, 65536), 65536 * 1024 // dim), dim, rng.choice(tuple(DTYPES)), rng.random() < 0.7)
    else:
        c = _adamw("", rng.randint(1, 8), log(16, 1024), log(16, 4096), rng.choice(tuple(DTYPES)),
                   rng.choice((8, 32)))
    del c["name"]
    return c


def _sizes(case):
    """Elements of each parameter of `layers` decoder layers and a class head: projections and their
    biases, sampling offsets and weights, the feed-forward block, three norms."""
    d, f = case["width"], case["hidden"]
    layer = [d * d, d] * 4 + [192 * d, 192, 96 * d, 96] + [f * d, f, d * f, d] + [d] * 6
    return layer * case["layers"] + [91 * d, 91]


def _starts(case):
    """Where each parameter lies in the flat buffers (a multiple of BLOCK), and their length."""
    ends = list(itertools.accumulate(-(-n // BLOCK) * BLOCK for n in _sizes(case)))
    return [0] + ends[:-1], ends[-1]


# --------------------------------------------------------------------------- inputs

def _state(case, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=device) * scale).to(dtype)

    if case["op"] == "linear":
        m, k, n = case["rows"], case["in"], case["out"]
        s = {"x": normal(m, k), "weight": normal(n, k, scale=k ** -0.5), "bias": normal(n, scale=0.1)}
        s["residual"] = normal(m, n) if case["residual"] else None
        s["grad"] = normal(m, n) if case["train"] else None
        leaves = ("x", "weight", "bias", "residual")
    elif case["op"] == "norm":
        m, d = case["rows"], case["dim"]
        s = {"x": normal(m, d, scale=2.0), "weight": 1 + normal(d, scale=0.2), "bias": normal(d, scale=0.2)}
        s["x"] += normal(m, 1)  # rows have a mean of their own
        s["grad"] = normal(m, d) if case["train"] else None
        leaves = ("x", "weight", "bias")
    else:
        sizes = _sizes(case)
        starts, total = _starts(case)
        first = torch.tensor(starts, device=device)
        spans = torch.tensor([b - a for a, b in zip(starts, starts[1:] + [total])], device=device)
        last = (first + torch.tensor(sizes, device=device)).repeat_interleave(spans, output_size=total)
        inside = torch.arange(total, device=device) < last  # the rest is padding
        spread = torch.exp(torch.randn(total, generator=g, device=device) * 1.5) * inside  # gradients differ in size
        s = {"param": (normal(total, scale=0.05, dtype=torch.float32) * inside).to(dt), "grad":
             (normal(total, scale=1e-3, dtype=torch.float32) * spread).to(dt), "step": 100}
        m = normal(total, scale=3e-4, dtype=torch.float32) * spread
        v = (1e-3 * spread) ** 2 * (0.5 + torch.rand(total, generator=g, device=device))
        if case["bits"] == 32:
            s["exp_avg"], s["exp_avg_sq"], s["scales"] = m, v, None
        else:
            blocks, tiny = total // BLOCK, 1e-30
            sm, sv = m.view(blocks, BLOCK).abs().amax(1), v.view(blocks, BLOCK).amax(1)
            a = (m.view(blocks, BLOCK).abs() / sm.clamp_min(tiny)[:, None]).sqrt() * 127
            b = (v.view(blocks, BLOCK) / sv.clamp_min(tiny)[:, None]).sqrt().sqrt() * 255
            s["exp_avg"] = (a.round().view(-1) * m.sign()).to(torch.int8)
            s["exp_avg_sq"] = torch.where(v > 0, b.round().clamp_min(1).view(-1), 0.0).to(torch.uint8)
            s["scales"] = (sm, sv)
        ends = [a + n for a, n in zip(starts, sizes)]

        def views(t):
            return [t[a:e] for a, e in zip(starts, ends)]

        def scale_views(t):
            return [t[a // BLOCK:-(-e // BLOCK)] for a, e in zip(starts, ends)]

        s["lists"] = [views(s[k]) for k in ("param", "grad", "exp_avg", "exp_avg_sq")]
        s["scale_lists"] = None if s["scales"] is None else tuple(scale_views(t) for t in s["scales"])
        s["starts"], s["spans"] = first, spans
        leaves = ()
    _ = [s[k].requires_grad_(case["train"]) for k in leaves if s[k] is not None]
    s["case"] = case
    return s


def prepare(case, seed):
    return _state(case, seed, torch.device("cuda"))


# --------------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if op == "linear":
        return _run_linear(state)
    return _run_norm(state) if op == "norm" else _run_adamw(state)


def _run_linear(s):
    act = s["case"]["act"]
    if own:
        from rfdetr_training_throughput_b200.linear import linear

        out = linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"])
        if s["grad"] is None:
            return {"out": out}
        wanted = [t for t in (s["x"], s["weight"], s["bias"], s["residual"]) if t is not None]
        grads = torch.autograd.grad(out, wanted, s["grad"])
        return {"out": out, "grads": list(grads)}
    with torch.no_grad():
        dt = s["x"].dtype
        x, w = s["x"].float(), s["weight"].float()
        pre = x @ w.t() + s["bias"].float()
        if act == "relu":
            h = pre * (pre > 0)
        elif act == "gelu":
            cdf = 0.5 + 0.5 * torch.erf(pre * math.sqrt(0.5))
            h = pre * cdf
        else:
            h = pre
        out = (h if s["residual"] is None else h + s["residual"].float()).to(dt)
        if s["grad"] is None:
            return {"out": out}
        dy = s["grad"].float()
        if act == "relu":
            dp = dy * (pre > 0)
        elif act == "gelu":
            dp = dy * (cdf + pre * torch.exp(-0.5 * pre * pre) * (1.0 / math.sqrt(2 * math.pi)))
        else:
            dp = dy
        grads = [(dp @ w).to(dt), (dp.t() @ x).to(dt), dp.sum(0, dtype=torch.float64).to(dt)]
        if s["residual"] is not None:
            grads.append(s["grad"])
        return {"out": out, "grads": grads}


def _run_norm(s):
    if own:
        from rfdetr_training_throughput_b200.norm import layer_norm

        out = layer_norm(s["x"], s["weight"], s["bias"], 1e-5)
        if s["grad"] is None:
            return {"out": out}
        return {"out": out, "grads": list(torch.autograd.grad(out, [s["x"], s["weight"], s["bias"]], s["grad"]))}
    with torch.no_grad():
        dt = s["x"].dtype
        x, w = s["x"].float(), s["weight"].float()
        mid = x - x.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt((mid * mid).mean(1, keepdim=True) + 1e-5)
        unit = mid * rstd
        out = (unit * w + s["bias"].float()).to(dt)
        if s["grad"] is None:
            return {"out": out}
        dy = s["grad"].float()
        t = dy * w
        dx = rstd * (t - t.mean(1, keepdim=True) - unit * (t * unit).mean(1, keepdim=True))
        grads = [dx.to(dt), (dy * unit).sum(0, dtype=torch.float64).to(dt), dy.sum(0, dtype=torch.float64).to(dt)]
        return {"out": out, "grads": grads}


def _run_adamw(s):
    s["step"] += 1
    eight = s["scales"] is not None
    if own:
        from rfdetr_training_throughput_b200.optim import adamw_step, dequantize_moments

        adamw_step(*s["lists"], s["step"], scales=s["scale_lists"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY)
        if eight:
            return {"param": s["param"], "moments": list(dequantize_moments(s["exp_avg"], s["exp_avg_sq"],
                                                                            *s["scales"]))}
        return {"param": s["param"], "moments": [s["exp_avg"], s["exp_avg_sq"]]}
    t, (b1, b2) = s["step"], BETAS
    g = s["grad"].float()
    m, v = _decode(s) if eight else (s["exp_avg"], s["exp_avg_sq"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    denom = torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** t)) + EPS
    p = s["param"].float() * (1 - LR * DECAY) - (m / denom) * (LR / (1 - b1 ** t))
    s["param"].copy_(p)
    if eight:
        _encode(s, m, v, t)
        return {"param": s["param"], "moments": list(_decode(s))}
    s["exp_avg"].copy_(m)
    s["exp_avg_sq"].copy_(v)
    return {"param": s["param"], "moments": [s["exp_avg"], s["exp_avg_sq"]]}


def _decode(s):
    """The moments that the codes stand for: m = scale * c|c| / 127^2, v = scale * (c / 255)^4."""
    sm, sv = s["scales"]
    a = s["exp_avg"].float() * (1 / 127)
    b = s["exp_avg_sq"].float() * (1 / 255)
    b = b * b
    m = sm[:, None] * (a * a.abs()).view(-1, BLOCK)
    v = sv[:, None] * (b * b).view(-1, BLOCK)
    return m.view(-1), v.view(-1)


def _mix(h):
    h = (h * 0x9E3779B1) & 0xFFFFFFFF
    h = h ^ (h >> 15)
    h = (h * 0x85C1E8B7) & 0xFFFFFFFF
    return h ^ (h >> 13)


def _encode(s, m, v, t):
    """Block maxima as scales; codes rounded down or up at random, by a hash of the step, the tensor's
    number and the element's place in it.  A second moment above zero keeps a code above zero."""
    sm, sv = m.view(-1, BLOCK).abs().amax(1), v.view(-1, BLOCK).amax(1)
    s["scales"][0].copy_(sm)
    s["scales"][1].copy_(sv)
    count = torch.arange(s["starts"].numel(), device=m.device)
    key = _mix((count * 0x632BE5AB + t * 0xC2B2AE35) & 0xFFFFFFFF)
    place = torch.arange(m.numel(), device=m.device)
    place = (place - s["starts"].repeat_interleave(s["spans"], output_size=m.numel())) & 0xFFFFFFFF
    h = _mix((place + key.repeat_interleave(s["spans"], output_size=m.numel())) & 0xFFFFFFFF)
    low, high = (h & 0xFFFF).float() * 2.0 ** -16, (h >> 16).float() * 2.0 ** -16
    a = torch.sqrt(m.view(-1, BLOCK).abs() / sm[:, None]).view(-1) * 127 + low
    b = torch.sqrt(torch.sqrt(v.view(-1, BLOCK) / sv[:, None])).view(-1) * 255 + high
    a = torch.nan_to_num(torch.floor(a), nan=0.0).clamp_max(127)
    b = torch.nan_to_num(torch.floor(b), nan=0.0).clamp_max(255)
    b = torch.where(v > 0, b.clamp_min(1), b)
    s["exp_avg"].copy_(torch.where(m < 0, -a, a))
    s["exp_avg_sq"].copy_(b)


# --------------------------------------------------------------------------- work

def work(case):
    """Bytes: each input read once and each output written once.  Flops: products and sums."""
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "linear":
        m, k, n = case["rows"], case["in"], case["out"]
        values = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        flops = 2 * m * k * n
        if case["train"]:
            values += m * n + m * k + n * k + n  # the gradient comes in; those of x, weight and bias go out
            flops *= 3
        return {"bytes": size * values, "flops": flops}
    if case["op"] == "norm":
        m, d = case["rows"], case["dim"]
        return {"bytes": size * ((4 if case["train"] else 2) * m * d + (4 if case["train"] else 2) * d),
                "flops": (20 if case["train"] else 8) * m * d}
    n = sum(_sizes(case))
    if case["bits"] == 32:
        return {"bytes": n * (3 * size + 16), "flops": 15 * n}
    # codes in and out, and the moments that are returned in 32 bits, with the scales
    return {"bytes": n * (3 * size + 4 + 8) + 16 * (n // BLOCK), "flops": 30 * n}


# --------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    """`run`'s outputs in 64 bits.  The 8-bit moments have none: they are random roundings to a
    grid, and a value next to a border may fall on either side of it in another precision."""
    s = _state(case, seed, torch.device("cuda"))
    if case["op"] == "adamw":
        return _exact_adamw(case, s)
    wide = {k: t.detach().double().requires_grad_(True) for k, t in s.items()
            if k in ("x", "weight", "bias", "residual") and t is not None}
    if case["op"] == "linear":
        out = torch.einsum("mk,nk->mn", wide["x"], wide["weight"]) + wide["bias"]
        if case["act"] == "relu":
            out = torch.clamp_min(out, 0)
        elif case["act"] == "gelu":
            out = out * torch.special.ndtr(out)
        if case["residual"]:
            out = out + wide["residual"]
    else:
        var, mean = torch.var_mean(wide["x"], dim=1, correction=0, keepdim=True)
        out = (wide["x"] - mean) * torch.rsqrt(var + 1e-5) * wide["weight"] + wide["bias"]
    if not case["train"]:
        return {"out": out.detach()}
    out.backward(s["grad"].double())
    return {"out": out.detach(), "grads": [t.grad for t in wide.values()]}


def _exact_adamw(case, s):
    t, g = s["step"] + 1, s["grad"].double()
    if case["bits"] == 8:
        level = np.arange(-127, 128) / 127.0
        first = torch.from_numpy(np.sign(level) * level ** 2).to(g.device)[s["exp_avg"].long() + 127]
        second = torch.from_numpy((np.arange(256) / 255.0) ** 4).to(g.device)[s["exp_avg_sq"].long()]
        m = first * s["scales"][0].double().repeat_interleave(BLOCK)
        v = second * s["scales"][1].double().repeat_interleave(BLOCK)
    else:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    m = torch.lerp(g, m, BETAS[0])
    v = torch.lerp(g.square(), v, BETAS[1])
    hat_m, hat_v = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
    p = s["param"].double()
    p = p - LR * (DECAY * p + hat_m / (hat_v.sqrt() + EPS))
    return {"param": p, "moments": [None, None] if case["bits"] == 8 else [m, v]}
