"""The layer operators' kernels start early and wait for the work before them: inputs that arrive by a
copy, a memset, another stream's kernel or a kernel that has only just been launched are the ones read,
and buffers that are overwritten right after a call were read before."""

import pytest
import torch

from rfdetr_training_throughput_b200.linear import linear
from rfdetr_training_throughput_b200.norm import layer_norm
from rfdetr_training_throughput_b200.optim import adamw_step, dequantize_moments, quantize_moments

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def operators():
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(256, 512, device=DEV, generator=g).to(torch.bfloat16)
    n = torch.randn(512, device=DEV, generator=g).to(torch.bfloat16)
    return {"product": (lambda x: linear(x, w, activation="gelu"), 3000), "row": (lambda x: linear(x, w), 1),
            "split": (lambda x: linear(x, w[:64]), 40), "norm": (lambda x: layer_norm(x, n, n), 3000)}


@pytest.mark.parametrize("name", ["product", "row", "split", "norm"])
def test_inputs_that_have_just_arrived(name):
    op, rows = operators()[name]
    batches = [torch.randn(rows, 512).to(torch.bfloat16).pin_memory() for _ in range(3)]
    want = [op(b.to(DEV)) for b in batches]
    zero = op(torch.zeros(rows, 512, device=DEV, dtype=torch.bfloat16))
    torch.cuda.synchronize()
    x = torch.empty(rows, 512, device=DEV, dtype=torch.bfloat16)
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    other = torch.empty_like(x)
    heavy = torch.randn(1500, 1500, device=DEV)
    got = []
    for i in range(12):
        k = i % 3
        x.copy_(batches[k], non_blocking=True)       # a copy right before
        got.append((k, op(x)))
        x.zero_()                                    # overwritten right after, and read again
        got.append((None, op(x)))
        with torch.cuda.stream(side):                # another stream's work, long enough to be waited for
            side.wait_stream(main)
            heavy @ heavy
            other.copy_(batches[k], non_blocking=True)
            other.neg_().neg_()
        main.wait_stream(side)
        got.append((k, op(other)))
        x.add_(other)                                # a kernel right before
        got.append((k, op(x)))
    torch.cuda.synchronize()
    for k, out in got:
        assert torch.equal(out, zero if k is None else want[k])


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_in_a_row(bits):
    """Steps whose gradients are written between them, with and without a device step counter, against
    the same steps with a synchronisation after every kernel."""
    def run(wait):
        torch.manual_seed(3)
        p = [torch.randn(n, device=DEV) for n in (300_000, 17, 4096)]
        m, v = [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]
        scales = None
        if bits == 8:
            m, v, sm, sv = map(list, zip(*(quantize_moments(a, b) for a, b in zip(m, v))))
            scales = (sm, sv)
        g = [torch.empty_like(x) for x in p]
        step = torch.zeros((), dtype=torch.int64, device=DEV)
        moments = []
        for t in range(1, 7):
            for i, x in enumerate(g):
                torch.sin(p[i] * t, out=x)
                wait()
            step.add_(1)
            wait()
            adamw_step(p, g, m, v, step if t % 2 else t, scales=scales, lr=1e-2)
            wait()
            if bits == 8:
                moments += dequantize_moments(m[0], v[0], scales[0][0], scales[1][0])
                wait()
        torch.cuda.synchronize()
        return p + m + v + moments

    for a, b in zip(run(lambda: None), run(torch.cuda.synchronize)):
        assert torch.equal(a, b)


def test_captured_step_whose_first_launch_is_empty():
    """More tensors than one launch takes, the first of them all empty, captured behind another kernel."""
    count = 700
    p = [torch.randn(0 if i < 600 else 100 + i, device=DEV) for i in range(count)]
    other = [x.clone() for x in p]
    state = [[torch.zeros_like(x) for x in p] for _ in range(4)]
    g = [torch.empty_like(x) for x in p]

    def one(t, params, m, v):
        torch._foreach_copy_(g[600:], [torch.sin(x) for x in params[600:]])
        adamw_step(params, g, m, v, t, lr=1e-2)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one(1, p, *state[:2])
    for t in range(3):
        graph.replay()
        one(1, other, *state[2:])
    torch.cuda.synchronize()
    for a, b in zip(p, other):
        assert torch.equal(a, b)
