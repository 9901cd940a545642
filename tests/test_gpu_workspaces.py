"""The workspaces the C ABI asks for are all that its kernels use: each call gets exactly that many bytes
inside a larger buffer, and what lies around them stays."""

import ctypes

import pytest
import torch

from rfdetr_training_throughput_b200 import _lib

pytestmark = pytest.mark.gpu

GUARD = 8 << 20
MARK = 0x5A


def guarded(size):
    buf = torch.full((size + 2 * GUARD,), MARK, dtype=torch.uint8, device="cuda")
    return buf, buf.data_ptr() + GUARD


def untouched(buf, size):
    return bool((buf[:GUARD] == MARK).all()) and bool((buf[GUARD + size:] == MARK).all())


# products that are split and ones that are not; columns read 8 at a time and one by one
SIZES = [(16384, 2048, 2048), (31200, 256, 2048), (31200, 2048, 256), (4096, 4096, 4096), (300, 256, 91),
         (5000, 72, 333), (64, 4096, 512), (1, 512, 4096), (40, 64, 8), (100000, 16, 64)]


@pytest.mark.parametrize("rows,inner,outer", SIZES)
@pytest.mark.parametrize("activation", [0, 2])
def test_linear(rows, inner, outer, activation):
    lib = _lib.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    g = torch.Generator(device="cuda").manual_seed(rows + outer)

    def matrix(m, n):  # with rows that TMA can read
        wide = torch.randn(m, (n + 7) // 8 * 8, device="cuda", generator=g).to(torch.bfloat16)
        return wide, wide.shape[1]

    x, ld_x = matrix(rows, inner)
    w, ld_w = matrix(outer, inner)
    bias = torch.randn(outer, device="cuda", generator=g)
    out = torch.empty(rows, outer, dtype=torch.bfloat16, device="cuda")
    pre = torch.empty_like(out)
    size = lib.rfm_linear_forward_workspace_bytes(rows, inner, outer)
    buf, at = guarded(size)
    a = _lib.Linear(x=x.data_ptr(), weight=w.data_ptr(), bias=bias.data_ptr(), out=out.data_ptr(), pre=pre.data_ptr(),
                    workspace=at, workspace_bytes=size, rows=rows, ld_x=ld_x, ld_weight=ld_w, in_features=inner,
                    out_features=outer, dtype=_lib.DTYPE_BF16, bias_dtype=_lib.DTYPE_F32, activation=activation)
    _lib.check("rfm_linear_forward", lib.rfm_linear_forward(ctypes.byref(a), stream))
    assert untouched(buf, size)
    del buf
    size = lib.rfm_linear_backward_workspace_bytes(rows, inner, outer)
    buf, at = guarded(size)
    dy = torch.randn(rows, outer, device="cuda", generator=g).to(torch.bfloat16)
    dp, ld_dp = matrix(rows, outer)
    gx, gw = torch.empty(rows, inner, device="cuda").bfloat16(), torch.empty(outer, inner, device="cuda").bfloat16()
    gb = torch.empty(outer, device="cuda")
    a = _lib.LinearGrad(x=x.data_ptr(), weight=w.data_ptr(), saved=pre.data_ptr(), grad_out=dy.data_ptr(),
                        grad_pre=dp.data_ptr(), grad_x=gx.data_ptr(), grad_weight=gw.data_ptr(),
                        grad_bias=gb.data_ptr(), workspace=at, workspace_bytes=size, rows=rows, ld_x=ld_x,
                        ld_weight=ld_w, ld_grad=outer, ld_grad_pre=ld_dp, in_features=inner, out_features=outer,
                        dtype=_lib.DTYPE_BF16, bias_dtype=_lib.DTYPE_F32, activation=activation)
    _lib.check("rfm_linear_backward", lib.rfm_linear_backward(ctypes.byref(a), stream))
    assert untouched(buf, size)
    if activation == 0:  # the sums that went through the workspace (a rounding a row at most)
        want, size = dy.double().sum(0), dy.double().abs().sum(0)
        assert bool(((gb.double() - want).abs() <= rows * 2.0 ** -24 * size + 2.0 ** -24 * want.abs()).all())


@pytest.mark.parametrize("rows,dim", [(1, 8), (31200, 256), (65536, 40), (5000, 1024), (3000, 393), (2000, 8192),
                                      (500, 9000), (7, 4100), (40000, 31)])
def test_layer_norm(rows, dim):
    lib = _lib.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    x, dy, dx = (torch.randn(rows, dim, device="cuda") for _ in range(3))
    mean, rstd = x.mean(1), 1 / x.std(1, correction=0).clamp_min(0.1)
    gw, gb = torch.empty(dim, device="cuda"), torch.empty(dim, device="cuda")
    size = lib.rfm_layer_norm_workspace_bytes(rows, dim)
    buf, at = guarded(size)
    _lib.check("rfm_layer_norm_backward", lib.rfm_layer_norm_backward(
        x.data_ptr(), dim, None, mean.data_ptr(), rstd.data_ptr(), dy.data_ptr(), dim, dx.data_ptr(), gw.data_ptr(),
        gb.data_ptr(), rows, dim, _lib.DTYPE_F32, _lib.DTYPE_F32, at, size, stream))
    assert untouched(buf, size)
    want, size = dy.double().sum(0), dy.double().abs().sum(0)
    assert bool(((gb.double() - want).abs() <= (rows + 64) * 2.0 ** -24 * size).all())
