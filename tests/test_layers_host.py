"""What the layer operators refuse before any CUDA call: host tensors, wrong types and shapes, and the C
ABI's own checks."""

import ctypes
import os
import re

import numpy as np
import pytest
import torch

from rfdetr_training_throughput_b200 import _lib
from rfdetr_training_throughput_b200.linear import linear
from rfdetr_training_throughput_b200.norm import layer_norm
from rfdetr_training_throughput_b200.optim import AdamW, adamw_step, dequantize_moments, quantize_moments

FAKE = 1 << 40  # never dereferenced: every call below fails its checks first
HEADER = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "rfm.h")).read()


def test_host_tensors_are_refused():
    x = torch.zeros(3, 8)
    with pytest.raises(ValueError, match="CUDA"):
        layer_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        linear(x, x)
    with pytest.raises(ValueError, match="activation"):
        linear(x, x, activation="tanh")
    with pytest.raises(ValueError, match="CUDA"):
        adamw_step([x], [x], [x], [x], 1)
    with pytest.raises(ValueError, match="CUDA"):
        dequantize_moments(x.to(torch.int8), x.to(torch.uint8), x, x)


def test_optimizer_arguments():
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(amsgrad=True), dict(maximize=True), dict(differentiable=True)):
        with pytest.raises(NotImplementedError):
            AdamW([p], **bad)
    for bad in (dict(moment_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=-0.1),
                dict(lr=torch.tensor(0.1))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    opt = AdamW([p], lr=1e-3)
    opt.step()  # no gradient: nothing to do
    assert not opt.state


def test_quantize_moments_on_the_host():
    """Nearest codes: |m| = s (c / 127)^2, so half a code near the top is off by s / 127 at most."""
    g = torch.Generator().manual_seed(0)
    m, v = torch.randn(700, generator=g), torch.rand(700, generator=g)
    cm, cv, sm, sv = quantize_moments(m, v)
    assert cm.dtype == torch.int8 and cv.dtype == torch.uint8 and sm.shape == sv.shape == (3,)
    a, b = cm.double() / 127, cv.double() / 255
    back_m = sm.double().repeat_interleave(256)[:700] * a * a.abs()
    back_v = sv.double().repeat_interleave(256)[:700] * b ** 4
    top_m, top_v = sm.double().repeat_interleave(256)[:700], sv.double().repeat_interleave(256)[:700]
    assert bool(((back_m - m).abs() <= top_m * (1 / 127 + 1e-4)).all())
    assert bool(((back_v - v).abs() <= top_v * (2 / 255 + 1e-4)).all())
    zero = quantize_moments(torch.zeros(5), torch.tensor([0.0, 1e-30, 1.0, 0.0, 0.0]))
    assert zero[0].tolist() == [0] * 5 and zero[1].tolist() == [0, 1, 255, 0, 0]


def test_adamw_struct_matches_header():
    body = re.search(r"typedef struct rfm_adamw_tensor \{(.*?)\} rfm_adamw_tensor;", HEADER, re.S).group(1)
    assert len([line for line in body.split(";") if line.strip() and "/*" not in line.strip()[:2]]) == \
        _lib.ADAMW_TENSOR_WORDS
    assert f"#define RFM_MOMENT_BLOCK {_lib.MOMENT_BLOCK}\n" in HEADER
    for name, value in (("F32", _lib.DTYPE_F32), ("BF16", _lib.DTYPE_BF16), ("F16", _lib.DTYPE_F16)):
        assert f"#define RFM_DTYPE_{name} {value}\n" in HEADER


def test_layer_norm_abi_refusals():
    lib = _lib.load()

    def forward(x=FAKE, ld=8, w=None, b=None, out=FAKE, mean=None, rstd=None, rows=2, dim=8, eps=1e-5, dtype=0, pt=0):
        return lib.rfm_layer_norm_forward(x, ld, w, b, out, mean, rstd, rows, dim, eps, dtype, pt, None)

    for bad in (dict(x=None), dict(out=None), dict(ld=7), dict(rows=-1), dict(dim=0), dict(dtype=3), dict(pt=-1),
                dict(mean=FAKE), dict(eps=-1.0), dict(eps=float("nan"))):
        assert forward(**bad) == 1, bad
    assert forward(rows=1 << 41) == 2
    assert forward(rows=0, x=None, out=None) == 0

    def backward(x=FAKE, ld=8, mean=FAKE, rstd=FAKE, dy=FAKE, ldg=8, dx=FAKE, dw=FAKE, db=FAKE, rows=2, dim=8,
                 ws=FAKE, size=1 << 30):
        return lib.rfm_layer_norm_backward(x, ld, None, mean, rstd, dy, ldg, dx, dw, db, rows, dim, 0, 0, ws, size,
                                           None)

    for bad in (dict(x=None), dict(mean=None), dict(rstd=None), dict(dy=None), dict(ldg=7), dict(ws=None),
                dict(size=8), dict(rows=-1)):
        assert backward(**bad) == 1, bad
    assert backward(dx=None, dw=None, db=None) == 0
    assert lib.rfm_layer_norm_workspace_bytes(-1, 8) < 0 and lib.rfm_layer_norm_workspace_bytes(4, 0) < 0


def test_adamw_abi_refusals():
    lib = _lib.load()

    def step(row=(), table=True, count=1, dtype=0, bits=32, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, t=1, dlr=None,
             dstep=None, ws=None):
        base = [FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 5, 0]
        for i, v in dict(row).items():
            base[i] = v
        arr = np.array([base], dtype=np.int64)
        return lib.rfm_adamw(arr.ctypes.data if table else None, count, dtype, bits, lr, b1, b2, eps, wd, t, dlr,
                             dstep, None, ws, None)

    for bad in (dict(table=False), dict(count=-1), dict(dtype=5), dict(bits=16), dict(lr=-1.0), dict(b1=1.0),
                dict(b2=-0.1), dict(eps=-1.0), dict(wd=-1.0), dict(t=0), dict(dlr=FAKE), dict(dstep=FAKE),
                dict(dstep=FAKE, ws=FAKE + 4), dict(lr=float("nan"))):
        assert step(**bad) == 1, bad
    for i in range(4):
        assert step(row={i: 0}) == 1, i
    for bad in ({0: FAKE + 2}, {1: FAKE + 1}, {2: FAKE + 2}, {6: -1}, {7: 1}):
        assert step(row=bad) == 1, bad
    assert step(row={4: 0}, bits=8) == 1 and step(row={5: FAKE + 2}, bits=8) == 1
    assert step(row={6: 1 << 43}) == 2
    assert step(row={6: 0}) == 0 and step(count=0, table=False) == 0

    def moments(a=FAKE, n=5):
        return lib.rfm_adamw_moments(a, FAKE, FAKE, FAKE, n, FAKE, FAKE, None)

    assert moments(n=-1) == 1 and moments(a=None) == 1 and moments(n=0) == 0 and moments(n=1 << 42) == 2
    assert ctypes.sizeof(ctypes.c_int64) * _lib.ADAMW_TENSOR_WORDS == 64


def test_linear_structs_match_header(tmp_path):
    """ctypes mirrors of rfm_linear / rfm_linear_grad against the header, compiled with gcc."""
    import shutil
    import subprocess

    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    names = [("rfm_linear", _lib.Linear, "ld_residual"), ("rfm_linear", _lib.Linear, "reserved"),
             ("rfm_linear_grad", _lib.LinearGrad, "ld_grad_pre"), ("rfm_linear_grad", _lib.LinearGrad, "reserved")]
    src = tmp_path / "sz.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "rfm.h"\nint main(void) {\n'
                   + "".join(f'  printf("%zu %zu ", sizeof({s}), offsetof({s}, {f}));\n' for s, _, f in names)
                   + "  return 0;\n}\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [v for _, c, f in names for v in (ctypes.sizeof(c), getattr(c, f).offset)]
    for name, value in _lib.ACTIVATIONS.items():
        assert f"#define RFM_ACT_{name.upper()} {value}\n" in HEADER


def test_linear_abi_refusals():
    lib = _lib.load()

    def forward(**bad):
        args = dict(x=FAKE, weight=FAKE, out=FAKE, rows=3, ld_x=16, ld_weight=16, in_features=16, out_features=8,
                    dtype=_lib.DTYPE_BF16, bias_dtype=_lib.DTYPE_BF16)
        return lib.rfm_linear_forward(ctypes.byref(_lib.Linear(**{**args, **bad})), None)

    for bad in (dict(x=None), dict(weight=None), dict(out=None), dict(rows=-1), dict(in_features=0),
                dict(out_features=0), dict(dtype=_lib.DTYPE_F32), dict(x=FAKE + 2), dict(weight=FAKE + 8),
                dict(ld_x=12), dict(ld_x=8), dict(ld_weight=20), dict(ld_weight=0), dict(activation=3),
                dict(activation=-1), dict(reserved=1), dict(bias=FAKE, bias_dtype=_lib.DTYPE_F16),
                dict(residual=FAKE, ld_residual=7)):
        assert forward(**bad) == 1, bad
    assert forward(rows=1 << 31) == 2 and forward(in_features=(1 << 30) + 1) == 2
    assert forward(rows=0, x=None, weight=None, out=None) == 0
    assert lib.rfm_linear_forward(None, None) == 1

    def backward(**bad):
        args = dict(x=FAKE, weight=FAKE, grad_out=FAKE, grad_x=FAKE, grad_weight=FAKE, grad_bias=FAKE, rows=3, ld_x=16,
                    ld_weight=16, ld_grad=8, in_features=16, out_features=8, dtype=_lib.DTYPE_BF16,
                    bias_dtype=_lib.DTYPE_BF16, workspace=FAKE, workspace_bytes=1 << 30)
        return lib.rfm_linear_backward(ctypes.byref(_lib.LinearGrad(**{**args, **bad})), None)

    for bad in (dict(x=None), dict(weight=None), dict(grad_out=None), dict(rows=-1), dict(ld_grad=7), dict(ld_x=8),
                dict(workspace=None), dict(workspace=FAKE + 4), dict(workspace_bytes=4), dict(reserved=2),
                dict(activation=1), dict(activation=1, saved=FAKE), dict(bias_dtype=_lib.DTYPE_F16),
                dict(activation=1, saved=FAKE, grad_pre=FAKE, ld_grad_pre=4),
                dict(grad_out=FAKE + 2)):  # dP needs a place of its own
        assert backward(**bad) == 1, bad
    assert backward(grad_x=None, grad_weight=None, grad_bias=None) == 0
    assert lib.rfm_linear_backward(None, None) == 1
    assert lib.rfm_linear_forward_workspace_bytes(-1, 8, 8) < 0 and lib.rfm_linear_forward_workspace_bytes(1, 8, 8) == 0
    assert lib.rfm_linear_backward_workspace_bytes(4, 0, 8) < 0
    assert lib.rfm_linear_faults(None) == 1
