"""What the 8-bit linear layers' faces refuse, without a device."""
import pytest
import torch

from purhie_b200.csrc import fp8
from purhie_b200.native import KernelError

E4M3 = torch.float8_e4m3fn


def f32(*shape):
    return torch.zeros(shape)


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def e4m3(*shape):
    return torch.zeros(shape).to(E4M3)


REFUSED = [
    ("matrix", lambda: fp8.quantize(f32(8))),
    ("matrix", lambda: fp8.quantize(f32(8, 0))),
    ("block_rows", lambda: fp8.quantize(f32(8, 8), block_rows=64)),
    ("rows of x", lambda: fp8.quantize(f32(8, 8).t()[:, ::2])),
    ("rows of x", lambda: fp8.quantize(f32(1, 8).expand(4, 8))),
    ("CUDA", lambda: fp8.quantize(f32(8, 8))),
    ("at most", lambda: fp8.add_rmsnorm(f32(1, 32769), None, f32(32769), 1e-6)),
    ("x must be", lambda: fp8.add_rmsnorm(bf16(2, 64), None, f32(64), 1e-6)),
    ("x must be", lambda: fp8.add_rmsnorm(f32(2, 128)[:, :64], None, f32(64), 1e-6)),
    ("weight", lambda: fp8.add_rmsnorm(f32(2, 64), None, f32(63), 1e-6)),
    ("weight", lambda: fp8.add_rmsnorm(f32(2, 64), None, bf16(64), 1e-6)),
    ("add must", lambda: fp8.add_rmsnorm(f32(2, 64), f32(3, 64), f32(64), 1e-6)),
    ("add must", lambda: fp8.add_rmsnorm(f32(2, 64), f32(2, 64), f32(64), 1e-6, add_splits=2)),
    ("add must", lambda: fp8.add_rmsnorm(f32(2, 64), f32(2, 64), f32(64), 1e-6, add_splits=0)),
    ("eps", lambda: fp8.add_rmsnorm(f32(2, 64), None, f32(64), -1.0)),
    ("eps", lambda: fp8.add_rmsnorm(f32(2, 64), None, f32(64), float("nan"))),
    ("rows must", lambda: fp8.add_rmsnorm(f32(2, 64), None, f32(64), 1e-6, rows=torch.zeros(1, dtype=torch.int64))),
    ("x_out", lambda: fp8.add_rmsnorm(f32(2, 64), None, f32(64), 1e-6, rows=torch.zeros(1, dtype=torch.int32), x_out=f32(2, 64))),
    ("CUDA", lambda: fp8.add_rmsnorm(f32(2, 64), f32(2, 64), f32(64), 1e-6)),
    ("gate_up", lambda: fp8.gated(f32(2, 63))),
    ("gate_up", lambda: fp8.gated(f32(2, 0))),
    ("gate_up", lambda: fp8.gated(f32(2, 64), splits=2)),
    ("gate_up", lambda: fp8.gated(f32(3, 2, 64), splits=2)),
    ("gate_up", lambda: fp8.gated(f32(2, 128)[:, :64])),
    ("CUDA", lambda: fp8.gated(f32(2, 64))),
    ("gate 'relu'", lambda: fp8._gate("relu")),
    ("float8", lambda: fp8.gemm(bf16(2, 64), f32(2, 1), e4m3(8, 64), f32(1, 1))),
    ("float8", lambda: fp8.gemm(e4m3(64, 2).t(), f32(2, 1), e4m3(8, 64), f32(1, 1))),
    ("do not fit", lambda: fp8.gemm(e4m3(2, 64), f32(2, 1), e4m3(8, 32), f32(1, 1))),
    ("do not fit", lambda: fp8.gemm(e4m3(2, 64), f32(2, 1), e4m3(0, 64), f32(0, 1))),
    ("x_scales", lambda: fp8.gemm(e4m3(2, 144), f32(2, 1), e4m3(8, 144), f32(1, 2))),
    ("w_scales", lambda: fp8.gemm(e4m3(2, 144), f32(2, 2), e4m3(129, 144), f32(1, 2))),
    ("CUDA", lambda: fp8.gemm(e4m3(2, 64), f32(2, 1), e4m3(8, 64), f32(1, 1))),
]


@pytest.mark.parametrize("text,call", REFUSED, ids=[f"{i}-{t.replace(' ', '_')}" for i, (t, _) in enumerate(REFUSED)])
def test_faces_refuse(text, call):
    with pytest.raises(KernelError, match=text):
        call()
