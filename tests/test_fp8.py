"""What the 8-bit linear layers' faces refuse, without a device."""
import pytest
import torch

from purhie_b200.csrc import fp8, ops
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
    ("alpha, limit and shift", lambda: fp8._gate((1.702, 7.0))),
    ("alpha, limit and shift", lambda: fp8._gate((1.702, 7.0, 1.0, 0.0))),
    ("float8", lambda: fp8.gemm(bf16(2, 64), f32(2, 1), e4m3(8, 64), f32(1, 1))),
    ("float8", lambda: fp8.gemm(e4m3(64, 2).t(), f32(2, 1), e4m3(8, 64), f32(1, 1))),
    ("do not fit", lambda: fp8.gemm(e4m3(2, 64), f32(2, 1), e4m3(8, 32), f32(1, 1))),
    ("do not fit", lambda: fp8.gemm(e4m3(2, 64), f32(2, 1), e4m3(0, 64), f32(0, 1))),
    ("x_scales", lambda: fp8.gemm(e4m3(2, 144), f32(2, 1), e4m3(8, 144), f32(1, 2))),
    ("w_scales", lambda: fp8.gemm(e4m3(2, 144), f32(2, 2), e4m3(129, 144), f32(1, 2))),
    ("multiple of 256", lambda: fp8.gemm_gated(e4m3(2, 64), f32(2, 1), e4m3(128, 64), f32(1, 1))),
    ("w_scales", lambda: fp8.gemm_gated(e4m3(2, 64), f32(2, 1), e4m3(256, 64), f32(1, 1))),
    ("CUDA", lambda: fp8.gemm_gated(e4m3(2, 64), f32(2, 1), e4m3(256, 64), f32(2, 1))),
    ("CUDA", lambda: fp8.gemm(e4m3(2, 64), f32(2, 1), e4m3(8, 64), f32(1, 1))),
]


@pytest.mark.parametrize("text,call", REFUSED, ids=[f"{i}-{t.replace(' ', '_')}" for i, (t, _) in enumerate(REFUSED)])
def test_faces_refuse(text, call):
    with pytest.raises(KernelError, match=text):
        call()


X, S = 1 << 20, 1 << 21          # addresses that nothing reads: every call below is refused on the host
C_REFUSED = [
    ("blocks are of", "ph_quantize_fp8", (X, 0, 8, X, S, 4, 8, 2, None)),
    ("bad arguments", "ph_quantize_fp8", (X, 0, 7, X, S, 4, 8, 1, None)),
    ("bad arguments", "ph_quantize_fp8", (X, 2, 8, X, S, 4, 8, 1, None)),
    ("bad arguments", "ph_quantize_fp8", (None, 0, 8, X, S, 4, 8, 1, None)),
    ("65535", "ph_quantize_fp8", (X, 0, 8, X, S, 65535 * 128 + 1, 8, 128, None)),
    ("too many blocks", "ph_quantize_fp8", (X, 0, 4096, X, S, 2 ** 31 - 1, 4096, 1, None)),
    ("at most 32768", "ph_add_rmsnorm_fp8", (X, None, 0, 1, 0, X, 1e-6, None, 1, 1, 32769, None, X, S, None)),
    ("bad arguments", "ph_add_rmsnorm_fp8", (X, X, 0, 0, 64, X, 1e-6, None, 1, 1, 64, None, X, S, None)),
    ("bad arguments", "ph_add_rmsnorm_fp8", (X, X, 0, 1, 64, X, float("nan"), None, 1, 1, 64, None, X, S, None)),
    ("not kept", "ph_add_rmsnorm_fp8", (X, X, 0, 1, 64, X, 1e-6, X, 1, 1, 64, X, X, S, None)),
    ("bad arguments", "ph_gated_fp8", (X, 0, 0, 0, X, S, 4, 8, None, None)),
    ("gate 3", "ph_gated_fp8", (X, 0, 1, 0, X, S, 4, 8, (fp8.c_float * 4)(0, 0, 0, 3), None)),
    ("too many blocks", "ph_gated_fp8", (X, 0, 1, 0, X, S, 2 ** 31 - 1, 256, None, None)),
    ("multiple of 16", "ph_gemm_fp8", (X, S, X, S, X, 0, 4, 8, 24, 16, 1, None, 0, None, None)),
    ("aligned", "ph_gemm_fp8", (X + 8, S, X, S, X, 0, 4, 8, 32, 16, 1, None, 0, None, None)),
    ("at most", "ph_quantize_fp8", (X, 0, 2 ** 31 - 1, X, S, 1, 2 ** 31 - 1, 1, None)),
    ("65535", "ph_quantize_fp8", (X, 0, 8, X, S, 2 ** 31 - 1, 8, 128, None)),
    ("at most", "ph_gemm_fp8", (X, S, X, S, X, 0, 4, 8, 2 ** 31 - 16, 16, 1, None, 0, None, None)),
    ("at most", "ph_gemm_fp8", (X, S, X, S, X, 0, 2 ** 31 - 1, 8, 32, 16, 1, None, 0, None, None)),
    ("no room", "ph_gemm_fp8", (X, S, X, S, None, 0, 4, 8, 256, 16, 1, None, 0, None, None)),
    ("no room", "ph_gemm_fp8", (X, S, X, S, X, 0, 4, 8, 256, 16, 2, None, 0, None, None)),
    ("summed here", "ph_gemm_fp8", (X, S, X, S, X, 0, 4, 8, 256, 16, 2, X + 4, 0, None, None)),
    ("parts of K", "ph_gemm_fp8", (X, S, X, S, X, 0, 4, 8, 256, 16, 3, X, 0, None, None)),
    ("tile 128", "ph_gemm_fp8", (X, S, X, S, X, 0, 4, 8, 256, 128, 1, None, 0, None, None)),
    ("one of 256", "ph_gemm_fp8_gated", (X, S, X, S, X, S, 4, 128, 32, None, None, None)),
    ("multiple of 16", "ph_gemm_fp8_gated", (X, S, X, S, X, S, 4, 256, 24, None, None, None)),
    ("aligned", "ph_gemm_fp8_gated", (X, S, X, S, X + 8, S, 4, 256, 32, None, None, None)),
    ("gate 5", "ph_gemm_fp8_gated", (X, S, X, S, X, S, 4, 256, 32, (fp8.c_float * 4)(0, 0, 0, 5), None, None)),
    ("no plan", "ph_gemm_fp8_plan", (0, 8, 32, 1, X, S)),
    ("no plan", "ph_gemm_fp8_plan", (4, 8, 32, 1, None, S)),
]


@pytest.mark.parametrize("text,name,args", C_REFUSED, ids=[f"{i}-{n}" for i, (_, n, _) in enumerate(C_REFUSED)])
def test_launchers_refuse(text, name, args):
    with pytest.raises(KernelError, match=text):
        ops.call("fp8", name, *args)


@pytest.mark.parametrize("whole", [True, False])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 6144, 4096), (8, 4096, 12288), (64, 24576, 4096), (65, 100, 40000), (203, 1000, 2064),
                                   (2048, 24576, 4096), (1 << 30, 8, 16), (4, 1 << 30, 16)])
def test_plans(M, N, K, whole):
    """What a plan gives can be launched, and what the caller gave stays."""
    tile, splits = fp8.plan(M, N, K, whole=whole)
    assert tile in (16, 32, 64, 96, 256) and 1 <= splits <= min(16, -(-K // 128))
    for given in (16, 256):
        assert fp8.plan(M, N, K, tile=given)[0] == given
    assert fp8.plan(M, N, K, splits=1)[1] == 1
    with pytest.raises(KernelError, match="not one of"):
        fp8.plan(M, N, K, tile=48)
    with pytest.raises(KernelError, match="parts of K"):
        fp8.plan(M, N, K, splits=17)
