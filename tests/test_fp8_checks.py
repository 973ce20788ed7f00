"""What the 8-bit linear layers' faces refuse, and how, without a device (beside test_fp8.py)."""
import pytest
import torch

from purhie_b200.csrc import fp8
from purhie_b200.native import KernelError

E4M3 = torch.float8_e4m3fn


def test_host_tensors_are_refused_without_compiling_anything(monkeypatch):
    """On a machine with neither a device nor a compiler the refusal is the library's error, as everywhere else."""
    def none(name):
        raise RuntimeError(f"{name} would be compiled")
    monkeypatch.setattr(fp8, "_calls", None)
    monkeypatch.setattr(fp8, "load_extension", none)
    x, w = torch.zeros(2, 64), torch.zeros(2, 64).to(E4M3)
    for call in (lambda: fp8.quantize(x), lambda: fp8.add_rmsnorm(x, None, x[0], 1e-6), lambda: fp8.gated(x), lambda: fp8.gemm(w, x[:, :1].contiguous(), w, x[:1, :1])):
        with pytest.raises(KernelError, match="CUDA"):
            call()


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


LONG = [
    ("gate_up", lambda n: fp8.gated(meta(n, 2, dtype=torch.bfloat16))),
    ("gate_up", lambda n: fp8.gated(meta(n, 1, 2), splits=n)),
    ("rows must", lambda n: fp8.add_rmsnorm(meta(1, 2), None, meta(2), 1e-6, rows=meta(n, dtype=torch.int32))),
    ("add must", lambda n: fp8.add_rmsnorm(meta(1, 2), meta(n, 1, 2), meta(2), 1e-6, add_splits=n)),
    ("matrix", lambda n: fp8.quantize(meta(n, 2))),
    ("matrix", lambda n: fp8.add_rmsnorm(meta(n, 2), None, meta(2), 1e-6)),
    ("matrix", lambda n: fp8.gemm(meta(n, 16, dtype=E4M3), meta(n, 1), meta(8, 16, dtype=E4M3), meta(1, 1))),
    ("matrix", lambda n: fp8.gemm_gated(meta(2, 16, dtype=E4M3), meta(2, 1), meta(n, 16, dtype=E4M3), meta(n // 128, 1))),
]


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 5])
@pytest.mark.parametrize("text,call", LONG, ids=[f"{i}-{t.replace(' ', '_')}" for i, (t, _) in enumerate(LONG)])
def test_counts_past_31_bits_are_refused(text, call, n):
    """The launchers count in 32 bits: 2^32 + 5 rows would be five."""
    with pytest.raises(KernelError, match=text):
        call(n)
