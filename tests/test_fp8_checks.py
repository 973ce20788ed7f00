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
