"""The compiled step of the 8-bit linear layers' faces beside the rest of Python: its lock, its errors."""
import ctypes
import subprocess
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"

# launchers that wait, for two seconds at most, until another thread has called open_gate
SLOW = """
#include <atomic>
#include <chrono>
#include <thread>
static std::atomic<int> gate{0};
static int waited() {
    for (int i = 0; i < 2000 && !gate.load(); ++i) std::this_thread::sleep_for(std::chrono::milliseconds(1));
    return gate.exchange(0) ? 0 : 1;
}
extern "C" void open_gate() { gate.store(1); }
extern "C" int slow_quantize(const void*, int, long long, void*, float*, int, int, int, void*) { return waited(); }
extern "C" int slow_norm(const float*, const void*, int, int, long long, const float*, float, const int*, int, int, int, float*, void*, float*, void*) { return waited(); }
extern "C" int slow_gated(const void*, int, int, long long, void*, float*, int, int, const float*, void*) { return waited(); }
extern "C" int slow_gemm(const void*, const float*, const void*, const float*, void*, int, int, int, int, int, int, float*, int, int*, void*) { return waited(); }
"""


@pytest.fixture
def slow(tmp_path):
    """The compiled step with launchers that wait for another thread; the real ones are put back."""
    from purhie_b200.csrc import fp8, ops
    (tmp_path / "slow.cpp").write_text(SLOW)
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-pthread", "-o", str(tmp_path / "slow.so"), str(tmp_path / "slow.cpp")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "slow.so"))
    step = fp8._calls or fp8._load_calls()
    address = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
    step.set_launchers(address(lib.slow_quantize), address(lib.slow_norm), address(lib.slow_gated), address(ops._fn("fp8", "ph_gemm_fp8_plan")[0]),
                       address(lib.slow_gemm))
    yield lib
    fp8._load_calls()


def test_a_launch_that_waits_lets_other_threads_run(slow):
    from purhie_b200.csrc import fp8
    x, w = torch.zeros(4, 256, device=DEV), torch.ones(256, device=DEV)
    q, s = torch.zeros(4, 256, device=DEV).to(torch.float8_e4m3fn), torch.ones(4, 2, device=DEV)
    for call in (lambda: fp8.quantize(x), lambda: fp8.add_rmsnorm(x, None, w, 1e-6), lambda: fp8.gated(x), lambda: fp8.gemm(q, s, q, s[:1])):
        timer = threading.Timer(0.05, slow.open_gate)
        timer.start()
        call()                                               # (a launcher that has waited for nothing gives a status, which raises)
        timer.join()


def test_no_memory_is_torch_s_error():
    """Where an output does not fit, the caller gets what every torch call would raise."""
    from purhie_b200.csrc import fp8
    x = torch.zeros(1 << 14, 1 << 13, dtype=torch.bfloat16, device=DEV)
    rows, ones = torch.zeros(1 << 14, 1 << 12, device=DEV), torch.ones(1 << 12, device=DEV)
    q, s = fp8.quantize(x)
    w, ws = fp8.quantize(x, block_rows=128)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    try:
        # room for 8 MiB more; the smallest output below is 64
        torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (8 << 20)) / total)
        for call in (lambda: fp8.quantize(x), lambda: fp8.gated(x), lambda: fp8.add_rmsnorm(rows, None, ones, 1e-6), lambda: fp8.gemm(q, s, w, ws)):
            with pytest.raises(torch.OutOfMemoryError):
                call()
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert fp8.gemm(q[:8], s[:8], w, ws).shape == (8, 1 << 14)
