"""What bench.py divides by."""
import pytest

import bench


def test_a_prefill_in_8_bits_is_held_to_the_8_bit_rate():
    """3 TFLOP in the layers' matrices and 1 elsewhere, in 2 ms beside a bf16 peak of 4,000 TFLOP/s."""
    assert bench.prefill_fraction(3e12, 1e12, 2.0, 4000.0, False) == pytest.approx(0.5)
    assert bench.prefill_fraction(3e12, 1e12, 2.0, 4000.0, True) == pytest.approx(2.5 / 8)
    # at the 8-bit rate itself the fraction is one
    assert bench.prefill_fraction(8e12, 0.0, 1.0, 4000.0, True) == pytest.approx(1.0)


def test_a_design_is_not_measured_in_bfloat16_when_8_bits_were_asked_for(monkeypatch, capsys):
    monkeypatch.setattr("sys.argv", ["bench.py", "--design", "bozosun", "--gemm", "fp8"])
    monkeypatch.setattr(bench, "design_bench", lambda args: pytest.fail("measured all the same"))
    assert bench.main() == 2 and "--gemm does not go with it" in capsys.readouterr().out
