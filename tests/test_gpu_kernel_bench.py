"""The throughput entries of the quantised cache, the 4-bit attention and the GEMM with epilogue run and name their floors."""
import pytest

pytestmark = pytest.mark.gpu


def test_operator_entries(cuda_device):
    import kernel_bench
    peaks = {"hbm_gbs": 6650.0, "bf16_tflops": 1590.0, "note": "of fallback"}
    entries = kernel_bench.operators(cuda_device, 0, 1, peaks, most_bytes=60_000_000)
    assert {e["kernel"] for e in entries} == {"write", "read", "attn", "gemm"}
    for e in entries:
        assert e["ms"] > 0 and 0 < e["floor_ms"] and e["frac_of_peak"] == pytest.approx(e["floor_ms"] / e["ms"])
