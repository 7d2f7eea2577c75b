"""Kernels that may be resident before their producer ends (programmatic dependent launch) read its output by ordinary loads: the
read-only path asks that data stay constant for the kernel's whole life, which begins before griddepcontrol.wait."""
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "tilelang-tpu_b200" / "csrc"


@pytest.mark.parametrize("name", ["attn_int4.cu", "kv_cache.cu", "gemm_epilogue.cu"])
def test_no_read_only_loads(name):
    code = re.sub(r"//[^\n]*", "", (CSRC / name).read_text())
    assert not re.findall(r"__ldg\s*\(|ld\.global\.nc|ld_stream|ld_cached|mla_len\s*\(", code)
