"""The paged attention kernels read LDS without waiting for copies in flight.

As tests/test_lds_waits.py, for paged_attention.hip: compiled to gfx950
assembly (no GPU needed), no compiler-emitted vmcnt wait stands directly before
an LDS read, and no kernel of it spills to scratch (a spill's reload would wait
for the copies too).
"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from ane_amd.build import HIP_FLAGS, hipcc
from tests.test_lds_waits import lds_read_waits

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("hipcc") is None and not Path("/opt/rocm/bin/hipcc").exists(),
                    reason="hipcc not available")
def test_no_wait_for_copies_and_no_spills(tmp_path):
    flags = [f for f in HIP_FLAGS if f != "-fPIC"]
    out = tmp_path / "paged_attention.s"
    subprocess.run([hipcc(), *flags, "--cuda-device-only", "-S", str(ROOT / "ane_amd" / "csrc" / "paged_attention.hip"),
                    "-o", str(out)], check=True, capture_output=True)
    asm = out.read_text()
    waits = lds_read_waits(asm)
    assert sum("k_attn" in k for k in waits) >= 16
    assert not {k: n for k, n in waits.items() if n}
    assert set(re.findall(r"; ScratchSize: (\d+)", asm)) == {"0"}


def test_multiplied_division_is_exact():
    """x / d as (x * magic) >> shift, the form the kernels use for page, token and
    row-tile numbers: every d it is used with, at and around multiples of d up to
    2^30, where a wrong magic shows first."""
    for d in list(range(1, 4097)) + [5000, 9999, 32768, 40000, 65535, 65536]:
        lg = (d - 1).bit_length()
        magic, shift = -(-(1 << (30 + lg)) // d), 30 + lg
        assert magic < 1 << 32
        for q in (0, 1, 2, 3, (1 << 29) // d, ((1 << 30) - 1) // d):
            for x in (q * d - 1, q * d, q * d + 1, q * d + d - 1):
                if 0 <= x < 1 << 30:
                    assert (x * magic) >> shift == x // d
                    assert x * magic < 1 << 64
