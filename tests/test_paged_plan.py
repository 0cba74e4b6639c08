"""The host's side of paged attention (ane_amd/csrc/paged_plan.hpp), compiled and
run as it is: no GPU needed."""
import shutil
import subprocess
from pathlib import Path

import pytest

from ane_amd.build import HIP_FLAGS, hipcc

ROOT = Path(__file__).resolve().parents[1]
SOURCE = r"""
#include <stdio.h>
#include "paged_plan.hpp"
using namespace ane;

// x / d by Div for every d of a cache, at and around multiples of d up to 2^30, where a
// wrong magic or shift shows first
static uint64_t wrong_quotients() {
    uint64_t bad = 0;
    auto sweep = [&](uint32_t d) {
        const Div by = div_by(d);
        const uint64_t top = (1ull << 30) - 1, qs[] = {0, 1, 2, 3, (1ull << 29) / d, top / d / 2, top / d - 1, top / d};
        for (uint64_t q : qs)
            for (int64_t x : {(int64_t)(q * d) - 1, (int64_t)(q * d), (int64_t)(q * d) + 1, (int64_t)(q * d + d) - 1, (int64_t)top})
                if (x >= 0 && x <= (int64_t)top) bad += by((uint32_t)x) != (uint32_t)x / d;
    };
    for (uint32_t d = 1; d <= 4096; d++) sweep(d);
    for (uint32_t d = 4097; d <= 65536; d += 1 + d / 997) sweep(d);
    for (uint32_t lg = 12; lg <= 16; lg++) sweep((1u << lg) - 1), sweep(1u << lg);
    return bad;
}

int main(int argc, char**) {
    if (argc == 1) return printf("%llu\n", (unsigned long long)wrong_quotients()), 0;
    ane_paged_cache c = {};
    uint32_t n, groups, max_prefix, max_len;
    c.page_size = 16;
    while (scanf("%u %u %u %u %u %u %u %u", &c.n_heads, &c.n_kv_heads, &c.head_dim, &c.max_pages, &n, &groups, &max_prefix,
                 &max_len) == 8)
        printf("%d\n", (int)shared_plan(&c, n, groups, max_prefix, max_len).each);
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("hipcc") is None and not Path("/opt/rocm/bin/hipcc").exists():
        pytest.skip("hipcc not available")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.hip").write_text(SOURCE)
    subprocess.run([hipcc(), *HIP_FLAGS, "--offload-host-only", "-I", str(ROOT / "ane_amd" / "csrc"), str(d / "plan.hip"), "-o",
                    str(d / "plan")], check=True, capture_output=True)
    return d / "plan"


def test_multiplied_division(program):
    """Page, token and row-tile numbers, as the kernels work them out."""
    got = subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout
    assert int(got) == 0


@pytest.mark.parametrize("n,groups,max_prefix,max_len,each", [
    (128, 0, 0, 512, True), (512, 0, 0, 100, True), (127, 0, 0, 100, False),  # 1024 (token, kv head) pairs and more
    (128, 0, 0, 513, False), (128, 0, 512, 1000, False),  # no groups, no prefix
    (128, 1, 400, 512, True), (128, 1, 488, 1000, True), (128, 1, 487, 1000, False), (128, 1, 1024, 1536, True),
    # a row in no group, or in one with a shorter prefix, may have max_len keys of its own
    (128, 1, 1025, 1537, False), (128, 1, 8192, 8192, False), (128, 1, 8000, 8300, False), (140, 3, 2000, 2200, False),
    # no bound on the prefixes, none at all
    (128, 1, 0, 4000, False), (128, 1, 0, 500, True), (128, 1, 0, 0, False)])
def test_a_wave_a_row_only_where_no_row_can_be_long(program, n, groups, max_prefix, max_len, each):
    got = subprocess.run([str(program), "plan"], input=f"32 8 128 1024 {n} {groups} {max_prefix} {max_len}\n", check=True,
                         capture_output=True, text=True).stdout
    assert bool(int(got)) is each
