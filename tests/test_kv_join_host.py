"""Launches of the join of shared attention's parts, without a GPU: up to 2^26 query
rows are joined whatever the value dims, by launches of fewer than 2^32 threads."""
import os
import subprocess

import pytest

from tests.test_kv_cache_launches import COMPILER, CSRC, HIP_INCLUDE

PROGRAM = r"""
#include "kv.hpp"
#include <cstdio>
int main() {
    const uint32_t workgroup = 256;
    for (uint32_t vdim = 1; vdim <= 256; ++vdim)
        for (uint64_t rows : {uint64_t{1}, uint64_t{12345}, uint64_t{1} << 25, (uint64_t{1} << 26) - 3, uint64_t{1} << 26}) {
            const uint64_t threads = (vdim + 3) / 4;
            uint64_t joined = 0, launches = 0;
            while (joined < rows) {
                const uint64_t most = icsdk::kv::join_rows(vdim), now = rows - joined < most ? rows - joined : most;
                if (now == 0 || now * threads + workgroup - 1 >= uint64_t{1} << 32) return std::printf("%u\n", vdim), 1;
                joined += now;
                ++launches;
            }
            if (launches > 2) return std::printf("%u launches\n", (unsigned)launches), 1;
        }
    return 0;
}
"""


@pytest.mark.skipif(not os.path.exists(COMPILER), reason="no HIP compiler")
def test_launches_of_the_join(tmp_path):
    source = tmp_path / "join.cpp"
    source.write_text(PROGRAM)
    binary = tmp_path / "join"
    subprocess.run([COMPILER, "-std=c++17", "-O1", "-D__HIP_PLATFORM_AMD__", "-I" + CSRC,
                    "-I" + os.path.join(CSRC, "..", "..", "include"), "-I" + HIP_INCLUDE, str(source), "-o", str(binary)],
                   check=True, capture_output=True)
    done = subprocess.run([str(binary)], capture_output=True, text=True, timeout=60)
    assert done.returncode == 0, done.stdout
