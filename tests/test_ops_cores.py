"""The calls of tests/int8_cores.py reach the cores that they are listed for: csrc/ops_policy.cpp, compiled as it is
for the host, is asked for each, so that a change of its rule cannot leave a core untested."""
import subprocess

import pytest

from int8_cores import CALLS, CORES
from test_api_fake_hip import CONTRACT, CSRC, ROOT, _clang

PROGRAM = """#include "ops.hpp"
#include <cstdio>
int main() {
    unsigned long long rows;
    unsigned input, output;
    while (std::scanf("%llu %u %u", &rows, &input, &output) == 3)
        std::printf("%u %u\\n", unsigned(stx::int8_plan(rows, input, output).core), stx::int8_k_blocks(input));
}
"""


def test_every_core_is_reached(tmp_path):
    cxx = _clang()
    if cxx is None:
        pytest.skip("no clang++ for the host build")
    src, exe = tmp_path / "plan.cpp", tmp_path / "plan"
    src.write_text(PROGRAM)
    subprocess.run([cxx, "-std=c++20", f"-I{CONTRACT / 'fake'}", f"-I{CONTRACT}", f"-I{ROOT / 'include'}", f"-I{CSRC}",
                    str(src), str(CSRC / "ops_policy.cpp"), "-o", str(exe)], check=True)
    asked = "\n".join(f"{rows} {I} {N}" for _, rows, I, N in CALLS)
    out = subprocess.run([str(exe)], input=asked, capture_output=True, text=True, check=True).stdout.split("\n")
    got = [tuple(map(int, line.split())) for line in out if line]
    assert len(got) == len(CALLS)
    for (core, *call), (index, _) in zip(CALLS, got):
        assert CORES[index] == core, (call, CORES[index])
    assert {c for c, *_ in CALLS} == set(CORES)
    # each core also runs a long sum whose eighths differ by a block
    for core in CORES:
        blocks = [k for (c, *_), (_, k) in zip(CALLS, got) if c == core]
        assert any(k >= 64 and k % 8 for k in blocks), (core, blocks)
