"""CPU check of the e4m3 scales' quotients: the steps that the kernels take (csrc/fp8_scale.hpp) end on the rounded quotient for
every mantissa, from every reciprocal that is at most a unit off."""
import subprocess

import pytest

from test_api_fake_hip import CONTRACT, CSRC, _clang


def test_every_mantissa(tmp_path):
    cxx = _clang()
    if cxx is None:
        pytest.skip("no clang++ for host-only builds")
    exe = tmp_path / "fp8_scale"
    res = subprocess.run([cxx, "-std=c++20", "-O2", "-ffp-contract=off", "-Wall", "-Wextra", "-Werror", f"-I{CSRC}",
                          str(CONTRACT / "fp8_scale_main.cpp"), "-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "all mantissas passed" in res.stdout, res.stdout + res.stderr
