"""CPU checks of the e4m3 layers (include/strix_trellis_fp8.h) and the beam operators (include/strix_trellis_beam.h).

Their C layers are compiled unchanged against the fake HIP runtime, with fake launchers that check every buffer a
kernel would touch, and run under AddressSanitizer and UndefinedBehaviorSanitizer: argument checks, failure mapping,
leaks, plans that only launch, sizing.  The exports and the ctypes mirror are held to the headers.
"""
import ctypes as C
import os
import re
import subprocess

import pytest

from strix_trellis import abi
from test_api_fake_hip import CONTRACT, CSRC, HOST_SOURCES, ROOT, _clang

HEADERS = ("strix_trellis_fp8.h", "strix_trellis_beam.h")
SOURCES = ["ops_api.cpp", "ops_policy.cpp", "fp8_api.cpp", "fp8_policy.cpp", "beam_api.cpp", "beam_policy.cpp"]
FAKES = ["fake_hip.cpp", "fake_launch.cpp", "fake_ops_launch.cpp", "fake_blocks_launch.cpp", "blocks_main.cpp"]


@pytest.mark.parametrize("sanitize", [True, False], ids=["asan_ubsan", "plain"])
def test_contract_fake_hip(tmp_path, sanitize):
    cxx = _clang()
    if cxx is None:
        pytest.skip("no clang++ for the host-only contract build")
    exe = tmp_path / "blocks_contract"
    cmd = [cxx, "-std=c++20", "-O1", "-g", "-fno-omit-frame-pointer", "-ffp-contract=off", "-Wall", "-Wextra",
           "-Werror", f"-I{CONTRACT / 'fake'}", f"-I{CONTRACT}", f"-I{ROOT / 'include'}", f"-I{CSRC}"]
    if sanitize:
        cmd += ["-fsanitize=address,undefined", "-fno-sanitize-recover=undefined"]
    cmd += [str(CSRC / s) for s in HOST_SOURCES + SOURCES] + [str(CONTRACT / s) for s in FAKES]
    res = subprocess.run(cmd + ["-o", str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout + res.stderr
    env = dict(os.environ, ASAN_OPTIONS="detect_leaks=1:abort_on_error=0",
               UBSAN_OPTIONS="print_stacktrace=1:halt_on_error=1")
    res = subprocess.run([str(exe)], capture_output=True, text=True, env=env, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "checks passed" in res.stdout


def test_every_declared_operator_is_exported_and_mirrored():
    lib = abi.load()
    for header, count in zip(HEADERS, (8, 5)):
        text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / header).read_text(), flags=re.S)
        names = sorted(set(re.findall(r"\b(strix_amd_[a-z0-9_]+)\s*\(", text)))
        assert len(names) == count, names
        for name in names:
            assert hasattr(lib, name) and name in abi._PROTOTYPES, name


def test_struct_layouts_match_c_compiler(tmp_path):
    structs = {"strix_amd_fp8_weights_desc": abi.Fp8WeightsDesc, "strix_amd_fp8_linear_desc": abi.Fp8LinearDesc,
               "strix_amd_fp8_gated_desc": abi.Fp8GatedDesc, "strix_amd_beam_select_desc": abi.BeamSelectDesc,
               "strix_amd_states": abi.States, "strix_amd_beam_reorder_desc": abi.BeamReorderDesc}
    lines = ["#include <stdio.h>", "#include <stddef.h>"] + [f'#include "{h}"' for h in HEADERS] + ["int main(void){"]
    for name, ct in structs.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        for field, *_ in ct._fields_:
            lines.append(f'printf("{name}.{field} %zu\\n", offsetof({name}, {field}));')
    src, exe = tmp_path / "sizes.c", tmp_path / "sizes"
    src.write_text("\n".join(lines + ["return 0;}"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)],
                   check=True)
    got = dict(l.split() for l in subprocess.run([str(exe)], capture_output=True, text=True).stdout.splitlines())
    for name, ct in structs.items():
        assert int(got[name]) == C.sizeof(ct), name
        for field, *_ in ct._fields_:
            assert int(got[f"{name}.{field}"]) == getattr(ct, field).offset, (name, field)


def test_entry_points_refuse_without_a_context():
    lib = abi.load()
    bad = abi.STATUS_CODE["INVALID_ARGUMENT"]
    out = C.c_void_p(9)
    assert lib.strix_amd_fp8_weights_prepare(None, None, None, C.byref(out)) == bad and out.value is None
    assert lib.strix_amd_fp8_weights_destroy(None) == bad
    for name in ("fp8_linear", "fp8_gated", "beam_select", "beam_reorder"):
        out = C.c_void_p(9)
        assert getattr(lib, f"strix_amd_{name}")(None, None, None) == bad
        assert getattr(lib, f"strix_amd_{name}_plan_create")(None, None, None, C.byref(out)) == bad
        assert out.value is None
    for name in ("fp8_linear", "fp8_gated", "beam_select"):
        need = C.c_uint64(7)
        assert getattr(lib, f"strix_amd_{name}_workspace_bytes")(None, None, C.byref(need)) == bad and need.value == 0
