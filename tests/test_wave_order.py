"""CPU check of epilogues in which a wave's lanes exchange sums through LDS without a barrier of the workgroup: the compiler,
which sees one lane, has to be told to keep the writes and the other lanes' reads in order.

The kernels are compiled for the device to LLVM IR.  Behind the last barrier of a kernel no path may hold an LDS write
and an LDS read, in either order, without the wave's own barrier (which holds the fences) in between.
"""
import re
import subprocess

import pytest

from test_api_fake_hip import CSRC, ROOT

FP8 = """#include "fp8_wide.hpp"
namespace stx { namespace {
template __global__ void fp8_wide_kernel<WideShape<8, 2, 1, 4, 2, false>, false, false>(Fp8Args);
template __global__ void fp8_wide_kernel<WideShape<8, 4, 2, 4, 1, false>, true, false>(Fp8Args);
template __global__ void fp8_wide_kernel<WideShape<4, 4, 2, 4, 1, true>, true, false>(Fp8Args);
} }
"""
INT8 = '#include "int8_linear.hip"\n'
GEMM = """#include "gemm_wide.hpp"
namespace stx {
template __global__ void gemm_wide_kernel<4, 0, 256, false>(GemmArgs);
template __global__ void gemm_wide_kernel<4, 0, 128, false>(GemmArgs);
}
"""
BARRIER = re.compile(r"s_barrier|llvm\.amdgcn\.s\.barrier")


def kernels(tmp_path, source, name):
    """{kernel: lines} of the kernels called `name`."""
    hip, ir = tmp_path / "unit.hip", tmp_path / "unit.ll"
    hip.write_text(source)
    try:
        res = subprocess.run(["hipcc", "-O1", "-std=c++20", "-ffp-contract=off", f"-I{ROOT / 'include'}", f"-I{CSRC}",
                              "--offload-arch=gfx950", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                              "--cuda-device-only", "-S", "-emit-llvm", str(hip), "-o", str(ir)],
                             capture_output=True, text=True)
    except FileNotFoundError:
        pytest.skip("no hipcc")
    assert res.returncode == 0, res.stderr
    found = {}
    for body in re.findall(r"^define [^\n]*amdgpu_kernel [^\n]*\{\n.*?^\}", ir.read_text(), flags=re.M | re.S):
        kernel = re.search(r"@(\w+)", body).group(1)
        if name in kernel:
            found[kernel] = body.splitlines()[1:-1]
    return found


def blocks_of(lines):
    """{label: (lines, successors)}, in the order of the text; the first block's label is "entry"."""
    blocks, label = {"entry": ([], [])}, "entry"
    for line in lines:
        at = re.match(r"^([\w.]+):", line)
        if at:
            label = at.group(1)
            blocks[label] = ([], [])
            continue
        blocks[label][0].append(line)
        if re.match(r"\s+(br|switch) ", line) or line.strip().startswith("i32 "):
            blocks[label][1].extend(re.findall(r"label %([\w.]+)", line))
    return blocks


def unordered(lines):
    """(LDS accesses behind the last barrier, those of them that follow the other kind without the wave's barrier)."""
    blocks = blocks_of(lines)
    behind = [(label, i) for label, (body, _) in blocks.items() for i, line in enumerate(body) if BARRIER.search(line)]
    last, first = behind[-1]
    seen, todo, bad, count = {}, [(last, frozenset())], set(), set()
    while todo:
        label, since = todo.pop()
        start = first + 1 if label == last and not seen else 0
        if label in seen and since <= seen[label]:
            continue
        seen[label] = seen.get(label, frozenset()) | since
        since = set(seen[label])
        for line in blocks[label][0][start:]:
            if "llvm.amdgcn.wave.barrier" in line or BARRIER.search(line):
                since.clear()
                continue
            access = re.search(r"\b(store|load) .*ptr addrspace\(3\)", line)
            if access:
                kind = access.group(1)
                count.add((label, line))
                if {"store": "load", "load": "store"}[kind] in since:
                    bad.add((label, line.strip()))
                since.add(kind)
        for to in blocks[label][1]:
            todo.append((to, frozenset(since)))
    return len(count), sorted(bad)


@pytest.mark.parametrize("source,name,kinds", [(FP8, "fp8_wide_kernel", 3), (INT8, "int8_wide_kernel", 2),
                                               (GEMM, "gemm_wide_kernel", 2)], ids=["fp8_wide", "int8_wide", "gemm_wide"])
def test_lanes_meet_in_order(tmp_path, source, name, kinds):
    found = kernels(tmp_path, source, name)
    assert len(found) == kinds, sorted(found)
    for kernel, lines in found.items():
        count, bad = unordered(lines)
        assert count >= 16, (kernel, count)   # the exchange is there
        assert not bad, (kernel, len(bad), bad[:4])
