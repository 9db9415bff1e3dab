"""The compiler's own report on the kernels of the attention over the paged cache:
none keeps registers in scratch memory, where each key's tile would fetch them, and
as many work-groups fit a CU as the cut of the work counts on."""
from __future__ import annotations

import concurrent.futures
import ctypes
import re
import shutil
import subprocess

import pytest

from fireprot_amd import build

SOURCES = ("paged_attention_plain", "paged_attention_fp8", "paged_attention_int8")


def report(source):
    """{mangled kernel: (registers, bytes of scratch a lane, registers spilled)}."""
    cmd = [build._hipcc(), *build.HIPCC_FLAGS, "-I", str(build.INCLUDE), "-I", str(build.CSRC),
           "--cuda-device-only", "-S", str(build.CSRC / f"{source}.hip"), "-o", "/dev/null",
           "-Rpass-analysis=kernel-resource-usage"]
    text = subprocess.run(cmd, capture_output=True, text=True, check=True).stderr
    found = re.findall(r"Function Name: (\S+).*?VGPRs: (\d+).*?ScratchSize \[bytes/lane\]: (\d+)"
                       r".*?VGPRs Spill: (\d+)", text, re.S)
    return {name: tuple(map(int, numbers)) for name, *numbers in found}


@pytest.fixture(scope="module")
def reports():
    try:
        build._hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        return list(pool.map(report, SOURCES))


def test_no_kernel_spills(reports):
    # three plain types, three query types over each 8-bit type; 32, 64 and 128
    # channels with one and two query tiles, 256 with one
    assert [len(r) for r in reports] == [21, 21, 21]
    for kernels in reports:
        for name, (registers, scratch, spilled) in kernels.items():
            assert (scratch, spilled) == (0, 0), (name, registers, scratch, spilled)


def test_work_groups_that_fit_a_compute_unit(reports, tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    (tmp_path / "shim.cpp").write_text(
        '#include "paged_layout.hpp"\n'
        'extern "C" int groups(int split, int dim, int tiles) {\n'
        "  return fpx::resident_groups(split, dim, tiles);\n}\n")
    subprocess.run([gxx, "-std=c++17", "-shared", "-fPIC", "-I", str(build.CSRC),
                    str(tmp_path / "shim.cpp"), "-o", str(tmp_path / "shim.so")], check=True)
    rule = ctypes.CDLL(str(tmp_path / "shim.so")).groups
    for kernels in reports:
        for name, (registers, _, _) in kernels.items():
            query, coded, dim, tiles = re.search(
                r"paged_attention_kernelI(f|DF16b|DF16_).*?(Cache)?E?Li(\d+)ELi(\d)E", name).groups()
            # a wave of each work-group on every SIMD, of 512 registers in steps of 8
            fit = 512 // (-(-registers // 8) * 8)
            split = coded is not None and query != "DF16b"
            assert fit >= rule(split, int(dim), int(tiles)), (name, registers)
