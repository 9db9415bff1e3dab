"""The compiler's report on the attention over 4-bit caches: no kernel keeps registers
in scratch memory, and as many work-groups fit a CU as the cut of the work counts on."""
from __future__ import annotations

import ctypes
import re
import shutil
import subprocess

import pytest

from fireprot_amd import build
from tests import test_paged_registers_cpu as plain


@pytest.fixture(scope="module")
def reports():
    try:
        build._hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    return [plain.report("paged_attention_fp4")]


def test_no_kernel_spills(reports):
    # three query types; four widths with one query tile, of one and two columns a query,
    # 32, 64 and 128 channels with two
    assert len(reports[0]) == 3 * (4 * 2 + 3)
    for name, (registers, scratch, spilled) in reports[0].items():
        assert (scratch, spilled) == (0, 0), (name, registers, scratch, spilled)


def test_work_groups_that_fit_a_compute_unit(reports, tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    (tmp_path / "shim.cpp").write_text(
        '#include "paged_layout.hpp"\n'
        'extern "C" int groups(int f32, int split, int dim, int tiles, int columns) {\n'
        "  return fpx::resident_groups4(f32, split, dim, tiles, columns == 2);\n}\n")
    subprocess.run([gxx, "-std=c++17", "-shared", "-fPIC", "-I", str(build.CSRC),
                    str(tmp_path / "shim.cpp"), "-o", str(tmp_path / "shim.so")], check=True)
    rule = ctypes.CDLL(str(tmp_path / "shim.so")).groups
    for name, (registers, _, _) in reports[0].items():
        query, dim, tiles, columns = re.search(
            r"paged_attention_kernelI(f|DF16b|DF16_).*?Li(\d+)ELi(\d)ELi(\d)E", name).groups()
        # a wave of each work-group on every SIMD, of 512 registers in steps of 8
        fit = 512 // (-(-registers // 8) * 8)
        wanted = rule(query == "f", query != "DF16b", int(dim), int(tiles), int(columns))
        assert fit >= wanted, (name, registers)
