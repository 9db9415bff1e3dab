"""The compiler's own report on the kernels of the attention over the paged cache:
none keeps registers in scratch memory, where each key's tile would fetch them."""
from __future__ import annotations

import concurrent.futures
import re
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


def test_no_kernel_spills():
    try:
        build._hipcc()
    except RuntimeError:
        pytest.skip("no hipcc")
    with concurrent.futures.ThreadPoolExecutor(len(SOURCES)) as pool:
        reports = list(pool.map(report, SOURCES))
    # three plain types, three query types over each 8-bit type; 32, 64 and 128
    # channels with one and two query tiles, 256 with one
    assert [len(r) for r in reports] == [21, 21, 21]
    for kernels in reports:
        for name, (registers, scratch, spilled) in kernels.items():
            assert (scratch, spilled) == (0, 0), (name, registers, scratch, spilled)
