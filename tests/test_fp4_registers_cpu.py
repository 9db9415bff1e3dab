"""The compiler's report on the attention over 4-bit caches: no kernel keeps registers
in scratch memory, and as many work-groups fit a CU as the cut of the work counts on."""
from __future__ import annotations

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
    plain.test_work_groups_that_fit_a_compute_unit(reports, tmp_path)
