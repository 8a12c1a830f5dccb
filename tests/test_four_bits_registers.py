"""CPU: no kernel over caches in four bits, over first positions or over lists of pages spills a vector register (see test_paged_registers.py)."""
import os

import pytest

from test_paged_registers import READELF, kernels


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
def test_no_kernel_spills_vector_registers(tmp_path):
    counts = {"paged_mx_attention_kernel": 5, "paged_first_attention_kernel": 15, "paged_combine_dealt_kernel": 2, "rope_store_mx_kernel": 4, "copy_pages_kernel": 16,
              "page_plan_kernel": 1, "fork_plan_kernel": 3, "compact_plan_kernel": 2, "page_few_kernel": 1}
    found = kernels(tmp_path)
    for name, count in counts.items():
        mine = {k: v for k, v in found.items() if name in k}
        assert len(mine) == count, (name, sorted(mine))
        for k, fields in mine.items():
            assert fields["vgpr_spill_count"] == 0 and fields["private_segment_fixed_size"] == 0, (k, fields)
