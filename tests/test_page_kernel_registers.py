"""CPU: the kernels over lists of pages that test_four_bits_registers.py does not name spill no vector register and have no private memory either."""
import os

import pytest

from test_paged_registers import READELF, kernels


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
def test_no_kernel_over_lists_spills_vector_registers(tmp_path):
    counts = {"page_fill_kernel": 2, "page_drop_kernel": 1, "fork_tables_kernel": 1, "fork_rows_kernel": 1, "fork_store_kernel": 1, "compact_tables_kernel": 1}
    found = kernels(tmp_path)
    for name, count in counts.items():
        mine = {k: v for k, v in found.items() if name in k}
        assert len(mine) == count, (name, sorted(mine))
        for k, fields in mine.items():
            assert fields["vgpr_spill_count"] == 0 and fields["private_segment_fixed_size"] == 0, (k, fields)
