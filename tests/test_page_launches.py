"""CPU: what the calls for the life of pages launch at the sizes that they take at most, on a HIP runtime without a device (see test_launches.py).  A
launch has fewer than 2^32 threads in each dimension and at most 65535 workgroups in the second and third: the runtime refuses others, and the call would
fail behind a first launch that has listed its moves."""
import pytest

from test_launches import launches, stub  # noqa: F401
from test_page_refusals import SETUP

WIDE = "max_pages=1 << 30, table_stride=1 << 30, page_size=1"
CALLS = ["do_%s(pool(%s%s%s))" % (call, sizes, seqs, pages) for call in ("resize", "fork", "compact") for sizes in (WIDE, "max_pages=1 << 26, table_stride=1 << 26, page_size=16",
                                                                                                                  "max_pages=(1 << 26) - 16, table_stride=1 << 26, page_size=16", "max_pages=5000, table_stride=5000")
         for seqs in ("", ", num_seqs=1", ", num_seqs=1024", ", num_seqs=1025", ", num_seqs=65535") for pages in ("", ", num_pages=1 << 28")]
CALLS += ["do_copy(count=1 << 20)", "do_compact(room=(1 << 31) - 1)", "do_fork(count=(1 << 31) - 1)"]


def test_no_launch_is_larger_than_the_runtime_takes(stub):  # noqa: F811
    for call, (ok, error, log) in zip(CALLS, stub(SETUP, calls=CALLS)):
        found = launches(log, "kernel")
        assert ok == 1 and found, (call, error)
        for _, name, x, y, z, threads, lds in found:
            assert 0 < int(x) * int(threads) < 2 ** 32 and 0 < int(y) < 65536 and 0 < int(z) < 65536 and int(lds) <= 160 * 1024, (call, name, x, y, z)


def test_which_kernels_a_fork_takes(stub):  # noqa: F811
    """the tables' kernel for 16 entries a workgroup, but for rows so long that it would be too many of them"""
    calls = ["do_fork(pool(%s, num_seqs=%d))" % (sizes, seqs) for sizes in ("max_pages=9000, table_stride=9000", "max_pages=1 << 26, table_stride=1 << 26, page_size=16", WIDE)
             for seqs in (2, 1024)]
    got = [["".join(k for k in ("plan", "tables", "rows", "store") if "fork_%s_kernel" % k in l[1]) for l in launches(log, "kernel")] for _, _, log in stub(SETUP, calls=calls)]
    assert got == [["plan", "tables"]] * 2 + [["plan", "rows", "store"]] * 4
