"""CPU: the scratch memory that sampling takes of a stream, on a HIP runtime without a device (see test_launches.py)."""
import pytest

from test_launches import launches, stub  # noqa: F401

CALL = """
a = space(64)
p = C.c_void_p(a.ctypes.data)
ok = L.TSHip_SampleTokensF32Device(N.TensorView2D(a.ctypes.data, rows, vocab, vocab, 1, rows * vocab * 4), p, p, None, None, None, p, None)
out.append([ok, L.TSHip_GetLastError().decode(), log()])
"""


@pytest.mark.parametrize("rows,vocab", [(1, 1), (1, 1 << 20), (64, 128256), (256, 128256), (500, 50000), (5000, 1000), (65535, 1), (65535, 512), (70000, 64), (200000, 300),
                                        (4000, 4097), (3000, 1 << 20)])
def test_the_scratch_of_a_call_stays_below_320_mib(stub, rows, vocab):  # noqa: F811
    """(and the quarter that a stream's workspace has to spare); every row is in one launch of each kernel"""
    ((ok, error, log),) = stub(CALL, rows=rows, vocab=vocab)
    assert ok == 1, error
    assert max(int(l[1]) for l in log if l[0] == "malloc") <= (5 << 26) * 5 / 4
    draws = launches(log, "sample_draw_kernel")
    assert sum(int(l[2]) for l in draws) == rows
    assert len(launches(log, "sample_top_kernel")) == len(launches(log, "sample_sums_kernel")) == len(draws)
    if rows * vocab <= 256 * 128256 and rows <= 4096:
        assert len(draws) == 1
