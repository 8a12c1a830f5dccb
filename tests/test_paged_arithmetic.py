"""CPU: the whole-number arithmetic of the attention over pages, compiled for the host from the library's own header."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
#include "tship_internal.h"
#include <cstdio>
#include <cstring>
using namespace tship;
int main(int argc, char** argv)
{
    long long a, b;
    while (std::scanf("%lld %lld", &a, &b) == 2)
        if (!std::strcmp(argv[1], "first_key")) std::printf("%d\\n", first_key((int)a, (int)b));
        else if (!std::strcmp(argv[1], "quotient")) std::printf("%u\\n", FastDiv((uint32_t)b).quot((uint32_t)a));
        else return 1;
}
"""


@pytest.fixture(scope="module")
def compiled(tmp_path_factory):
    where = tmp_path_factory.mktemp("arithmetic")
    (where / "a.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-w", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-I" + os.path.join(ROOT, "tensorsharp_amd", "csrc"),
                    str(where / "a.cpp"), "-o", str(where / "a")], check=True)

    def run(name, pairs):
        text = "\n".join(f"{int(a)} {int(b)}" for a, b in pairs)
        out = subprocess.run([str(where / "a"), name], input=text, capture_output=True, text=True, check=True).stdout
        return [int(v) for v in out.split()]
    return run


def test_first_key_of_a_window(compiled):
    """max(0, p - window + 1) as whole numbers without a width, for positions in front of the sequence and windows up to the largest too"""
    edge = [0, 1, 2, 5, 127, 128, 129, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1]
    positions = edge + [-v for v in edge if v] + [-2 ** 31] + [int(v) for v in np.random.default_rng(0).integers(-2 ** 31, 2 ** 31, 50)]
    pairs = [(p, w) for p in positions for w in edge]
    for (p, w), got in zip(pairs, compiled("first_key", pairs)):
        assert got == (max(0, p - w + 1) if w else 0), (p, w, got)


def test_the_quotient_by_a_page_size_or_group(compiled):
    """the multiplication and shift that stand for it, for every dividend next to a multiple that it could miss"""
    rng = np.random.default_rng(0)
    divisors = [1, 2, 3, 5, 7, 16, 24, 100, 255, 256, 4095, 4096, 65537, 2 ** 30 - 1, 2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1] + [int(v) for v in rng.integers(1, 2 ** 31, 200)]
    pairs = []
    for d in divisors:
        near = np.arange(0, 2 ** 31, max(d, 2 ** 31 // 100), dtype=np.int64)[:150] // d * d
        pairs += [(int(n), d) for n in np.concatenate([near, near - 1, near + d - 1, rng.integers(0, 2 ** 31, 100), [0, 2 ** 31 - 1]]) if 0 <= n < 2 ** 31]
    assert compiled("quotient", pairs) == [n // d for n, d in pairs]


def test_a_window_of_more_than_32_bits_is_refused():
    """a call from C would take its lower bits: 2^32 + 5 as 5"""
    from tensorsharp_amd import HipBasicOps
    for window in (2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 31 - 1, -2 ** 32 + 7):
        with pytest.raises(ValueError, match="window below 2"):
            HipBasicOps.PagedAttention(None, None, None, None, None, 1.0, window=window)
