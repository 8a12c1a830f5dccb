"""CPU: what the built library says of its own kernels' registers.  A vector operand of the attention over pages that the compiler spilled was once
brought back with one of its four registers missing, so no instantiation may spill any."""
import os
import re
import struct
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
READELF = "/opt/rocm/llvm/bin/llvm-readelf"


def kernels(tmp_path):
    """{mangled name: {field: number}} of every kernel in the library, from the notes of its code objects"""
    with open(os.path.join(ROOT, "tensorsharp_amd", "libTsHipOps.so"), "rb") as f:
        data = f.read()
    out, at = {}, data.find(b"__CLANG_OFFLOAD_BUNDLE__")
    while at >= 0:
        entry = at + 32
        for _ in range(struct.unpack_from("<Q", data, at + 24)[0]):
            offset, size, length = struct.unpack_from("<QQQ", data, entry)
            name = data[entry + 24:entry + 24 + length]
            entry += 24 + length
            if size and b"gfx950" in name:
                path = tmp_path / f"{at}.elf"
                path.write_bytes(data[at + offset:at + offset + size])
                notes = subprocess.run([READELF, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
                for text in re.split(r"\n  - \.", notes)[1:]:
                    found = re.search(r"\.name:\s+(\S+)", text)
                    if found:
                        out[found.group(1)] = {k: int(v) for k, v in re.findall(r"\.(\w+):\s+(\d+)\s*$", text, re.M)}
        at = data.find(b"__CLANG_OFFLOAD_BUNDLE__", at + 1)
    return out


@pytest.mark.skipif(not os.path.exists(READELF), reason="no llvm-readelf")
def test_the_attention_over_pages_spills_no_vector_registers(tmp_path):
    found = {k: v for k, v in kernels(tmp_path).items() if "paged_attention_kernel" in k or "paged_combine_kernel" in k}
    assert len(found) == 3 * 5 + 2, sorted(found)
    for name, fields in found.items():
        assert fields["vgpr_spill_count"] == 0 and fields["private_segment_fixed_size"] == 0, (name, fields)
