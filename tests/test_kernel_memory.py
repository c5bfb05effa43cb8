"""What the compiler put into scratch memory, from the built library's own metadata (no GPU)."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from rhizome_amd import _abi

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(blob):
    """The gfx950 code objects of every offload bundle in a library."""
    at = blob.find(MAGIC)
    while at >= 0:
        p = at + len(MAGIC) + 8
        for _ in range(struct.unpack_from("<Q", blob, at + len(MAGIC))[0]):
            offset, size, name = struct.unpack_from("<QQQ", blob, p)
            if b"gfx950" in blob[p + 24:p + 24 + name] and size:
                yield blob[at + offset:at + offset + size]
            p += 24 + name
        at = blob.find(MAGIC, at + 1)


def test_no_kernel_keeps_an_array_in_scratch(tmp_path):
    """An array in registers that is indexed at run time goes to memory whole, without counting as spilled."""
    readelf = shutil.which("llvm-readelf", path=os.pathsep.join([os.environ.get("PATH", ""), "/opt/rocm/llvm/bin"]))
    if readelf is None:
        pytest.skip("no llvm-readelf")
    kernels = 0
    for i, code in enumerate(code_objects(open(_abi.LIB_PATH, "rb").read())):
        path = tmp_path / f"{i}.elf"
        path.write_bytes(code)
        notes = subprocess.run([readelf, "--notes", str(path)], capture_output=True, text=True, check=True).stdout
        for kernel in notes.split(".agpr_count:")[1:]:
            field = {name: re.search(rf"\.{name}:\s+(\S+)", kernel).group(1)
                     for name in ("name", "private_segment_fixed_size", "vgpr_spill_count")}
            kernels += 1
            spilled = 4 * int(field["vgpr_spill_count"])
            assert int(field["private_segment_fixed_size"]) <= spilled + 4, field
    assert kernels > 100, "the library's kernels"
