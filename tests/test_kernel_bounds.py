"""Loads through buffer resources have every byte of their way past the base in the
lane offset: the scalar offset is documented as left out of the bounds check, so a
load with one may read past its tensor (host logic, no GPU)."""
import os
import re
import shutil
import struct
import subprocess

import pytest

import mxfp4hip as M

MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(path):
    """The gfx950 code objects of a library, as the compiler bundled them."""
    with open(path, "rb") as f:
        data = f.read()
    at = data.find(MAGIC)
    while at >= 0:
        entry = at + len(MAGIC) + 8
        for _ in range(struct.unpack_from("<Q", data, at + len(MAGIC))[0]):
            off, size, name = struct.unpack_from("<QQQ", data, entry)
            if size and b"gfx950" in data[entry + 24:entry + 24 + name]:
                yield data[at + off:at + off + size]
            entry += 24 + name
        at = data.find(MAGIC, at + 1)


def test_buffer_loads_have_no_scalar_offset(tmp_path):
    objdump = shutil.which("llvm-objdump") or os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "llvm-objdump")
    if not os.path.exists(objdump):
        pytest.skip("llvm-objdump is not installed")
    loads, kernel, bad = 0, "", set()
    for i, code in enumerate(code_objects(M.LIB_PATH)):
        path = tmp_path / f"{i}.co"
        path.write_bytes(code)
        for line in subprocess.run([objdump, "-d", str(path)], capture_output=True, text=True, check=True).stdout.splitlines():
            if head := re.match(r"[0-9a-f]+ <(.+)>:", line):
                kernel = head[1]
            elif load := re.search(r"\bbuffer_load_\w+ v\w+(?:\[\S+\])?, s\[\S+\], (\S+)", line):
                loads += 1
                if load[1] != "0":
                    bad.add(kernel)
    assert loads > 100 and not bad
