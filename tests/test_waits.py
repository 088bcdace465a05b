"""Wait states that the hardware leaves to the program, in the machine code of the kernels as they were built."""
import os
import re
import shutil
import struct
import subprocess

import pytest

from conftest import REPO

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(path):
    """The gfx950 code objects in the bundles that a library holds."""
    with open(path, "rb") as f:
        data = f.read()
    at = data.find(MAGIC)
    while at >= 0:
        n, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(n):
            off, size, name = struct.unpack_from("<QQQ", data, p)
            if data[p + 24:p + 24 + name].decode().endswith("gfx950"):
                yield data[at + off:at + off + size]
            p += 24 + name
        at = data.find(MAGIC, at + 1)


def test_loads_to_lds_wait_for_m0(tmp_path):
    """One wait state lies between a scalar write of m0 and a load from memory to LDS that takes its address from there: the
    compiler puts it where it makes such code itself, inline assembly has its own."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    loads, bad = 0, []
    for i, code in enumerate(code_objects(os.path.join(REPO, "nemo-c_amd", "libnemoasr_hip.so"))):
        (tmp_path / f"{i}.o").write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(tmp_path / f"{i}.o")], capture_output=True, text=True, check=True).stdout
        kernel = before = ""
        for line in text.splitlines():
            if line.endswith(">:"):
                kernel = line
            if "_load_lds_" in line:
                loads += 1
                if re.match(r"\s*s_\w+ m0,", before):
                    bad.append((kernel, before.split("//")[0].strip(), line.split("//")[0].strip()))
            before = line
    assert loads and not bad, (loads, len(bad), bad[:5])
