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


@pytest.fixture(scope="module")
def loads(tmp_path_factory):
    """(kernel, the instructions before, the load) of every load to LDS, of the library as it was built."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no disassembler")
    d, out = tmp_path_factory.mktemp("code"), []
    for i, code in enumerate(code_objects(os.path.join(REPO, "nemo-c_amd", "libnemoasr_hip.so"))):
        (d / f"{i}.o").write_bytes(code)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(d / f"{i}.o")], capture_output=True, text=True, check=True).stdout
        lines, kernel = text.splitlines(), ""
        for n, line in enumerate(lines):
            if line.endswith(">:"):
                kernel, begin = line, n + 1
            elif "_load_lds_" in line:
                out.append((kernel, *([x.split("//")[0].strip() for x in part] for part in (lines[max(begin, n - 6):n], [line]))))
    assert out
    return [(kernel, before, load[0]) for kernel, before, load in out]


def test_loads_to_lds_wait_for_m0(loads):
    """One wait state lies between a scalar write of m0 and a load from memory to LDS that takes its address from there: the
    compiler puts it where it makes such code itself, inline assembly has its own."""
    bad = [x for x in loads if x[1] and re.match(r"s_\w+ m0,", x[1][-1])]
    assert not bad, (len(loads), len(bad), bad[:5])


def test_loads_to_lds_wait_for_their_base(loads):
    """Five wait states lie between a vector instruction that writes a scalar register and a load that has its base there; the
    compiler does not see to it for a load in an assembly block."""
    bad = []
    for kernel, before, load in loads:
        base = re.search(r", s\[(\d+):(\d+)\]", load)
        need = set(range(int(base.group(1)), int(base.group(2)) + 1)) if base else set()
        states = 0
        for x in reversed(before):
            to = re.match(r"([vs])_\w+ s(?:\[(\d+):(\d+)\]|(\d+))", x)
            if to:
                writes = {int(to.group(4))} if to.group(4) else set(range(int(to.group(2)), int(to.group(3)) + 1))
                if to.group(1) == "v" and writes & need and states < 5:
                    bad.append((kernel, x, load))
                need -= writes
            nop = re.match(r"s_nop (\w+)", x)
            states += int(nop.group(1), 0) + 1 if nop else 1
    assert not bad, (len(loads), len(bad), bad[:5])
