"""The built library's device code as text: kernels and their instructions, from the
disassembler of the toolchain that built it."""

import os
import re
import shutil
import subprocess

import pytest

from xpu_kernels.int8 import _lib as L

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")


class Op(tuple):
    """(mnemonic, [operand]) with the instruction's address, and where it may branch to."""
    at, target = 0, None


def kernels(directory, wanted):
    """{symbol: [Op]} of the kernels whose symbol contains one of ``wanted``;
    ``directory`` takes the library's code objects."""
    objdump = os.path.join(LLVM, "llvm-objdump")
    if not os.path.exists(objdump):
        pytest.skip("no llvm-objdump in " + LLVM)
    path = L.library_path()
    assert path is not None, "libxpuint8.so is not built (run __graft_entry__.build())"
    copy = shutil.copy(path, directory)
    subprocess.run([objdump, "--offloading", copy], cwd=directory, check=True, capture_output=True)
    out = {}
    for name in sorted(os.listdir(directory)):
        if "gfx950" not in name:
            continue
        code = os.path.join(directory, name)
        table = subprocess.run([objdump, "-t", code], check=True, capture_output=True, text=True).stdout
        names = [s for s in re.findall(r"\.text\s+\S+ (?:\.\w+ )?(\S+)$", table, re.M)
                 if any(w in s for w in wanted)]
        if not names:
            continue
        text = subprocess.run([objdump, "-d", "--mcpu=gfx950", "--no-show-raw-insn",
                               "--disassemble-symbols=" + ",".join(names), code],
                              check=True, capture_output=True, text=True).stdout
        body = None
        for line in text.splitlines():
            head = re.match(r"[0-9a-f]+ <(.+)>:$", line)
            if head:
                body = out.setdefault(head[1], [])
            elif line.startswith("\t") and "//" in line and body is not None:
                code_line, note = line.split("//", 1)
                parts = code_line.split(None, 1)
                op = Op((parts[0], [o.strip() for o in parts[1].split(",")] if len(parts) > 1 else []))
                op.at = int(note.split(":")[0], 16)
                if op[0].startswith(("s_cbranch", "s_branch")):
                    offset = int(op[1][0])                # dwords from the next instruction, 16 bits
                    op.target = op.at + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)
                body.append(op)
    return out


def registers(operand, bank):
    """The numbers of the registers v.. or a.. (``bank``) that an operand names."""
    m = re.match(r"[-|]*" + bank + r"(?:(\d+)|\[(\d+):(\d+)\])", operand)
    if not m:
        return set()
    return {int(m[1])} if m[1] else set(range(int(m[2]), int(m[3]) + 1))
