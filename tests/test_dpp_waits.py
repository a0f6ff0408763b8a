"""The built kernels' reads across lanes (DPP). A vector register that a vector instruction
writes may be read across lanes two instructions later at the earliest. The compiler sees to
that for its own instructions, not for those in asm statements, which it does not look into."""
import os
import re
import shutil
import struct
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen38-3090-cuda-server_amd")
LIBRARY = os.path.join(PKG, "libqwen_w4a16.so")
OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
APART = 2


def code_objects(data: bytes):
    """The gfx950 code objects of the library's offload bundles."""
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        p = at + len(MAGIC) + 8
        for _ in range(count):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            name = data[p + 24:p + 24 + length]
            p += 24 + length
            if b"gfx950" in name and size:
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, at + 1)


def registers(operand: str) -> set:
    m = re.fullmatch(r"-?\|?v\[(\d+):(\d+)\]\|?", operand) or re.fullmatch(r"-?\|?v(\d+)\|?", operand)
    if not m:
        return set()
    return set(range(int(m[1]), int(m[m.lastindex]) + 1))


def operands(line: str) -> list:
    parts = line.split("//")[0].strip().split(None, 1)
    return [parts[0]] + ([a.strip().split()[0] for a in re.split(r",(?![^\[]*\])", parts[1])] if len(parts) > 1 else [])


def written(line: str) -> set:
    op = operands(line)
    if not op[0].startswith("v_") or op[0].startswith(("v_cmp", "v_readlane", "v_readfirstlane")):
        return set()
    return registers(op[1]) if len(op) > 1 else set()


def too_near(text: str):
    """The lines that read across lanes what one of the two instructions before them wrote, and
    the number of lines looked at."""
    bad, seen, before = [], 0, []
    for line in text.splitlines():
        if not line.startswith("\t"):
            if line.endswith(">:"):
                before = []
            continue
        s = line.strip()
        if s.startswith("s_nop"):
            before += [""] * (int(operands(s)[1], 0) + 1)
        else:
            if "_dpp " in s:
                seen += 1
                source = registers(operands(s)[2])
                if any(source & written(b) for b in before[-APART:] if b):
                    bad.append(s)
            before.append(s)
        del before[:-APART]
    return bad, seen


def test_too_near_sees_what_it_looks_for():
    read = "\tv_fmac_f32_dpp v3, v7, v9 quad_perm:[0,0,0,0] row_mask:0xf bank_mask:0xf // 0: 0"
    mov, other = "\tv_mov_b32_e32 v7, v1 // 0: 0", "\tv_add_f32_e32 v4, v1, v2 // 0: 0"
    pair = "\tv_lshlrev_b64 v[6:7], 1, v[2:3]"
    for text, bad in (([mov, read], 1), ([mov, other, read], 1), ([mov, other, other, read], 0), ([mov, "\ts_nop 0", read], 1),
                      ([mov, "\ts_nop 1", read], 0), ([pair, read], 1), ([other, read], 0),
                      (["\tds_read_b32 v7, v1", read], 0), (["\tv_mov_b32_e32 v9, v1", read], 0)):
        assert too_near("\n".join(text)) == ([read.strip()] if bad else [], 1), text


def test_built_kernels():
    if not os.path.exists(LIBRARY) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library, or no disassembler")
    data, total = open(LIBRARY, "rb").read(), 0
    objects = list(code_objects(data))
    assert objects
    for code in objects:
        r = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "/dev/stdin"], input=code, capture_output=True)
        assert r.returncode == 0, r.stderr
        bad, seen = too_near(r.stdout.decode())
        assert not bad, bad[:5]
        total += seen
    assert total > 1000
