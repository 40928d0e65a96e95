"""What the tile kernels of differential attention rest on and the compiler does
not check, read from the code built here: their accumulators live in named
registers (v128 and a128 upwards) that inline assembly alone may touch, and the
compiler puts no wait states around MFMAs written in inline assembly.  CPU only:
the library is disassembled, not loaded."""

from __future__ import annotations

import re
import shutil
import struct
import subprocess
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parents[1] / "proxy-attention-lab_amd" / "proxy_attention_lab"
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"
# the inline assembly's instructions: products, and element moves, scalings and joins
ON_ACCUMULATORS = {"v_mfma_f32_32x32x16_f16", "v_mfma_f32_32x32x16_bf16", "v_mov_b32_e32", "v_mul_f32_e32", "v_fma_f32",
                   "v_fmac_f32_e32", "v_accvgpr_read_b32", "v_accvgpr_write_b32"}
D_STATES = 18  # wait states from a 32x32x16 MFMA to a read of its result by anything but the next sum
AB_STATES = 2  # from a vector instruction's result to an MFMA that multiplies it


def code_objects(lib: Path):
    data = lib.read_bytes()
    at = data.find(MAGIC)
    while at >= 0:
        (n,) = struct.unpack_from("<Q", data, at + 24)
        pos = at + 32
        for _ in range(n):
            offset, size, name_len = struct.unpack_from("<QQQ", data, pos)
            name = data[pos + 24: pos + 24 + name_len]
            pos += 24 + name_len
            if b"gfx950" in name and size:
                yield data[at + offset: at + offset + size]
        at = data.find(MAGIC, at + 32)


def registers(operand: str) -> set:
    t = operand.strip().split(" ")[0]
    if m := re.fullmatch(r"([va])\[(\d+):(\d+)\]", t):
        return {(m[1], i) for i in range(int(m[2]), int(m[3]) + 1)}
    m = re.fullmatch(r"([va])(\d+)", t)
    return {(m[1], int(m[2]))} if m else set()


def faults(lines):
    """(instructions on the accumulators that are not the inline assembly's, MFMAs too
    near behind an operand's conversion, uses too near behind an MFMA)"""
    touched, early, late, products = [], [], [], 0
    recent = []   # (wait states, registers written)
    pending = []  # (result, age, text) of MFMAs
    for text in lines:
        op, _, rest = text.partition(" ")
        args = [a.strip() for a in rest.split(",")] if rest else []
        if op.startswith("s_cbranch") or op in ("s_branch", "s_setpc_b64"):
            recent.append((1, set()))
            continue
        used = set().union(*map(registers, args)) if args else set()
        if op not in ON_ACCUMULATORS and any(i >= 128 for _, i in used):
            touched.append(text)
        states = int(args[0], 0) + 1 if op == "s_nop" else 1
        if "mfma" in op:
            products += 1
            ab, c = registers(args[1]) | registers(args[2]), registers(args[3])
            seen = 0
            for s, written in reversed(recent):
                if seen >= AB_STATES:
                    break
                if written & ab:
                    early.append(text)
                    break
                seen += s
            late += [text for d, age, _ in pending if d & ab or (d & c and d != c)]
            wrote = set()
        else:
            late += [f"{text}  behind  {t}" for d, age, t in pending if d & used]
            wrote = registers(args[0]) if op.startswith("v_") and args else set()
            if "swap" in op:
                wrote |= registers(args[1])
        pending = [(d, age + states, t) for d, age, t in pending if age + states < D_STATES]
        if "mfma" in op:
            pending.append((registers(args[0]), 0, text))
        recent = recent[-4:] + [(states, wrote)]
    return touched, early, late, products


@pytest.mark.skipif(not Path(OBJDUMP).exists(), reason="needs the ROCm disassembler")
@pytest.mark.parametrize("name", ["libpal_hip.so", "libpal_hip_debug.so"])
def test_tile_kernels(name, tmp_path):
    lib = PACKAGE / name
    if not lib.exists():
        pytest.skip(f"{name} is not built")
    kernels = {}
    for i, blob in enumerate(code_objects(lib)):
        if b"diff_tile_kernel" not in blob:
            continue
        path = tmp_path / f"{i}.co"
        path.write_bytes(blob)
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], capture_output=True, text=True,
                              check=True).stdout
        current = None
        for line in text.splitlines():
            if m := re.match(r"(?:[0-9a-f]+ )?<(\w+)>:", line):
                current = kernels.setdefault(m[1], []) if "diff_tile_kernel" in m[1] else None
            elif current is not None and line.strip():
                current.append(line.split("//")[0].split(";")[0].strip())
    assert len(kernels) == 24, sorted(kernels)  # 2 types x (4 head sizes + 2 over fp8 pages) x 2 page sizes
    for kernel, lines in kernels.items():
        touched, early, late, products = faults(lines)
        assert products >= 36, (kernel, products)
        assert not touched, (kernel, touched[:5])
        assert not early, (kernel, early[:5])
        assert not late, (kernel, late[:5])
