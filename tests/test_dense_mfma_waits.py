"""The large dense kernel's MFMAs are written in assembly, so the compiler inserts none of the two waits
that stand between a vector instruction and an MFMA that reads what it wrote: no such pair lies
closer in the built library's own listing."""

import os
import re
import subprocess

import pytest

from bux_amd import _lib
from test_dense_code import OBJDUMP, _images

WAITS = 2


def _registers(operand):
    """The vector registers that an operand names."""
    found = re.fullmatch(r"v(?:(\d+)|\[(\d+):(\d+)\])", operand.strip())
    if not found:
        return set()
    one, lo, hi = found.groups()
    return {int(one)} if one else set(range(int(lo), int(hi) + 1))


def too_close(instructions):
    """(writer, MFMA) of every MFMA that reads, as A or B, what a vector instruction wrote under
    WAITS wait states before. An instruction between them is one, s_nop n is n + 1."""
    bad = []
    for i, line in enumerate(instructions):
        if not line.startswith("v_mfma"):
            continue
        _, a, b, _ = line.split(None, 1)[1].split(",")
        read = _registers(a) | _registers(b)
        waits, at = 0, i - 1
        while at >= 0 and waits < WAITS:
            name, _, rest = instructions[at].partition(" ")
            if name == "s_nop":
                waits += int(rest.strip(), 0) + 1
            else:
                vector = name.startswith("v_") and not name.startswith("v_mfma")
                if vector and _registers(rest.split(",")[0]) & read:
                    bad.append((instructions[at], line))
                waits += 1
            at -= 1
    return bad


MFMA = "v_mfma_f32_16x16x32_bf16 a[0:3], v[8:11], v[4:7], a[0:3]"


@pytest.mark.parametrize("before, close", [
    (["v_and_b32_e32 v9, v1, v2"], True),
    (["v_mov_b32_e32 v4, v1", "s_add_u32 m0, s0, s1"], True),
    (["v_mov_b32_e32 v4, v1", "s_nop 0"], True),
    (["v_mov_b32_e32 v4, v1", "s_nop 1"], False),
    (["v_mov_b32_e32 v4, v1", "s_add_u32 m0, s0, s1", "s_nop 0"], False),
    (["v_mov_b32_e32 v12, v9"], False),
    (["v_pk_add_u16 v[10:11], v[0:1], v[2:3]"], True),
    (["ds_read_b128 v[8:11], v1"], False),
    ([MFMA], False),
], ids=str)
def test_the_rule(before, close):
    assert bool(too_close(before + [MFMA])) == close


def test_nothing_writes_an_operand_just_before_its_mfma(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    if not os.path.exists(_lib.PATH):
        pytest.fail(f"{_lib.PATH} is not built: run python -m bux_amd.build")
    with open(_lib.PATH, "rb") as f:
        images = [i for i in _images(f.read()) if b"12large_kernel" in i and b"amdhsa.kernels" in i]
    seen = 0
    for n, image in enumerate(images):
        elf = tmp_path / f"{n}.elf"
        elf.write_bytes(image)
        listing = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(elf)], check=True,
                                 capture_output=True, text=True).stdout
        for body in re.split(r"^[0-9a-f]+ <", listing, flags=re.M)[1:]:
            if "12large_kernel" not in body.split(">")[0]:
                continue
            instructions = [line.split("//")[0].strip() for line in body.splitlines()[1:]]
            instructions = [line for line in instructions if line]
            assert sum(line.startswith("v_mfma") for line in instructions) == 256
            assert not too_close(instructions), too_close(instructions)[:3]
            seen += 1
    assert seen == 10
