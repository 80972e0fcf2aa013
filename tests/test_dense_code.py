"""What the large dense kernel's machine code has to keep, from the built library's own listing: its
MFMAs are written in assembly, which the compiler inserts no waits for, so nothing between them
may move their sums from one register to another."""

import os
import re
import subprocess

import pytest

from bux_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def _images(image: bytes):
    """Every ELF embedded in the library."""
    at = image.find(b"\x7fELF", 1)
    while at >= 0:
        end = image.find(b"\x7fELF", at + 1)
        yield image[at:end if end >= 0 else len(image)]
        at = end


def test_sums_stay_in_their_registers_between_mfmas(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    if not os.path.exists(_lib.PATH):
        pytest.fail(f"{_lib.PATH} is not built: run python -m bux_amd.build")
    with open(_lib.PATH, "rb") as f:
        images = [i for i in _images(f.read()) if b"12large_kernel" in i and b"amdhsa.kernels" in i]
    assert images
    seen = 0
    for n, image in enumerate(images):
        elf = tmp_path / f"{n}.elf"
        elf.write_bytes(image)
        listing = subprocess.run([OBJDUMP, "-d", str(elf)], check=True, capture_output=True,
                                 text=True).stdout
        for body in re.split(r"^[0-9a-f]+ <", listing, flags=re.M)[1:]:
            if "12large_kernel" not in body.split(">")[0]:
                continue
            lines = body.splitlines()
            at = [i for i, line in enumerate(lines) if "v_mfma_f32_16x16x32_bf16" in line]
            # a pair's two steps and the last pair's, 64 each
            assert len(at) == 256, body.split(">")[0]
            moves = [line for line in lines[at[0]:at[-1]] if "v_accvgpr" in line or "scratch_" in line]
            assert not moves, moves[:3]
            seen += 1
    assert seen == 10
