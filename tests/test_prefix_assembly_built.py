"""The built library holds the code whose assembly is searched: the attention
kernels, compiled once more with the build's flags, are in it byte for byte."""

from __future__ import annotations

import struct
import subprocess

import pytest

from test_prefix_assembly import CSRC, _build, left_behind, misplaced


def _text(elf: bytes) -> bytes:
    """The section .text of a 64-bit ELF file."""
    assert elf[:5] == b"\x7fELF\x02"
    table, = struct.unpack_from("<Q", elf, 0x28)
    size, count, names = struct.unpack_from("<HHH", elf, 0x3A)
    sections = [struct.unpack_from("<IIQQQQ", elf, table + i * size) for i in range(count)]
    for name, _, _, _, offset, length in sections:
        at = sections[names][4] + name
        if elf[at:elf.index(b"\0", at)] == b".text":
            return elf[offset:offset + length]
    raise AssertionError("no .text")


def test_the_built_library_holds_the_searched_code(tmp_path):
    build = _build()
    try:
        hipcc = build._hipcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    source = CSRC / "prefix_attention.hip"
    command = [hipcc, *build.COMMON_FLAGS, *build.EXTRA_FLAGS[source.name], "--cuda-device-only", "-c", "-save-temps=obj",
               str(source), "-o", str(tmp_path / "code.co")]
    subprocess.run(command, check=True, capture_output=True, timeout=600)
    assembly, = tmp_path.glob("*.s")
    linked, = tmp_path.glob("*.out")
    searched = assembly.read_text()
    assert searched.count("s_or_b64 exec, exec,") > 10
    assert misplaced(searched) == [] and left_behind(searched) == []
    code, library = _text(linked.read_bytes()), build.OUTPUT.read_bytes()
    assert len(code) > 100_000 and code in library
    changed = bytearray(code)
    changed[len(code) // 2] ^= 1
    assert bytes(changed) not in library
