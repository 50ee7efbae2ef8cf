"""What the compiler makes of the attention kernels' divergent places.

A block in which lanes that took no part come back begins by restoring the
execution mask.  The compiler has been seen to put the copy of a register before
that (a zero that starts an accumulation: the lanes that had been off kept what
was there), so the assembly is searched for vector instructions in that place."""

from __future__ import annotations

import importlib.util
import re
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "nanovllm-dsa-offload_amd" / "csrc"


def _build():
    spec = importlib.util.spec_from_file_location("nvdsa_build_for_assembly", CSRC / "build.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def misplaced(text: str) -> list[str]:
    """Vector instructions between a label that a skipped region ends at and the
    restoring of the execution mask that follows it.  (Lane writes go by their
    lane number, whatever the mask.)"""
    skipped = set(re.findall(r"s_cbranch_execz\s+(\.LBB\S+)", text)) - set(re.findall(r"s_cbranch_execnz\s+(\.LBB\S+)", text))
    found, pending = [], None
    for line in text.split("\n"):
        label = re.match(r"^(\.LBB\S+?):", line)
        if label:
            pending = [] if label[1] in skipped else None
        elif pending is None:
            continue
        elif re.match(r"\s+s_or_b64 exec, exec,", line):
            found += pending
            pending = None
        elif re.match(r"^; %bb|\s+(s_\w+ exec,|s_\w*saveexec|s_c?branch|s_endpgm)", line):
            pending = None
        elif re.match(r"\s+(v_(?!writelane)|ds_|global_|flat_|buffer_|scratch_)", line):
            pending.append(line.strip())
    return found


def _registers(text: str) -> set[str]:
    ranges = re.findall(r"\b([va])\[(\d+):(\d+)\]", text)
    return {f"{k}{i}" for k, a, b in ranges for i in range(int(a), int(b) + 1)} | set(re.findall(r"\b([va]\d+)\b", text))


def left_behind(text: str) -> list[str]:
    """Copies and constants in a masked region that nothing in it reads.  (A
    region without a branch around it has no label at its end.)"""
    found, region = [], None
    for line in text.split("\n"):
        body = line.split(";")[0].strip()
        if "saveexec" in body:
            region = []
        elif re.match(r"(\.LBB|_Z)\S*:|s_(andn2|xor|mov)_b64 exec", body):
            region = None
        elif region is not None and re.match(r"s_or_b64 exec, exec,", body):
            for n, text_of in enumerate(region):
                copy = re.match(r"(?:v_mov_b32\S*|v_accvgpr_\w+)\s+([va]\d+|[va]\[\d+:\d+\]),", text_of)
                reads = [u if re.match(r"(ds_write|global_store|scratch_store)", u) else u.partition(",")[2] for u in region[n + 1:]]
                if copy and not any(_registers(copy[1]) & _registers(u) for u in reads):
                    found.append(text_of)
            region = None
        elif region is not None and body and not body.startswith("."):
            region.append(body)
    return found


def test_the_search_finds_a_misplaced_copy():
    text = "\ts_and_saveexec_b64 s[0:1], vcc\n\ts_cbranch_execz .LBB0_2\n; %bb.1:\n\tv_mov_b32_e32 v1, 0\n.LBB0_2:\n"
    assert misplaced(text + "\ts_or_b64 exec, exec, s[0:1]\n\tv_mov_b32_e32 v2, v3\n") == []
    assert misplaced(text + "\tv_accvgpr_write_b32 a16, v156\n\ts_or_b64 exec, exec, s[0:1]\n") == ["v_accvgpr_write_b32 a16, v156"]
    text = "\ts_and_saveexec_b64 s[0:1], vcc\n\tv_mov_b32_e32 v1, 0\n\tds_write_b32 v2, v1\n"
    assert left_behind(text + "\ts_or_b64 exec, exec, s[0:1]\n") == []
    assert left_behind(text + "\tv_mov_b32_e32 v9, 4\n\ts_or_b64 exec, exec, s[0:1]\n") == ["v_mov_b32_e32 v9, 4"]


def test_attention_kernels_restore_all_lanes_first(tmp_path):
    build = _build()
    try:
        hipcc = build._hipcc()
    except RuntimeError as e:
        pytest.skip(str(e))
    out = tmp_path / "prefix_attention.s"
    command = [hipcc, *build.COMMON_FLAGS, *build.EXTRA_FLAGS["prefix_attention.hip"], "--cuda-device-only", "-S",
               str(CSRC / "prefix_attention.hip"), "-o", str(out)]
    subprocess.run(command, check=True, capture_output=True, timeout=600)
    text = out.read_text()
    assert text.count("s_or_b64 exec, exec,") > 10
    assert misplaced(text) == [] and left_behind(text) == []
