"""Loads straight into LDS in the built library: one wait state lies between the scalar write of M0 and a load that takes its LDS address from there
(the compiler fills it for its own loads, not inside inline assembly), and the kernels whose loads are assembly use M0 for nothing else.  Where such a load
takes its base from scalar registers, five wait states lie between a vector instruction that may have written them and the load."""
import os
import re
import shutil
import subprocess

import pytest

from im2im_uq_amd import _lib

OBJDUMP = "/opt/rocm/lib/llvm/bin/llvm-objdump"
LABEL = re.compile(r"^[0-9a-f]+ <([^>]+)>:")
DMA = re.compile(r"^\s*(global_load_lds_|(buffer|scratch)_load_\w+.*\blds\b)")
WRITES_M0 = re.compile(r"^\s*s_\w+\s+m0\b")
SETS_ADDRESS = re.compile(r"^\s*s_mov_b32\s+m0,\s*s\d+\s*$")
READS_M0 = re.compile(r"^\s*(v_movrel|s_movrel|s_sendmsg|ds_gws)")                # without naming it


def instructions(tmp):
    """(kernel, text) of every instruction of the library's device code"""
    copy = os.path.join(tmp, "lib.so")
    shutil.copy(_lib.LIB_PATH, copy)
    subprocess.run([OBJDUMP, "--offloading", copy], check=True, capture_output=True)
    for f in sorted(f for f in os.listdir(tmp) if "amdgcn" in f):
        p = subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", os.path.join(tmp, f)], stdout=subprocess.PIPE, text=True)
        kernel = "?"
        for line in p.stdout:
            m = LABEL.match(line)
            if m:
                kernel = m.group(1)
            elif line[:1].isspace():
                yield kernel, line.split("//")[0]
        p.wait()


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="llvm-objdump not available")
def test_wait_state_before_every_load_into_lds(tmp_path):
    bare, early, other, loads, before = {}, {}, {}, 0, ""
    for kernel, text in instructions(str(tmp_path)):
        if DMA.match(text):
            loads += 1
            if WRITES_M0.match(before):
                bare[kernel] = bare.get(kernel, 0) + 1
            wait = re.match(r"\s*s_nop\s+(\d+)", before)
            if "attn_" in kernel and "s[" in text and not (wait and int(wait.group(1)) >= 3):           # and the s_mov before it
                early[kernel] = early.get(kernel, 0) + 1
        if "attn_" in kernel and ((re.search(r"\bm0\b", text) and not SETS_ADDRESS.match(text)) or READS_M0.match(text)):
            other.setdefault(kernel, text.strip())
        before = text
    assert loads > 1000, "no loads into LDS found"
    assert not bare, f"{sum(bare.values())} of {loads} loads right behind the write of M0: {bare}"
    assert not early, f"{sum(early.values())} of {loads} loads too early behind a write of their base: {early}"
    assert not other, other
