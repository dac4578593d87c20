"""Loads from memory straight into LDS take their LDS address from M0.  gfx950 wants one wait
state between a scalar write of M0 and such a load, and five between a vector write of a scalar
register and a load that reads it; the compiler keeps both for its own instructions but does not
look inside inline assembly, where these loads are written.  CPU only: disassembles the library's
own build."""

import os
import re
import subprocess

import pytest

from test_code_objects import LLVM, _code_objects

SCALARS = re.compile(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(m0|vcc)\b")


def scalars(text):
    out = set()
    for lo, hi, one, name in SCALARS.findall(text):
        out |= {name} if name else set(range(int(lo or one), int(hi or one) + 1))
    return out


def instructions(co):
    text = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--mcpu=gfx950",
                           "--no-show-raw-insn", str(co)], check=True, capture_output=True,
                          text=True).stdout
    for line in text.splitlines():
        if re.match(r"[0-9a-f]+ <", line):
            yield "label", ""
        elif m := re.match(r"\s+([a-z]\S*)\s*(.*?)(?:\s*//.*)?$", line):
            yield m[1], m[2]


def too_early(before, load):
    """What of the instructions in front of a load (nearest last) it does not wait for."""
    reads, states = scalars(load), 0
    for op, args in reversed(before):
        if op == "label" or states >= 5:
            break
        writes = scalars(args.split(",")[0])
        if op.startswith("s_") and "m0" in writes and states < 1 or \
                op.startswith("v_") and writes & reads:
            return f"{op} {args}, {states} wait states, {load}"
        states += int(args, 0) + 1 if op == "s_nop" else 1
    return None


def test_loads_into_lds_wait_for_their_scalars(tmp_path):
    if not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("llvm-objdump not available")
    loads = 0
    for co in _code_objects(tmp_path):
        code = list(instructions(co))
        for i, (op, args) in enumerate(code):
            if op.startswith("buffer_load") and "lds" in args.split():
                loads += 1
                assert not (off := too_early(code[max(0, i - 8):i], args)), off
    assert loads >= 100


def test_the_check_sees_what_it_is_for():
    load = "v1, s[4:7], s9 offen lds"
    assert too_early([("s_mov_b32", "m0, s3")], load)
    assert not too_early([("s_mov_b32", "m0, s3"), ("s_nop", "0")], load)
    assert too_early([("v_readfirstlane_b32", "s9, v2"), ("s_nop", "3")], load)
    assert not too_early([("v_readfirstlane_b32", "s9, v2"), ("s_nop", "4")], load)
    assert not too_early([("v_readfirstlane_b32", "s8, v2")], load)
