#!/usr/bin/env python3
"""Static check of the loads that go straight to LDS in the compiled kernels (gfx950 ISA text, `hipcc -S`).

csrc/block_tile.hpp issues them by inline asm: `s_mov_b32 m0`, `s_nop`, `buffer_load_dword(x4) .. lds`.  m0 is a reserved register,
which no clobber list may name, so the compiler is not told that it changes: the kernels are right as long as nothing else in them
uses it.  This script proves that for the BINARY: every instruction that names m0 is the move of such a statement, and every such
load stands behind its own move.  (The counted waits behind these loads need no check: loads return in order among loads, and
whatever the compiler adds -- a spill's loads or stores -- only makes `vmcnt(N)` wait for more.)

    python tools/check_lds_loads.py file.s [...]        exit code 1 on a violation, or where a file has no such load
"""
import re
import sys

LOAD = re.compile(r"^buffer_load_dword(x4)? .* lds\b")
MOVE = re.compile(r"^s_mov_b32 m0, s\d+$")


def check(lines):
    """(violations, loads) of a listing's lines"""
    bad, loads, in_asm, moved = [], 0, False, False
    for no, raw in lines:
        text = raw.strip()
        if text.startswith((";;#ASMSTART", ";;#ASMEND")):
            in_asm, moved = text.startswith(";;#ASMSTART"), False
            continue
        text = " ".join(text.split(";", 1)[0].split())
        if not text or text.startswith("."):
            continue
        if in_asm and MOVE.match(text):
            moved = True
        elif re.search(r"\bm0\b", text):
            bad.append((no, text, "uses m0"))
        if LOAD.match(text):
            loads += 1
            if not (in_asm and moved):
                bad.append((no, text, "has no move of m0 in front of it"))
    return bad, loads


def main(paths):
    rc = 0
    for path in paths:
        with open(path) as f:
            bad, loads = check(enumerate(f, 1))
        for no, text, why in bad[:8]:
            print(f"{path}:{no}: `{text}` {why}")
        print(f"check_lds_loads: {path}: {loads} loads to LDS, {len(bad)} violation(s)")
        rc |= bool(bad) or loads == 0
    return int(rc)


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
