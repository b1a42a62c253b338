#!/usr/bin/env python3
"""Static check of the loads that go straight to LDS in the compiled kernels (gfx950 ISA text, `hipcc -S`).

csrc/block_tile.hpp issues them by inline asm: `s_mov_b32 m0`, `s_nop`, `buffer_load_dword(x4) .. lds`.  m0 is a reserved register,
which no clobber list may name, so the compiler is not told that it changes: the kernels are right as long as nothing else in them
uses it.  This script proves that for the BINARY: every instruction that names m0 is the move of such a statement, and every such
load stands behind its own move.  And since the compiler's hazard recognizer does not look into a statement: the statement itself
lets WAITS wait states pass before its load, which a vector memory instruction needs behind a vector instruction that writes one
of its scalar registers (v_readfirstlane of the buffer's address, v_readlane of a spilled one).  (The counted waits behind these loads need no check: loads return in order among loads, and
whatever the compiler adds -- a spill's loads or stores -- only makes `vmcnt(N)` wait for more.)

    python tools/check_lds_loads.py file.s [...]        exit code 1 on a violation, or where a file has no such load
"""
import re
import sys

LOAD = re.compile(r"^buffer_load_dword(x4)? .* lds\b")
MOVE = re.compile(r"^s_mov_b32 m0, s\d+$")
NOP = re.compile(r"^s_nop (\d+)$")
WAITS = 5


def check(lines):
    """(violations, loads) of a listing's lines"""
    bad, loads, in_asm, moved, waited = [], 0, False, False, 0
    for no, raw in lines:
        text = raw.strip()
        if text.startswith((";;#ASMSTART", ";;#ASMEND")):
            in_asm, moved, waited = text.startswith(";;#ASMSTART"), False, 0
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
            elif waited < WAITS:
                bad.append((no, text, f"comes {waited} wait states behind what stands in front of the statement, {WAITS} are needed"))
        nop = NOP.match(text)
        waited += int(nop.group(1)) + 1 if nop else 1
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
