#!/usr/bin/env python3
"""Static check of register spills at the joins of divergent branches in the compiled kernels (gfx950 ISA text, `hipcc -S`).

Behind a branch that some lanes of a wave do not take stands `s_or_b64 exec, exec, ..`, which switches them on again.  The compiler
(ROCm 7.2) has put a vector register away (v_accvgpr_write of a vector register, a scratch store) IN FRONT of that instruction, in the
same block: the register of the lanes that were off is then not kept, and comes back as whatever lay there -- a thread's own number in
the case that was seen, and an address made of it.  This script finds such places; they are mended in the source, by code without that
branch or with fewer registers.

    python tools/check_spills.py file.s [...]        exit code 1 where there is one
"""
import re
import sys

LABEL = re.compile(r"^\.LBB\d+_\d+:")
JOIN = re.compile(r"^s_or_b64 exec, exec, ")
SPILL = re.compile(r"^(v_accvgpr_write_b32 a\d+, v\d+|scratch_store_|buffer_store_dword v\d+, off, )")
OTHER = re.compile(r"^s_(cbranch|branch|endpgm)|\bexec\b")


def check(lines):
    """[(line, spill)] of a listing's lines"""
    bad, block = [], None
    for no, raw in lines:
        if LABEL.match(raw):
            block = []
            continue
        text = raw.split(";", 1)[0].strip()
        if not text or text.startswith(".") or block is None:
            continue
        if JOIN.match(text):
            bad += block
            block = None
        elif OTHER.search(text):
            block = None
        elif SPILL.match(text):
            block.append((no, text))
    return bad


def main(paths):
    total = 0
    for path in paths:
        with open(path) as f:
            bad = check(enumerate(f, 1))
        for no, text in bad[:8]:
            print(f"{path}:{no}: `{text}` puts a register away before all lanes are on again")
        total += len(bad)
    print(f"check_spills: {len(paths)} files, {total} violation(s)")
    return 1 if total else 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
