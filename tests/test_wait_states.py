"""Loads from memory to LDS that are written in assembly: the compiler counts no wait states before them, so the compiled
code is read for the two that such a load needs (one after a scalar instruction has set m0, five after a vector instruction
has written m0 or the scalar registers of its address)."""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LINE = re.compile(r"^\t(\S+) ?(.*?) *// ([0-9A-F]+): [0-9A-F ]+?(?:<(.+)\+0x([0-9a-f]+)>)?$")


def scalars(arg):
    m = re.match(r"s\[(\d+):(\d+)\]$", arg)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.match(r"s(\d+)$", arg)
    return {int(m[1])} if m else {arg} if arg in ("m0", "vcc", "vcc_lo", "vcc_hi") else set()


def functions(text):
    """name -> instructions [(mnemonic, operands, index of the target or None)]"""
    for part in re.split(r"^(?=[0-9a-f]* ?<\S+>:$)", text, flags=re.M):
        head = re.match(r"[0-9a-f]* ?<(\S+)>:$", part, re.M)
        if not head or "_load_lds" not in part and " lds" not in part:
            continue
        rows = [m.groups() for m in map(LINE.match, part.split("\n")) if m]
        at = {int(r[2], 16): i for i, r in enumerate(rows)}
        base = int(rows[0][2], 16)
        yield head[1], [(r[0], [a.strip() for a in r[1].split(",")] if r[1] else [],
                         at.get(base + int(r[4], 16)) if r[3] and "branch" in r[0] else None) for r in rows]


def loads_too_early(code):
    """(loads looked at, what is wrong with them), every way there counted: over falling through and over branches."""
    come = {}
    for i, (op, _, to) in enumerate(code):
        if to is not None:
            come.setdefault(to, []).append(i)
    n, bad = 0, []

    def look(i, need, ws, load):
        """Instruction i comes before `load` with ws wait states between them."""
        while ws < 5 and i >= 0:
            op, args, _ = code[i]
            wrote = scalars(args[0]) if args else set()
            if op.startswith("v_") and wrote & need:
                bad.append(f"{op} {', '.join(args)} {ws} before {load}")
                return
            if ws == 0 and op.startswith("s_") and wrote & need & {"m0"}:
                bad.append(f"{op} {', '.join(args)} right before {load}")
                return
            ws += int(args[0], 0) + 1 if op == "s_nop" else 1
            for j in come.get(i, []):
                look(j, need, ws, load)
            if i > 0 and code[i - 1][0] in ("s_branch", "s_endpgm", "s_setpc_b64"):
                return
            i -= 1

    for i, (op, args, _) in enumerate(code):
        if "_load_lds" in op or op.startswith("buffer_load") and args and args[-1].endswith(" lds"):
            n += 1
            need = set().union({"m0"}, *(scalars(w) for a in args for w in a.split()))
            text = f"{op} {', '.join(args)}"
            for j in come.get(i, []):
                look(j, need, 0, text)
            if not (i > 0 and code[i - 1][0] in ("s_branch", "s_endpgm", "s_setpc_b64")):
                look(i - 1, need, 0, text)
    return n, bad


def test_what_is_wrong_is_found():
    def code(*lines):
        return [(t.split()[0], [a.strip() for a in t.split(" ", 1)[1].split(",")] if " " in t else [], to) for t, to in lines]

    load = ("global_load_lds_dwordx4 v1, s[4:5]", None)
    read, other = ("v_readlane_b32 s5, v9, 3", None), ("v_add_u32 v1, v2, v3", None)
    assert loads_too_early(code(read, other, load)) == (1, ["v_readlane_b32 s5, v9, 3 1 before global_load_lds_dwordx4 v1, s[4:5]"])
    assert loads_too_early(code(read, ("s_nop 3", None), load))[1] != []
    assert loads_too_early(code(read, ("s_nop 4", None), load)) == (1, [])
    assert loads_too_early(code(("v_readlane_b32 s6, v9, 3", None), load)) == (1, [])
    assert loads_too_early(code(("s_mov_b32 m0, s9", None), load))[1] != []
    assert loads_too_early(code(("s_mov_b32 m0, s9", None), ("s_nop 0", None), load)) == (1, [])
    # over a branch back to the load, and past what only another way comes by
    assert loads_too_early(code(load, read, ("s_cbranch_scc1 9", 0)))[1] != []
    assert loads_too_early(code(("s_cbranch_scc1 9", 3), read, ("s_branch 9", 1), load)) == (1, [])


def test_loads_to_lds_come_late_enough(q, tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    lib = shutil.copy(q.LIB_PATH, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", lib], cwd=tmp_path, check=True, capture_output=True)
    seen = 0
    for f in sorted(tmp_path.glob("*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-leading-addr", f], check=True, capture_output=True, text=True).stdout
        for name, code in functions(text):
            n, bad = loads_too_early(code)
            assert not bad, (name, bad)
            seen += n
    assert seen >= 100, seen
