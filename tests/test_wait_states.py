"""Wait states in front of the loads that write LDS directly (load_to_lds in mma.h).  They are written in inline asm, which the compiler
does not look into: a scalar register that a vector instruction has written may be read by a memory instruction five wait states later
at the earliest, and m0 by a load into LDS one after it was written; nothing else in a function with such loads may read m0.  The built library's own code is looked over, along every way that
leads to such a load, whatever the compiler knew of its operands."""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
VALU_TO_VMEM, M0_TO_LDS = 5, 1

LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]{12}):")


def parse(text):
    """[(address, mnemonic, operands)] of a listing, with None where a function begins."""
    code = []
    for line in text.splitlines():
        m = LINE.match(line)
        if m:
            code.append((int(m[3], 16), m[1], m[2]))
        elif line.endswith(">:"):
            code.append(None)
    return code


def scalars(operand):
    """The numbers of the scalar registers that an operand names."""
    m = re.match(r"s\[(\d+):(\d+)\]$", operand) or re.match(r"s(\d+)$", operand)
    return set(range(int(m[1]), int(m[m.lastindex]) + 1)) if m else set()


def split(operands):
    return [o.split()[0] if o.split() else "" for o in re.split(r",\s*(?![^\[]*\])", operands)]


def written_by_vector(mnemonic, operands):
    if not mnemonic.startswith("v_"):
        return set()
    ops = split(operands)
    out = scalars(ops[0])
    if len(ops) > 1 and re.search(r"_co_|div_scale|mad_[ui]64", mnemonic):
        out |= scalars(ops[1])
    return out


def faults(code):
    """(address, register, wait states there are) of the loads into LDS that come too early."""
    at = {c[0]: i for i, c in enumerate(code) if c}
    sources = {}
    for i, c in enumerate(code):
        if c and re.match(r"s_c?branch", c[1]):
            step = int(c[2].split()[0])
            target = at.get(c[0] + 4 + 4 * (step - 65536 if step >= 32768 else step))
            if target is not None:
                sources.setdefault(target, []).append(i)
    found, loads = [], 0
    for i, c in enumerate(code):
        if not c or not c[1].startswith("buffer_load") or not re.search(r"\blds\b", c[2]):
            continue
        loads += 1
        reads = set().union(*(scalars(o) for o in split(c[2])))
        seen, todo = set(), [(j, 0) for j in [i - 1] + sources.get(i, [])]
        while todo:
            j, states = todo.pop()
            if j < 0 or code[j] is None or (j, states) in seen or states >= VALU_TO_VMEM:
                continue
            seen.add((j, states))
            _, mnemonic, operands = code[j]
            if mnemonic in ("s_branch", "s_endpgm", "s_setpc_b64") and j == i - 1 and states == 0:
                continue                        # (nothing falls through)
            for r in sorted(written_by_vector(mnemonic, operands) & reads):
                found.append((hex(c[0]), "s%d" % r, states))
            if mnemonic.startswith("s_") and split(operands)[0] == "m0" and states < M0_TO_LDS:
                found.append((hex(c[0]), "m0", states))
            states += int(operands.split()[0], 0) + 1 if mnemonic == "s_nop" else 1
            before = [k for k in [j - 1] + sources.get(j, [])
                      if not (k == j - 1 and k >= 0 and code[k] and code[k][1] in ("s_branch", "s_endpgm", "s_setpc_b64"))]
            todo += [(k, states) for k in before]
    return found, loads


def other_uses_of_m0(code):
    """(address, instruction) of what names m0 in a function with loads into LDS, but for the s_mov_b32 of such a load."""
    found, function, loads = [], [], False
    for c in code + [None]:
        if c is None:
            if loads:
                found += function
            function, loads = [], False
            continue
        loads |= c[1].startswith("buffer_load") and bool(re.search(r"\blds\b", c[2]))
        if re.search(r"\bm0\b", c[2]) and not (c[1] == "s_mov_b32" and split(c[2])[0] == "m0") \
                or c[1].startswith(("s_sendmsg", "v_movrel", "s_set_gpr_idx", "v_interp", "ds_gws")):
            function.append((hex(c[0]), c[1], c[2]))
    return found


def listing(*lines):
    return "0000000000001000 <f>:\n" + "".join("\t%s // %012X: 00000000\n" % (t, 0x1000 + 4 * i) for i, t in enumerate(lines))


def test_the_looking_over_itself():
    load = "buffer_load_dwordx4 v1, s[4:7], s9 offen lds"
    for lines, bad in (
            (("v_readfirstlane_b32 s9, v0", "s_mov_b32 m0, s3", "s_nop 0", load), True),
            (("v_readfirstlane_b32 s9, v0", "s_mov_b32 m0, s3", "s_nop 2", load), True),
            (("v_readfirstlane_b32 s9, v0", "s_mov_b32 m0, s3", "s_nop 3", load), False),
            (("v_readfirstlane_b32 s6, v0", "v_mov_b32 v2, v3", "s_nop 2", load), True),
            (("v_cmp_gt_i32 s[6:7], v0, v1", "s_nop 3", load), True),
            (("v_add_co_u32 v5, s[8:9], v0, v1", "s_nop 3", load), True),
            (("v_readfirstlane_b32 s8, v0", load), False),
            (("s_mov_b32 m0, s3", load), True),
            (("v_readfirstlane_b32 s9, v0", "s_branch 1", "s_endpgm", "s_nop 2", load), True),      # round the end of the program
            (("v_readfirstlane_b32 s9, v0", "s_branch 1", "s_endpgm", "s_nop 3", load), False),
            (("s_nop 4", load, "v_readfirstlane_b32 s9, v0", "s_cbranch_vccnz 65532"), False),      # back to the s_nop
            (("s_nop 4", load, "v_readfirstlane_b32 s9, v0", "s_cbranch_vccnz 65533"), True)):      # back to the load
        found, loads = faults(parse(listing(*lines)))
        assert loads == 1 and bool(found) == bad, (lines, found)
    for line, bad in (("s_mov_b32 m0, s3", False), ("s_mov_b32 s3, m0", True), ("v_readlane_b32 s1, v0, m0", True), ("s_set_gpr_idx_on s0, gpr_idx(SRC0)", True)):
        assert bool(other_uses_of_m0(parse(listing(line, load)))) == bad, line
        assert not other_uses_of_m0(parse(listing(line)))


def test_loads_into_lds_wait_for_their_scalars(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump here")
    import ane_amd.bridge as br
    shutil.copy(br.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    found, loads, m0 = [], 0, []
    for name in sorted(os.listdir(tmp_path)):
        if not name.endswith("gfx950"):
            continue
        text = subprocess.run([OBJDUMP, "-d", name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout
        if " lds" not in text:
            continue
        code = parse(text)
        f, n = faults(code)
        m0 += other_uses_of_m0(code)
        found += [(name,) + x for x in f]
        loads += n
    assert loads > 1000
    assert not found, (len(found), found[:5])
    assert not m0, (len(m0), m0[:5])
