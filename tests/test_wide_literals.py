"""64-bit constants of the built library's device code.  An instruction holds 32 bits of a constant behind it; a 64-bit move extends them as an
integer.  The compiler has been seen to set a pair of scalar registers to the double -inf (0xfff0000000000000) by one such move with the lower 32 bits
behind it, and the pair was 0 then, with no error.  It takes any double whose lower half is zero for a constant of 32 bits, so what such a move leaves is a
literal of 0: a number that never needs a literal, as those from -16 to 64 do not.  Every literal of a 64-bit instruction is looked at for these."""
import os
import re
import shutil
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LINE = re.compile(r"^\t(\S+)\s.*// ([0-9A-F]{12}): ([0-9A-F]{8}) ([0-9A-F]{8})$")


def literal(mnemonic, word, second):
    """The literal behind a 64-bit instruction, or None: it has one where a source's field is 255."""
    if not re.search(r"_[bfiu]64", mnemonic):
        return None
    if word >> 23 == 0b101111101:                       # SOP1
        fields = [word & 255]
    elif word >> 23 in (0b101111110, 0b101111111) or word >> 28 == 0b1011:       # SOPC, SOPP, SOPK
        fields = [word & 255, word >> 8 & 255] if word >> 23 == 0b101111110 else []
    elif word >> 30 == 0b10:                            # SOP2
        fields = [word & 255, word >> 8 & 255]
    elif word >> 31 == 0:                               # VOP1, VOP2, VOPC
        fields = [word & 511]
    else:
        fields = []
    return second if 255 in fields else None


def faults(text):
    """(address, instruction) of 64-bit instructions with a literal that needs none, and the number of those with any."""
    found, n = [], 0
    for line in text.splitlines():
        m = LINE.match(line)
        value = literal(m[1], int(m[3], 16), int(m[4], 16)) if m else None
        if value is None:
            continue
        n += 1
        if value <= 64 or value >= 0xfffffff0:
            found.append((m[2], line.split("//")[0].strip()))
    return found, n


def test_the_looking_over_itself():
    for line, have, bad in (("s_mov_b64 s[22:23], 0x0 // 000000001000: BE9601FF 00000000", 1, True),
                            ("s_mov_b64 s[22:23], 0 // 000000001000: BE960180", 0, False),
                            ("s_mov_b64 s[2:3], 0x80 // 000000001000: BE8201FF 00000080", 1, False),
                            ("s_mov_b64 s[2:3], 0xffffff00 // 000000001000: BE8201FF FFFFFF00", 1, False),
                            ("s_and_b64 s[2:3], s[4:5], 0x0 // 000000001000: 8682FF04 00000000", 1, True),
                            ("s_cmp_eq_u64 s[2:3], 0x0 // 000000001000: BF12FF02 00000000", 1, True),
                            ("v_mov_b64_e32 v[2:3], 0x0 // 000000001000: 7E0470FF 00000000", 1, True),
                            ("v_mov_b64_e32 v[2:3], 0x60 // 000000001000: 7E0470FF 00000060", 1, False),
                            ("s_mov_b32 s2, 0x0 // 000000001000: BE8200FF 00000000", 0, False),
                            ("v_add_f64 v[0:1], v[2:3], 0 // 000000001000: D2800000 00010102", 0, False),
                            ("s_load_dwordx2 s[4:5], s[0:1], 0x0 // 000000001000: C0060100 00000000", 0, False)):
        found, n = faults("\t" + line)
        assert n == have and bool(found) == bad, line


def test_no_constant_is_cut_off(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump here")
    import ane_amd.bridge as br
    shutil.copy(br.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    found, n = [], 0
    for name in sorted(os.listdir(tmp_path)):
        if name.endswith("gfx950"):
            f, some = faults(subprocess.run([OBJDUMP, "-d", name], cwd=tmp_path, check=True, capture_output=True, text=True).stdout)
            found += [(name,) + x for x in f]
            n += some
    assert n > 100
    assert not found, (len(found), found[:5])
