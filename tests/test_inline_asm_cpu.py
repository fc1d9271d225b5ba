"""What the kernels' inline assembly owes the compiler, read from the sources."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "recommendsystem_amd", "csrc")


def statements():
    """The instructions of every asm statement: (file, list of them)."""
    for f in sorted(glob.glob(os.path.join(CSRC, "*.h*"))):
        for m in re.finditer(r"\basm\s*(?:volatile)?\s*\(\s*((?:\"(?:[^\"\\]|\\.)*\"\s*)+)", open(f).read()):
            text = "".join(re.findall(r"\"((?:[^\"\\]|\\.)*)\"", m.group(1)))
            yield os.path.basename(f), [i.strip() for i in re.split(r"\\n|\\t|;", text) if i.strip()]


def test_m0_is_given_back():
    """m0 is reserved: no clobber list may name it, and the compiler may keep a value in it across any statement."""
    seen = 0
    for f, ins in statements():
        writes = [i for i in ins if re.match(r"s_\w+\s+m0\b", i)]
        if writes:
            seen += 1
            save = re.fullmatch(r"s_mov_b32 (%\d), m0", ins[0])
            assert save and ins[-1] == f"s_mov_b32 m0, {save.group(1)}", (f, ins)
    assert seen >= 1
