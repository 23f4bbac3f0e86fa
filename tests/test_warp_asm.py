"""Inline assembly that all lanes of a warp execute together (`.sync`) has to
be volatile: the compiler may move an asm without that into a branch that only
some lanes take, when its results are used only there.  Read from the sources."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "ouroboros-kernelsmith_b200", "csrc")


def statements():
    """(file, line, text) of every asm statement."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        src = re.sub(r"//[^\n]*", "", open(path).read())
        for m in re.finditer(r"\basm\b(.*?);\s*\n", src, flags=re.S):
            yield os.path.basename(path), src.count("\n", 0, m.start()) + 1, m.group(1)


def test_warp_collective_asm_is_volatile():
    found = 0
    for name, line, text in statements():
        if re.search(r"\.sync\b|\bbar\.sync", text):
            found += 1
            assert text.lstrip().startswith("volatile"), f"{name}:{line}: .sync without volatile"
    assert found >= 6   # the products' mma, the transposition, the named barrier
