"""What the kernels' inline assembly tells the compiler about itself (no GPU)."""
import glob
import os
import re

from rhizome_amd import build

BLOCK = re.compile(r"\basm\s+volatile\s*\((.*?)\)\s*;", re.S)


def blocks():
    for path in sorted(glob.glob(os.path.join(build.CSRC, "*"))):
        for block in BLOCK.findall(open(path).read()):
            yield os.path.basename(path), block


def test_m0_comes_from_the_compiler():
    """A load into LDS takes its place there from m0: as an operand, so that the
    compiler sets the register and knows it; a block that wrote it would do so
    behind the compiler's back (it is reserved, and no clobber names it)."""
    loads = [(name, block) for name, block in blocks() if "_load_lds_" in block]
    assert len(loads) >= 3
    for name, block in loads:
        assert '"{m0}"' in block, f"{name}: {block}"
    for name, block in blocks():
        assert not re.search(r"\bs_\w+ m0\b", block), f"{name}: {block}"
