"""LDS-DMA written as inline asm holds its own wait states.

On gfx9 a vector memory instruction that reads an SGPR needs five wait states
after a vector instruction wrote it.  The descriptors of these loads come from
v_readfirstlane (or v_readlane, where the compiler has spilled them), and the
compiler counts the states for its own instructions only: with two in the asm
block, the correlation losses' gradient had loads two and three states behind the
write of their descriptor's address."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "droid-slam_amd", "csrc")
FILES = sorted(glob.glob(os.path.join(CSRC, "*.h*")) + glob.glob(os.path.join(CSRC, "ab", "*.inc")))


def _states(lines):
    """Wait states of the instructions in front of the load."""
    n = 0
    for ln in lines:
        m = re.match(r"s_nop\s+(\d+)$", ln)
        n += int(m.group(1)) + 1 if m else 1
    return n


def test_every_lds_dma_block_waits_for_its_descriptor():
    found = 0
    for path in FILES:
        for m in re.finditer(r'asm\s+volatile\(\s*"((?:[^"\\]|\\.)*)"', open(path).read()):
            lines = [ln.strip() for ln in m.group(1).replace("\\t", "").split("\\n") if ln.strip()]
            for k, ln in enumerate(lines):
                if re.match(r"(buffer|global)_load\w* .*\blds$", ln):
                    found += 1
                    assert _states(lines[:k]) >= 5, "%s: %s" % (os.path.basename(path), " / ".join(lines))
    assert found >= 4
