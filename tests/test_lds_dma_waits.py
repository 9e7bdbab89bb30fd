"""LDS-DMA written as inline asm keeps the wait states that the compiler counts for
its own loads only.

On gfx9 a vector memory instruction that reads an SGPR needs five wait states after
a vector instruction wrote it.  The descriptors of some of these loads come from
v_readfirstlane (or v_readlane, where the compiler has spilled them): the
correlation losses' gradient had loads two and three states behind it.  Checked in
the built libraries, over every path that reaches a load."""
import bisect
import glob
import os
import re
import shutil
import subprocess

import pytest

LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "droid-slam_amd", "lib")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def _sgprs(text):
    out = {int(a) for a in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        out |= set(range(int(a), int(b) + 1))
    return out


def _too_early(listing):
    """(load, write, wait states) of every LDS load that reads a vector
    instruction's SGPR less than five wait states after it, and the loads' number."""
    code, base, name, targets = [], {}, None, []
    for ln in listing.splitlines():
        m = re.match(r"^([0-9a-f]+) <(.+)>:$", ln)
        if m:
            name, base[m.group(2)] = m.group(2), int(m.group(1), 16)
            continue
        m = re.match(r"^\s+(\S.*?)\s*// ([0-9A-F]+):(.*)$", ln)
        if m and name:
            code.append((int(m.group(2), 16), m.group(1)))
            t = re.search(r"<(.+?)(?:\+0x([0-9a-f]+))?>", m.group(3))
            if t and m.group(1).startswith(("s_cbranch", "s_branch")):
                targets.append((len(code) - 1, t.group(1), int(t.group(2) or "0", 16)))
    at = [a for a, _ in code]
    jumps = {}
    for k, sym, off in targets:
        jumps.setdefault(bisect.bisect_left(at, base[sym] + off), []).append(k)
    bad, loads = [], 0
    for k, (_, text) in enumerate(code):
        if not re.match(r"(buffer|global)_load\w* .*\blds$", text):
            continue
        loads += 1
        seen, todo = set(), [(k, 0)]
        used = _sgprs(text)
        while todo:
            i, states = todo.pop()
            if (i, states) in seen or states >= 5:
                continue
            seen.add((i, states))
            before = list(jumps.get(i, []))
            if i and not code[i - 1][1].startswith(("s_branch", "s_endpgm", "s_setpc")):
                before.append(i - 1)
            for p in before:
                t = code[p][1]
                dst = t.split(None, 1)[1].split(",")[0] if t.startswith("v_") and " " in t else ""
                if dst.startswith("s") and _sgprs(dst) & used:
                    bad.append((text, t, states))
                n = int(t.split()[1], 0) + 1 if t.startswith("s_nop") else 1
                todo.append((p, states + n))
    return bad, loads


def test_the_count_itself():
    head = "0000000000000000 <k>:\n"
    ins = lambda *texts: head + "".join("\t%s   // %012X: 00000000\n" % (t, 4 * n) for n, t in enumerate(texts))
    load = "buffer_load_dword v1, s[4:7], 0 offen lds"
    write = "v_readfirstlane_b32 s5, v2"
    for gap, early in ((("s_nop 3",), True), (("s_nop 4",), False), (("s_mov_b32 m0, s1", "s_nop 0"), True),
                       (("s_mov_b32 m0, s1", "s_nop 3"), False), ((), True)):
        bad, loads = _too_early(ins(write, *gap, load))
        assert loads == 1 and bool(bad) == early, gap
    assert not _too_early(ins("v_readfirstlane_b32 s8, v2", load))[0]
    # over a branch: the write's block jumps to the load
    text = ins(write, "s_branch 1", "s_endpgm", load).replace("s_branch 1   // 000000000004: 00000000",
                                                              "s_branch 1   // 000000000004: 00000000 <k+0xc>")
    assert _too_early(text)[0]


@pytest.mark.parametrize("lib", ["libdroid_hip.so", os.path.join("ab", "libdroid_hip.so")])
def test_every_lds_load_of_the_library(lib, tmp_path):
    path = os.path.join(LIB, lib)
    if not os.path.exists(path) or not os.path.exists(OBJDUMP):
        pytest.skip("needs the built library and ROCm's llvm-objdump")
    shutil.copy(path, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    total = 0
    for obj in glob.glob(str(tmp_path / "*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", obj], check=True, capture_output=True, text=True).stdout
        bad, loads = _too_early(text)
        total += loads
        assert not bad, bad[:4]
    assert total > 100
