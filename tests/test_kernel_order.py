"""What the built kernels of the gated front rely on without a value to show for it: the order of loads where a step barrier
waits for a counted number of them, and stores whose range check has to see their whole offset.

A step ends with a wait that leaves the youngest `pend` loads open, counted by hand for one order of issue: an LDS DMA that
the compiler put behind loads it should precede would be left open, and other waves would read LDS before it has
landed.  The GPU code of the built library is listed with llvm-objdump and its loads are read off between the barriers."""
import os
import re
import shutil
import subprocess

import pytest

import gq

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
Q4_0, Q8_0, Q4_K, Q6_K = gq.FMT_Q4_0, gq.FMT_Q8_0, gq.FMT_Q4_K, gq.FMT_Q6_K

pytestmark = pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: instruction lines} of the gated front's kernels."""
    tmp = tmp_path_factory.mktemp("code")
    lib = shutil.copy(gq.LIB_PATH, tmp)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True, cwd=tmp)
    out = {}
    for f in sorted(tmp.iterdir()):
        if not f.name.endswith("gfx950"):
            continue
        names = subprocess.run([OBJDUMP, "-t", f], check=True, capture_output=True, text=True).stdout
        if "k_front_dx" not in names:
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], check=True, capture_output=True, text=True).stdout
        lines = []
        for line in text.splitlines():
            m = re.match(r"[0-9a-f]+ <(.*)>:", line)
            if m:
                lines = out.setdefault(m[1], [])
            else:
                lines.append(line.strip())
    return {n: t for n, t in out.items() if "k_front_" in n}


def instances(kernels, name):
    """(template arguments, lines) of every instantiation."""
    found = []
    for n, lines in kernels.items():
        m = re.search(name + r"I((?:Li\d+E)+)E", n)
        if m:
            found.append((tuple(int(v) for v in re.findall(r"Li(\d+)E", m[1])), lines))
    assert found
    return found


def loads(lines):
    """The vector memory loads between the barriers, in order: D an LDS DMA, v a load into registers."""
    parts = [""]
    for line in lines:
        if line.startswith("s_barrier"):
            parts.append("")
        elif re.match(r"(buffer|global|flat)_load", line):
            parts[-1] += "D" if re.search(r"\blds\b", line) else "v"
    return parts


def test_backward_loads(kernels):
    seen = set()
    for (fmt, wn, kg, tm, pd), lines in instances(kernels, "k_front_dx"):
        nd = 32 * tm // (8 * wn) + 4 * (2 if fmt in (Q8_0, Q6_K) else 1)
        sl = 2 if fmt == Q6_K else 1
        parts = loads(lines)
        what = f"k_front_dx<{fmt},{wn},{kg},{tm},{pd}>: {parts[:pd + 1]}"
        assert parts[0] == "v" * sl + "D" * (nd * (pd - 1)) + "v" * sl, what
        for p in parts[1:pd + 1]:
            assert p == "D" * nd + "v" * sl, what
        assert not any("D" in p for p in parts[pd + 1:]), what
        seen.add(fmt)
    assert seen == {Q4_0, Q8_0, Q4_K, Q6_K}


def test_forward_loads(kernels):
    per_column = {Q4_0: 3, Q8_0: 3, Q4_K: 3, Q6_K: 6}  # loads of a weight column block and step
    seen = set()
    for (fmt, bm, wn, nj, pd, kg), lines in instances(kernels, "k_front_rb"):
        na, nw = bm // (8 * wn), 2 * per_column[fmt] * nj
        parts = loads(lines)
        what = f"k_front_rb<{fmt},{bm},{wn},{nj},{pd},{kg}>: {parts[:pd + 1]}"
        # (one more load: the row scales, whose place is free, since the wait for them comes before the first barrier)
        first = ("D" * na + "v" * nw) * (pd - 1) + "v" * nw
        assert parts[0] in ("v" + first, first + "v"), what
        for p in parts[1:pd + 1]:
            assert p == "D" * na + "v" * nw, what
        assert not any("D" in p for p in parts[pd + 1:]), what
        seen.add(fmt)
    assert seen == {Q4_0, Q8_0, Q4_K, Q6_K}


def test_store_offsets(kernels):
    """Rows past the last are kept out of memory by a buffer's range, which is only sure to count the lane's offset: no
    store of the front has a scalar one."""
    n = 0
    for (fmt, bm, wn, nj, pd, kg), lines in instances(kernels, "k_front_rb"):
        for line in lines:
            m = re.match(r"buffer_store_\w+ \w+, v\d+, s\[\d+:\d+\], (\S+) ", line)
            assert m or not line.startswith("buffer_store"), line
            if m:
                n += 1
                assert m[1] == "0", f"k_front_rb<{fmt},{bm},{wn},{nj},{pd},{kg}>: {line}"
    assert n > 0
