"""The built tiled kernel of the product with its epilogue: the order of its loads, which its step barriers count on, and stores whose range
check sees their whole offset (as in test_kernel_order, for k_lin_rb)."""
import os
import re
import shutil
import subprocess

import pytest

import gq
from test_kernel_order import OBJDUMP, Q4_0, Q4_K, Q6_K, Q8_0, instances, loads

pytestmark = pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: instruction lines} of the tiled kernels."""
    tmp = tmp_path_factory.mktemp("code")
    lib = shutil.copy(gq.LIB_PATH, tmp)
    subprocess.run([OBJDUMP, "--offloading", lib], check=True, capture_output=True, cwd=tmp)
    out = {}
    for f in sorted(tmp.iterdir()):
        if not f.name.endswith("gfx950"):
            continue
        names = subprocess.run([OBJDUMP, "-t", f], check=True, capture_output=True, text=True).stdout
        if "k_lin_rb" not in names:
            continue
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], check=True, capture_output=True, text=True).stdout
        lines = []
        for line in text.splitlines():
            m = re.match(r"[0-9a-f]+ <(.*)>:", line)
            if m:
                lines = out.setdefault(m[1], [])
            else:
                lines.append(line.strip())
    return {n: t for n, t in out.items() if "k_lin_rb" in n}


def test_loads(kernels):
    per_column = {Q4_0: 3, Q8_0: 3, Q4_K: 3, Q6_K: 6}  # loads of a weight column block and step
    seen = set()
    for (fmt, bm, wn, nj, pd, kg), lines in instances(kernels, "k_lin_rb"):
        na, nw = bm // (8 * wn), per_column[fmt] * nj
        parts = loads(lines)
        what = f"k_lin_rb<{fmt},{bm},{wn},{nj},{pd},{kg}>: {parts[:pd + 2]}"
        # (one more load: the row scales, whose place is free, since the wait for them comes before the first barrier)
        first = ("D" * na + "v" * nw) * (pd - 1) + "v" * nw
        assert parts[0] in ("v" + first, first + "v"), what
        for p in parts[1:pd + 1]:
            assert p == "D" * na + "v" * nw, what
        assert not any("D" in p for p in parts[pd + 1:]), what
        seen.add(fmt)
    assert seen == {Q4_0, Q8_0, Q4_K, Q6_K}


def test_store_offsets(kernels):
    """Rows past the last are kept out of memory by a buffer's range, which is only sure to count the lane's offset: no load or store of
    outputs has a scalar one."""
    stores = residuals = 0
    for (fmt, bm, wn, nj, pd, kg), lines in instances(kernels, "k_lin_rb"):
        for line in lines:
            store = line.startswith("buffer_store")
            # residuals are loaded one at a time, by 16 or 32 bits; so are Q6_K's scales, with a scalar offset that stays in range
            resid = fmt != Q6_K and re.match(r"buffer_load_(ushort|dword) ", line)
            if store or resid:
                m = re.match(r"buffer_\w+ \w+, v\d+, s\[\d+:\d+\], (\S+) ", line)
                assert m and m[1] == "0", f"k_lin_rb<{fmt},{bm},{wn},{nj},{pd},{kg}>: {line}"
                stores, residuals = stores + bool(store), residuals + bool(resid)
    assert stores > 0 and residuals > 0
