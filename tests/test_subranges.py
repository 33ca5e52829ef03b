"""The sub-ranges that the multi-query kernels walk a view in (CPU): subrange_keys and
subrange_end (dvattention_amd/csrc/dv_chunk.h), compiled for the host, over pages of 1 to
2^31 - 1 rows and ranges up to the last key an int can name.  The sub-ranges cover
[la, lb) in order, and the pages of each fit the page cache."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dvattention_amd", "csrc")
CAP = 2048  # page ids cached per sub-range

MAIN = r"""
#include <stdio.h>
#include "dv_chunk.h"
int main(int, char**) {
    using namespace dv::chunk;
    static_assert(kPageCap == %d, "entries");
    int bs, la, lb;
    while (scanf("%%d %%d %%d", &bs, &la, &lb) == 3) {
        const int span = subrange_keys(bs);
        int n = 0;
        printf("%%d", span);
        for (int sa = la, sbnd; sa < lb && n < 5000; sa = sbnd, ++n) {
            sbnd = subrange_end(sa, lb, span);
            printf(" %%d", sbnd);
        }
        printf("\n");
    }
}
""" % CAP


def test_subranges(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src, exe = tmp_path / "ranges.cpp", tmp_path / "ranges"
    src.write_text(MAIN)
    csrc = [f"-I{CSRC}", f"-I{os.path.join(os.path.dirname(os.path.dirname(CSRC)), 'include')}"]
    subprocess.run([hipcc, "-x", "hip", "--cuda-host-only", "-O1", "-std=c++17", *csrc, str(src), "-o", str(exe)],
                   check=True)
    last = 2 ** 31 - 1
    cases = [(bs, la, lb)
             for bs in (1, 5, 16, 24, 64, 4096, 524800, 524801, 1 << 20, 1049600, 1049601, 1 << 21, 3 << 20, 1 << 30, last)
             for la, lb in ((0, 1), (0, 32), (7, 300), (1000, 100000), (0, 2046 * min(bs, 1000) + 1),
                            (last - 2 ** 18 * min(bs, 4), last), (0, last if bs >= 4096 else 10 ** 6))]
    out = subprocess.run([str(exe)], input="\n".join("%d %d %d" % c for c in cases), capture_output=True, text=True,
                         check=True).stdout.splitlines()
    assert len(out) == len(cases)
    for (bs, la, lb), line in zip(cases, out):
        span, *ends = (int(x) for x in line.split())
        assert 0 < span <= 2 ** 30 and span == min((CAP - 2) * bs, 2 ** 30) or bs > 2 ** 30 // (CAP - 2) and span == 2 ** 30
        starts = [la] + ends[:-1]
        assert ends[-1] == lb and all(a < b <= a + span for a, b in zip(starts, ends))
        # from row bs - 1 of a page on
        assert -(-(bs - 1 + span) // bs) <= CAP
