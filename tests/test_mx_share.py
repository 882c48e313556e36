"""How a decode launch of the MX4 products divides its weight units over the CTAs: the kernel's
own arithmetic (csrc/mx_share.cuh), compiled for the host."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "easyinfra_b200", "csrc")
MAIN = """
#include "mx_share.cuh"
extern "C" void shares(unsigned total, unsigned u, unsigned grid, unsigned* out) {
  for (unsigned b = 0; b < grid; ++b) {
    const b200moe::MxShare s = b200moe::mx_share(total, u, grid, b);
    out[2 * b] = s.pos;
    out[2 * b + 1] = s.end;
  }
}
"""


@pytest.fixture(scope="module")
def shares(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    d = tmp_path_factory.mktemp("share")
    src, so = d / "share.cpp", d / "share.so"
    src.write_text(MAIN)
    subprocess.run(["g++", "-O1", "-shared", "-fPIC", "-x", "c++", "-I", CSRC, "-o", str(so), str(src)], check=True)
    fn = ctypes.CDLL(str(so)).shares
    fn.argtypes = [ctypes.c_uint, ctypes.c_uint, ctypes.c_uint, ctypes.c_void_p]

    def run(total, u, grid):
        out = (ctypes.c_uint * (2 * grid))()
        fn(total, u, grid, out)
        return list(zip(out[::2], out[1::2]))
    return run


# segments (experts' m-tiles) and units of 64 weight rows in each; the last ones have more
# units than 2^32 / 148
@pytest.mark.parametrize("segs,u", [(0, 2), (1, 2), (8, 24), (8, 12), (60, 32), (128, 24), (1, 176), (7, 448), (300, 44),
                                    (1, 2 ** 24), (1, 2 ** 25 - 2), (2, 2 ** 25 - 2), (60, 2 ** 25 - 2), (1, 2 ** 31 - 2)])
@pytest.mark.parametrize("grid", [1, 2, 4, 147, 148])
def test_shares_cover_every_unit_once(shares, segs, u, grid):
    total = segs * u
    assert total < 2 ** 31
    got = shares(total, u, grid)
    at = 0
    for pos, end in got:
        assert pos == at and end >= pos
        at = end
    assert at == total
    sizes = [end - pos for pos, end in got]
    largest = -(-total // grid)
    assert max(sizes) <= largest + largest // 8            # what the rule promises
    parts = grid // segs if segs else 0
    if parts and -(-u // parts) <= largest + largest // 8:  # equal parts of every segment
        want = [s * u + i * u // parts for s in range(segs) for i in range(parts)]
        assert [pos for pos, _ in got[:segs * parts]] == want
    else:
        assert max(sizes) - min(sizes) <= 1
