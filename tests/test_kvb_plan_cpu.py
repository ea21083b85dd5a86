"""The shares that prompt attention over the block-scaled KV cache deals its tiles
out in (csrc/kvb_plan.cuh), compiled for the host: they are 64-bit sums, and a
million rows of 64 query heads on one KV head pass 2^31."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
SOURCE = r"""
#include <cstdio>
#include <cstdlib>
#include "kvb_plan.cuh"
using namespace w8a8;
int main(int, char** v) {
    const int most = 148, heads = atoi(v[1]), units = atoi(v[2]), tiles0 = atoi(v[3]), grow = atoi(v[4]);
    // unit u: tiles0 + grow * u tiles
    auto before = [&](int u) { return (int64_t)u * (kUnitCost + tiles0) + (int64_t)grow * u * (u - 1) / 2; };
    auto tiles = [&](int u) { return tiles0 + grow * u; };
    for (int c = 0; c < most; ++c) {
        const RowsShare w = share_of(c, most, before(units), heads, units, before, tiles);
        printf("%lld %lld %d %d %d\n", (long long)w.lo, (long long)w.hi, w.h, w.u, w.join);
    }
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("plan")
    (d / "plan.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "torch2riscv_accelerator_b200", "csrc"),
                    str(d / "plan.cpp"), "-o", str(d / "plan")], check=True)
    return str(d / "plan")


@pytest.mark.parametrize("heads,units,tiles0,grow", [
    (1, 1, 1, 0), (2, 3, 5, 0), (8, 40, 1, 1), (3, 200, 16, 0),
    (1, 65536, 1, 1),                                        # 2^31 tiles: units of up to 65,536
    (1, 524288, 4096, 0), (2, 524288, 4096, 0), (1, 100000, 50000, 0), (9, 1000003, 70001, 0)])
def test_shares_of_any_size(program, heads, units, tiles0, grow):
    out = subprocess.run([program, str(heads), str(units), str(tiles0), str(grow)], capture_output=True, text=True, check=True)
    shares = [tuple(map(int, line.split())) for line in out.stdout.splitlines()]
    before = lambda u: u * (2 + tiles0) + grow * u * (u - 1) // 2
    total = before(units)
    work = total * heads
    ctas = min(work, 148)
    assert [s[:2] for s in shares[:ctas]] == [(work * c // ctas, work * (c + 1) // ctas) for c in range(ctas)]
    assert all(lo == hi and join == -1 for lo, hi, _, _, join in shares[ctas:])
    for c, (lo, hi, h, u, join) in enumerate(shares[:ctas]):
        begin, end = h * total + before(u), h * total + before(u + 1)
        assert begin <= lo < end and 0 <= h < heads and 0 <= u < units
        # the first share that begins inside the unit's tiles joins it, up to the one that holds its last tile
        first = lo > begin + 2 and (c == 0 or shares[c - 1][0] <= begin + 2)
        last = next(i for i in range(c, ctas) if shares[i][1] >= end)
        assert join == (last if first else -1)
