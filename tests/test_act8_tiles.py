"""The tile rule of the plane kernels (csrc/act8.h) on the host: every shape gets a kernel that is built, and every kernel that is built is
some shape's."""
import os
import shutil
import subprocess

import pytest

import __graft_entry__ as g

SOURCE = r"""
#include "act8.h"
#include <cstdio>
#include <set>
#include <tuple>
#include <vector>
int main() {
    const std::vector<int> planes{8, 9, 15, 16, 17, 24, 31, 33, 40, 63, 64, 65, 72, 100, 120, 128, 129, 176, 200, 250, 256, 257, 300, 361, 511, 512, 513, 777, 1000,
                                  1024, 2047, 2048, 2500, 4096, 5000, 8192, 16384, 65536, 1 << 20};
    for (const auto& mb : std::vector<std::pair<int, int>>{{8, 2}, {4, 4}, {8, 4}}) {
        const int most = mb.first, bytes = mb.second;
        std::set<std::tuple<int, int, int>> seen;
        for (int C = 1; C <= 520 * most; ++C)
            for (int HW : planes)
                for (long long N : {1, 2, 3, 7, 16, 33, 75, 100, 149, 150, 200, 255, 256, 3000}) {
                    const TileCfg t = tile_pick(N, C, HW, most, bytes);
                    if (!t.lpx) continue;
                    const int cpt = t.cpt <= 1 ? 1 : t.cpt <= 2 ? 2 : t.cpt <= 4 ? 4 : 8;
                    if (t.cpt > most || t.cpt * t.nw * 64 / t.lpx < C) { printf("tile too small: N %lld C %d HW %d\n", N, C, HW); return 1; }
                    if (!tile_used(t.lpx, cpt, t.nw, most, bytes)) { printf("not built: lpx %d cpt %d waves %d, N %lld C %d HW %d\n", t.lpx, cpt, t.nw, N, C, HW); return 1; }
                    seen.insert({t.nw, t.lpx, cpt});
                }
        for (int nw : {4, 8})
            for (int lpx = nw == 4 ? 32 : 8; lpx >= 1; lpx >>= 1)
                for (int cpt = 1; cpt <= most; cpt <<= 1)
                    if (tile_used(lpx, cpt, nw, most, bytes) && !seen.count({nw, lpx, cpt})) { printf("never asked for: lpx %d cpt %d waves %d, %d %d\n", lpx, cpt, nw, most, bytes); return 1; }
    }
    puts("ok");
}
"""


def test_tiles_that_are_built_are_those_that_shapes_ask_for(tmp_path):
    hipcc = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    src, exe = tmp_path / "tiles.hip", tmp_path / "tiles"
    src.write_text(SOURCE)
    subprocess.check_call([hipcc, "--offload-arch=gfx950", "--offload-host-only", "-O1", "-std=c++17", "-I" + os.path.join(g.PKG, "csrc"), str(src), "-o", str(exe)],
                          stderr=subprocess.DEVNULL)
    assert subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True).stdout.strip() == "ok"


def test_counts_near_32_bits(hific):
    """Rows up to 2^31 - 1: the workspace of the backward pass stays the one of a little fewer."""
    from hific_amd import lib
    ws = lib.raw("hific_norm8_bwd_ws_bytes")
    for c in (8, 64, 129, 960, 4096, 16384):
        want = ws(2 ** 31 - 2000, c, 1)
        assert 0 < want < 1 << 30
        for n in (2 ** 31 - 33, 2 ** 31 - 31, 2 ** 31 - 9, 2 ** 31 - 1):
            assert ws(n, c, 1) == want, (n, c)
