"""How the prefix attention over 8-bit pages cuts its tiles (csrc/sxq_paged.h), enumerated on the CPU as
the kernel uses it: pieces and cut tiles stay within the workspace's room, sizes within 32 bits; and the
workspaces it asks for."""
import ctypes
import os
import shutil
import subprocess

import pytest

from syrinx_amd import _lib
from syrinx_amd.paged import KvPages

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = r"""
#include <cstdint>
#include <cstdio>
#include <vector>
#include "sxq_paged.h"
using namespace sxq;
#define EXPECT(c) do { if (!(c)) { std::printf("failed: %s\n", #c); return 1; } } while (0)

int main() {
    // of one tile: a quarter more than a share stays whole, else the fewest pieces of a share or less
    for (int piece = 1; piece <= 300; ++piece)
        for (int keys = 0; keys <= 3000; ++keys) {
            const int n = kv_pieces(keys, piece);
            EXPECT((n > 1) == (4 * keys > 5 * piece));
            if (n > 1) EXPECT((n - 1) * piece < keys && keys <= n * piece);
            // and no more than 8/5 of its shares
            if (n > 1) EXPECT(5 * (int64_t)n * piece <= 8 * (int64_t)keys);
        }
    // the largest there are
    for (int piece : {1, 2, 3, 1 << 10, 1 << 29, 1 << 30, (1 << 30) + (1 << 20) + 511})
        for (int keys : {0, 1, 1 << 24, 1 << 25, 1 << 30}) {
            const int64_t k = keys, p = piece;
            EXPECT(kv_pieces(keys, piece) == (4 * k > 5 * p ? (k + p - 1) / p : 1));
        }
    // any tiles: fewer pieces of cut ones than 2 * places, fewer cut ones than places
    uint32_t r = 1;
    auto next = [&](int n) { r = r * 1664525u + 1013904223u; return (int)((r >> 8) % (uint32_t)n); };
    for (int turn = 0; turn < 20000; ++turn) {
        const int places = 1 + next(512), least = next(2) ? 1 : 4, tiles = 1 + next(turn % 8 ? 60 : 2500), top = 1 << (1 + next(20));
        std::vector<int> keys(tiles);
        int64_t work = 0;
        for (int& k : keys) work += k = next(next(4) ? top : top / 2 + 1);
        const int64_t share = (work + places - 1) / places, piece = share < least ? least : share;
        int64_t cut = 0, pieces = 0;
        for (int k : keys) {
            const int n = kv_pieces(k, (int)piece);
            if (n > 1) ++cut, pieces += n;
        }
        EXPECT(cut <= places && pieces <= 2 * places);
    }
    std::printf("ok\n");
}
"""


def test_pieces(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not installed")
    src, exe = tmp_path / "cut.cpp", tmp_path / "cut"
    src.write_text(DRIVER)
    subprocess.run([gxx, "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "syrinx_amd", "csrc"), str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def _workspace(nh, nkv, hd, n_q):
    p, size = KvPages(24, nkv, hd, 32, 4, None, None, nkv * 32 * hd, 32 * hd, hd, None, None, nkv * 2, 2), ctypes.c_size_t()
    assert _lib.lib().sxq_kv_prefix_attention_workspace(ctypes.byref(p), n_q, nh, ctypes.byref(size)) == _lib.OK
    return size.value


@pytest.mark.parametrize("nh,nkv,hd", [(32, 8, 128), (14, 2, 64), (16, 1, 256), (64, 1, 128), (8, 8, 16), (300, 2, 64)])
def test_a_workspace_is_of_the_tiles_that_its_calls_take(nh, nkv, hd):
    """Calls of few rows are taken by tiles of 32 of them: their workspace has no room for the pieces of
    tiles of 128.  More queries never need less: a workspace is good for any smaller call."""
    few, many = 1, 1 + 32768 // nh
    assert 3 * _workspace(nh, nkv, hd, few) < _workspace(nh, nkv, hd, many)
    sizes = [_workspace(nh, nkv, hd, n) for n in range(1, 2 * many, max(1, many // 300))]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))
