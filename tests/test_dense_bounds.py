"""Where the bf16 tile kernel's descriptors end (csrc/dense_bounds.hpp), tried on the host for every lane of a step: what the
operand has is before the end, what it does not have is behind it, whatever the row's length and stride."""
import os
import shutil
import subprocess

import pytest

from util import PKG_DIR

PROGRAM = r"""
#include "dense_bounds.hpp"
#include <cstdio>
#include <initializer_list>

// Straight: lane of tile row r, chunk c (of four) of the step at k0. A chunk beyond K is asked for behind any end by the kernel.
static int straight(int rows, int K, int ld)
{
    int wrong = 0;
    for (int k0 = 0; k0 < K + 32; k0 += 32) {
        const int krem = K - k0;
        const long end = alpha::tile_end_straight(rows, (unsigned)ld, krem);
        const long size = ((long)(rows - 1) * ld + (K + 7) / 8 * 8) * 2;     // the operand's bytes, its rows whole chunks long
        for (int r = 0; r < 256; r++)
            for (int c = 0; c < 4; c++) {
                if (c * 8 >= krem) continue;
                const long at = ((long)r * ld + c * 8) * 2;
                const bool read = at + 16 <= end;
                if (read != (r < rows)) wrong++;
                if (read && k0 * 2 + at + 16 > size) wrong++;
            }
        if (krem <= 0 && end > (long)(rows - 1) * ld * 2) wrong++;
    }
    return wrong;
}

// T: lane of k row r, chunk c of a tile of 256 columns that begins at column 0 of `columns` left.
static int transposed(int columns, int K, int ld)
{
    int wrong = 0;
    for (int k0 = 0; k0 < K + 32; k0 += 32) {
        const int krem = K - k0;
        const long end = alpha::tile_end_t(columns, (unsigned)ld, krem);
        const long size = ((long)(K - 1) * ld + (columns + 7) / 8 * 8) * 2;
        for (int r = 0; r < 32; r++)
            for (int c = 0; c < 32; c++) {
                const long at = ((long)r * ld + c * 8) * 2;
                const bool read = at + 16 <= end;
                if (read && (long)k0 * ld * 2 + at + 16 > size) wrong++;
                if (r < krem && c * 8 < columns && !read) wrong++;
                if (r >= krem && read) wrong++;
            }
    }
    return wrong;
}

int main()
{
    int wrong = 0;
    for (int K : {1, 7, 8, 9, 16, 23, 24, 25, 31, 32, 33, 40, 56, 63, 64, 65, 96, 1000})
        for (int more : {0, 8, 16, 24, 200})
            for (int rows : {1, 2, 3, 100, 127, 160, 255, 256}) {
                const int ld = (K + 7) / 8 * 8 + more;
                const int w = straight(rows, K, ld);
                if (w) printf("straight: %d rows, K %d, ld %d: %d\n", rows, K, ld, w);
                wrong += w;
            }
    for (int K : {1, 5, 31, 32, 33, 64, 70})
        for (int columns : {1, 8, 9, 40, 255, 256, 1000})
            for (int more : {0, 8, 64}) {
                const int w = transposed(columns, K, (columns + 7) / 8 * 8 + more);
                if (w) printf("k as rows: %d columns, K %d: %d\n", columns, K, w);
                wrong += w;
            }
    // the largest stride: no end wraps
    if (alpha::tile_end_straight(256, 1u << 22, 1 << 22) != (255ull * (1 << 22) + 32) * 2) wrong++;
    printf("%d wrong\n", wrong);
    return wrong != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not found")
def test_every_lane_of_a_step_reads_the_operand_and_nothing_behind_it(tmp_path):
    src, exe = tmp_path / "bounds.cpp", tmp_path / "bounds"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(PKG_DIR, "csrc"), "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0, r.stdout[-2000:]
