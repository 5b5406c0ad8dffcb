"""The loads of the linear layers' operands (panel_walk.h): every load of every tile, slice and step asks for the right 16 bytes or is kept
out by its vector offset, and none reaches past the tensor, whether the range check counts the scalar offset or not.  The header is
compiled for the host."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ane_amd", "csrc")

PROGRAM = r"""
#include "panel_walk.h"
#include <stdio.h>
#include <stdlib.h>
#include <initializer_list>
typedef unsigned long long u64;
static long checked = 0;

// One workgroup's walk over steps [sum0, sum1) for the B indexes from index0 on; some of the threads and steps of a long one.
template <int B, bool COLUMNS, int THREADS>
static void walk(int rows, int S, int cols, int index0, int sum0, int sum1) {
    typedef PanelWalk<B, COLUMNS, THREADS> W;
    const u64 total = (u64)rows * cols * 2;
    const bool big = total > 1 << 24;
    for (int t = 0; t < THREADS; t += big ? 37 : 1) {
        W w = {};
        u64 base = w.begin(rows, S, cols, index0, sum0, t);
        for (int at = sum0; at < sum1; at += 64) {
            const int left = sum1 - at;
            const u64 room = w.bytes < 0xffffff00ull ? w.bytes : 0xffffff00ull;
            for (int i = 0; i < W::PANELS; i++)
                for (int j = 0; j < W::PER; j++, checked++) {
                    const int row = t / 8 + j * W::APART, chunk = (t % 8) ^ panel_swz(row);
                    const u64 r = COLUMNS ? (u64)at + row : (u64)index0 + row, n = COLUMNS ? index0 + i * 64 + chunk * 8 : at + chunk * 8;
                    const bool there = COLUMNS ? row < left && n < (u64)cols : r < (u64)rows && chunk * 8 < left;
                    const unsigned v = w.plain(left) ? w.voff[i] : w.voffset(i, j, left, t), s = w.soffset(j);
                    const u64 want = ((n / S * rows + r) * S + n % S) * 2;
                    bool ok;
                    if (!there) ok = v == OUTSIDE;
                    else ok = v != OUTSIDE && base + v + s == want && want + 16 <= total && (u64)v + s + 16 <= room;
                    if (!ok) {
                        printf("B %d columns %d threads %d: %d rows of %d, S %d, index %d sum %d of %d..%d, thread %d panel %d load %d: voffset %u soffset %u\n",
                               B, COLUMNS, THREADS, rows, cols, S, index0, at, sum0, sum1, t, i, j, v, s);
                        exit(1);
                    }
                }
            base += w.advance();
        }
    }
}

// every tile of a tensor, the sum in one piece and in slices of four panels
template <int B, int THREADS>
static void tensor(int rows, int S, int batch) {
    const int cols = S * batch;
    if (cols > S && (256.0 / S + 2) * rows * S * 2 + 512.0 * S >= 4e9) return;      // (such a tensor is copied first)
    const bool big = (double)rows * cols > 1 << 23;
    for (int slice : {1 << 30, 256}) {
        if (big && slice == 256) continue;
        for (int i0 = big ? (cols - 1) / B * B : 0; i0 < cols; i0 += B)
            for (int s0 = 0; s0 < rows; s0 += slice < rows ? slice : rows)
                walk<B, true, THREADS>(rows, S, cols, i0, s0, slice < rows - s0 ? s0 + slice : rows);
        for (int i0 = big ? (rows - 1) / B * B : 0; i0 < rows; i0 += B)
            for (int s0 = 0; s0 < cols; s0 += slice < cols ? slice : cols)
                walk<B, false, THREADS>(rows, S, cols, i0, s0, slice < cols - s0 ? s0 + slice : cols);
    }
    // a sum that ends within the last chunks (the columns behind it are a copy's zeros)
    for (int end : {cols - 1, cols - 7}) if (end > 0 && !big) walk<B, false, THREADS>(rows, S, cols, 0, 0, end);
}
int main() {
    const int sizes[][3] = {{1, 8, 1}, {3, 8, 9}, {64, 64, 1}, {65, 64, 3}, {70, 72, 1}, {33, 40, 3}, {130, 256, 2}, {9, 520, 1}, {96, 1024, 1}, {100, 8, 40},
                            {255, 136, 5}, {257, 200, 3}, {300, 24, 11}, {512, 128, 4}, {1000, 8, 1}, {77, 4096, 1}, {200, 1608, 1}, {385, 320, 2},
                            {1100, 1 << 21, 1}, {1100, (1 << 21) - 8, 1}, {1 << 22, 512, 1}, {1 << 22, 264, 1}, {1 << 20, 8, 33}, {300, 1 << 22, 1}, {300, (1 << 22) - 56, 1}};
    for (auto &s : sizes) {
        tensor<64, 256>(s[0], s[1], s[2]);
        tensor<128, 512>(s[0], s[1], s[2]);
        tensor<256, 512>(s[0], s[1], s[2]);
        fflush(stdout);
    }
    printf("%ld\n", checked);
    return 0;
}
"""


def test_every_load_of_every_walk(tmp_path):
    src, exe = tmp_path / "walk.cpp", tmp_path / "walk"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and int(out.stdout) > 1000000, out.stdout
