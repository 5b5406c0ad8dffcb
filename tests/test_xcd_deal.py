"""Units of work dealt to the XCDs (xcd.h): each once, neighbours together, and of a launch of two kinds an even share of each to every XCD,
the first kind's first.  The header is compiled for the host."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ane_amd", "csrc")

PROGRAM = r"""
#include "xcd.h"
#include <stdio.h>
#include <vector>
int main() {
    long launches = 0;
    for (int n0 = 0; n0 <= 70; n0++)
        for (int n1 = 0; n1 <= 130; n1++, launches++) {
            const int n = n0 + n1;
            std::vector<int> seen(n, 0), of[2][8], all;
            for (int b = 0; b < n; b++) {
                const DealtUnit d = xcd_deal(b, n0, n);
                if (d.unit < 0 || d.unit >= (d.second ? n1 : n0)) return printf("%d + %d: workgroup %d\n", n0, n1, b), 1;
                seen[d.second ? n0 + d.unit : d.unit]++;
                if (!d.second && !of[1][b & 7].empty()) return printf("%d + %d: a first unit behind a second one\n", n0, n1), 1;
                of[d.second][b & 7].push_back(d.unit);
            }
            for (int u = 0; u < n; u++)
                if (seen[u] != 1) return printf("%d + %d: unit %d %d times\n", n0, n1, u, seen[u]), 1;
            for (int kind = 0; kind < 2; kind++)
                for (int x = 0; x < 8; x++) {
                    const auto &mine = of[kind][x];
                    const int share = (kind ? n1 : n0) / 8;
                    if ((int)mine.size() < share || (int)mine.size() > share + 1) return printf("%d + %d: XCD %d has %d of kind %d\n", n0, n1, x, (int)mine.size(), kind), 1;
                    for (size_t i = 1; i < mine.size(); i++)
                        if (mine[i] != mine[i - 1] + 1) return printf("%d + %d: XCD %d, units apart\n", n0, n1, x), 1;
                }
        }
    printf("%ld\n", launches);
    return 0;
}
"""


def test_every_unit_of_every_launch(tmp_path):
    src, exe = tmp_path / "deal.cpp", tmp_path / "deal"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and int(out.stdout) > 1000, out.stdout
