"""How attention over a paged cache deals out its tiles (deal.h, compiled for the host): every tile has one workgroup, a shared unit's workgroups are
the ones that it waits for, also where the places of a launch are as many as 32 bits count.  No GPU."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ane_amd", "csrc")

PROGRAM = r"""
#include "deal.h"
#include <algorithm>
#include <climits>
#include <map>
#include <math.h>
#include <random>
#include <stdio.h>
#include <vector>
typedef long long ll;
constexpr int BEGIN = 8, SHORT = 9;

// A launch of columns with n tiles to each of their `units` units, from the definition, in 64 bits and unit by unit.
static int check(const std::vector<int> &n, int units, int most, int grain, int piece, int few) {
    ll total = 0;
    for (int t : n) total += t ? (ll)(t + BEGIN) * units : 0;
    if (total > INT_MAX) return puts("a test of more places than there are"), 1;
    int groups = deal_groups((int)total, most, grain);
    if (piece > 0) groups = deal_fewer(groups, (int)total, piece, units, few);
    ll want = std::min<ll>((total + grain - 1) / grain, most);
    if (piece > 0) {
        const ll pieces = ((total + piece - 1) / piece + units - 1) / units * units;
        if (pieces <= few) want = std::min(want, pieces);
    }
    if (groups != want) return printf("%d groups for %lld of %lld places, pieces of %d, %d units\n", groups, want, total, piece, units), 1;
    if (total == 0) return 0;
    const Deal d = deal_out((int)total, groups);
    if (d.border(0) != 0 || d.border(d.groups) != total) return puts("ends"), 1;
    for (int w = 0; w < d.groups; w++) {
        const ll size = (ll)d.border(w + 1) - d.border(w);
        if (size < total / d.groups || size > total / d.groups + 1) return printf("workgroup %d has %lld\n", w, size), 1;
        if (d.border_at(d.border(w)) != w || d.border_at(d.border(w + 1) - 1) != w) return printf("border %d\n", w), 1;
    }
    // where the borders lie: (column, unit, tile)
    struct At { size_t col; int unit, tile; };
    std::vector<At> at;
    size_t c = 0;
    ll start = 0;
    for (int w = 0; w <= d.groups; w++) {
        const ll x = d.border(w);
        while (c < n.size() && (n[c] == 0 || x >= start + (ll)(n[c] + BEGIN) * units)) start += n[c] ? (ll)(n[c] + BEGIN) * units : 0, c++;
        if (c == n.size()) { at.push_back({c, 0, 0}); continue; }
        const DealPlace p = deal_place((int)(x - start), n[c], BEGIN, SHORT);
        if (p.unit < 0 || p.unit > units || p.tile < 0 || (p.tile && (p.tile < SHORT || n[c] - p.tile < SHORT || p.unit == units)))
            return printf("place %d %d\n", p.unit, p.tile), 1;
        at.push_back(p.unit == units ? At{c + 1, 0, 0} : At{c, p.unit, p.tile});
        while (at.back().col < n.size() && at.back().tile == 0 && n[at.back().col] == 0) at.back().col++;
    }
    auto before = [](const At &a, const At &b) { return a.col != b.col ? a.col < b.col : a.unit != b.unit ? a.unit < b.unit : a.tile < b.tile; };
    // who has tiles of a unit: for those that a border cuts, in order
    std::map<std::pair<size_t, int>, std::vector<int>> cuts;
    for (int w = 0; w < d.groups; w++) {
        if (before(at[w + 1], at[w])) return printf("borders %d and %d\n", w, w + 1), 1;
        if (w && at[w].tile) cuts[{at[w].col, at[w].unit}].push_back(w);
    }
    std::vector<int> sides(2 * d.groups, 0);
    std::map<int, int> counted;
    size_t col = 0;
    start = 0;
    for (auto &u : cuts) {
        while (col < u.first.first) start += n[col] ? (ll)(n[col] + BEGIN) * units : 0, col++;
        const DealShared s = deal_shared(d, (int)(start + (ll)u.first.second * (n[col] + BEGIN)), n[col], BEGIN, SHORT);
        // the borders inside are those of workgroups first + 1 .. last, one after the other
        const std::vector<int> &w = u.second;
        if (s.last - s.first != (int)w.size()) return printf("%d cuts, workgroups %d to %d\n", (int)w.size(), s.first, s.last), 1;
        for (size_t i = 0; i < w.size(); i++)
            if (w[i] != s.first + 1 + (int)i || (i && at[w[i]].tile <= at[w[i - 1]].tile)) return puts("cuts out of order"), 1;
        // a slot for each workgroup and end: the first one leaves the unit that it ends with, the others the one they begin with
        for (int j = s.first; j <= s.last; j++)
            if (sides[2 * j + (j == s.first)]++) return printf("two units in a slot of workgroup %d\n", j), 1;
        if (counted[s.first]++) return printf("two units are counted at %d\n", s.first), 1;
    }
    return 0;
}

int main() {
    std::mt19937 rng(1);
    auto to = [&](int a, int b) { return std::uniform_int_distribution<int>(a, b)(rng); };
    auto spread = [&](double hi) { return (int)floor(exp(std::uniform_real_distribution<double>(0, log(hi + 1))(rng))); };
    long done = 0;
    for (int i = 0; i < 20000; i++, done++) {
        std::vector<int> n(spread(300));
        const double longest = 1 + spread(5000);
        for (int &t : n) t = to(0, 9) ? spread(longest) : 0;
        const int units = std::vector<int>{1, 2, 3, 5, 8, 12, 130}[to(0, 6)], parts = to(1, 4), most = parts == 1 ? 512 : 512 / (8 * parts) * 8;
        const int heads = to(1, 16), top = n.empty() ? 0 : *std::max_element(n.begin(), n.end());
        if (check(n, units, most, heads >= 8 ? 16 : 8, to(0, 1) ? std::max(1, (int)(sqrtf((float)top * heads) / 3)) : 0, 256 / parts)) return 1;
    }
    // as many places as a launch may have (2^31 - 256) and a few less, in one column and in several, pieces of 1 to 10922
    constexpr ll COUNT = 0x7fffff00;
    for (int units : {1, 2, 3, 7, 12, 31, 32, 33, 64, 130, 4096})
        for (int cols : {1, 2, 5, 300})
            for (int less : {0, 1, 100, 5000, 20000})
                for (int heads : {1, 2, 8, 15, 16})
                    for (int most : {8, 64, 512}) {
                        const ll n = (COUNT - less) / units / cols - BEGIN;
                        if (n < 1 || n > 1 << 26) continue;
                        for (int piece : {0, 1, std::max(1, (int)(sqrtf((float)n * heads) / 3)), 10922})
                            for (int few : {4, 256, 512}) {
                                if (check(std::vector<int>(cols, (int)n), units, most, heads >= 8 ? 16 : 8, piece, few)) return 1;
                                done++;
                            }
                    }
    printf("%ld\n", done);
    return 0;
}
"""


def test_every_tile_has_one_workgroup(tmp_path):
    src, exe = tmp_path / "deal.cpp", tmp_path / "deal"
    src.write_text(PROGRAM)
    flags = ["-std=c++17", "-O2", "-Wall", "-Werror", "-ftrapv"]
    subprocess.run(["g++"] + flags + ["-I", CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0 and int(out.stdout) > 30000, out.stdout + out.stderr
