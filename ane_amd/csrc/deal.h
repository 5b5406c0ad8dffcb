// deal.h — how attention over a paged cache deals its tiles out to workgroups.  Plain C++, which the host and the device compile alike.
//
// A column's units are its KV heads.  The units of all columns, one after the other, form a line on which a unit of n tiles takes n + begin
// places, the first `begin` for what it takes to begin one.  Workgroup w of `groups` has the places from border(w) to border(w + 1); a border
// that would cut off fewer than `least` tiles of a unit is moved to the unit's beginning or end.
//
// All of it is counted in 32 bits, for lines of up to 2^31 - 1 places; only quotients that are rounded up need the sign's bit as well.
#pragma once

#define DEAL_FN constexpr __attribute__((always_inline))

DEAL_FN int deal_ceil(int a, int b) { return (int)(((unsigned)a + (unsigned)b - 1u) / (unsigned)b); }

struct Deal {
    int groups, share, more;        // the first `more` workgroups have share + 1 places, the others share
    DEAL_FN int border(int w) const { return w * share + (w < more ? w : more); }
    // the last border that is not behind x
    DEAL_FN int border_at(int x) const {
        const int longer = more * (share + 1);
        return x < longer ? x / (share + 1) : more + (x - longer) / share;
    }
};

// Workgroups for a line of `total` places: `most` there are, each should have `grain` places at least.
DEAL_FN int deal_groups(int total, int most, int grain) {
    const int groups = deal_ceil(total, grain);
    return groups < most ? groups : most;
}
// No more of them than there are pieces of `piece` places, a multiple of the units, if that is at most `few`.
DEAL_FN int deal_fewer(int groups, int total, int piece, int units, int few) {
    const int pieces = deal_ceil(deal_ceil(total, piece), units) * units;
    return pieces <= few && pieces < groups ? pieces : groups;
}
DEAL_FN Deal deal_out(int total, int groups) {
    const int share = total / groups;
    return {groups, share, total - share * groups};
}

struct DealPlace { int unit, tile; };
// Where a border lies that is `places` behind the beginning of a column whose units have n tiles each.
DEAL_FN DealPlace deal_place(int places, int n, int begin, int least) {
    const int unit = places / (n + begin), tile = places - unit * (n + begin) - begin;
    if (tile >= least && n - tile >= least) return {unit, tile};
    return {unit + (tile >= n - tile), 0};
}

// The workgroups that share a unit, whose places begin at `start`: those before the first and behind the last border that cuts it.
struct DealShared { int first, last; };
DEAL_FN DealShared deal_shared(const Deal &d, int start, int n, int begin, int least) {
    return {d.border_at(start + begin + least - 1), d.border_at(start + begin + n - least)};
}
