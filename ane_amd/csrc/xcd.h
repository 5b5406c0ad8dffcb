// xcd.h — which unit of work a workgroup has.  Plain C++, which the host and the device compile alike.
#pragma once

// MI355X has 8 XCDs, each with a private L2; consecutive workgroup ids are dealt round-robin
// to the XCDs.  This maps the hardware id to a logical id so that consecutive LOGICAL ids
// (neighbouring tiles that share cache lines) run on the same XCD.
constexpr __attribute__((always_inline)) int xcd_remap(int bid, int n) {
    const int q = n >> 3, r = n & 7;
    const int xcd = bid & 7, idx = bid >> 3;
    return xcd * q + (xcd < r ? xcd : r) + idx;
}

// The same for a launch of two kinds of units, n0 of the first and n in all: every XCD has its share of each kind, the first one's first.
struct DealtUnit { bool second; int unit; };
constexpr __attribute__((always_inline)) DealtUnit xcd_deal(int bid, int n0, int n) {
    const bool second = bid >= n0;
    return {second, second ? xcd_remap(bid - n0, n - n0) : xcd_remap(bid, n0)};
}
