// panel_walk.h — which bytes of a tensor the loads of one operand of a product ask for (linear.hip), and how a panel of LDS is laid out
// (mma.h).  Plain C++, which the host and the device compile alike.
//
// A load reads 16 bytes at voffset + soffset from where its buffer begins.  What must not be read has OUTSIDE for its voffset: the range
// check compares that; whether the scalar offset counts too is not the same in every description of it, so no load relies on it.
#pragma once

constexpr unsigned OUTSIDE = 0xfffffff0u;

constexpr int panel_swz(int row) { return (row >> 1 & 1) << 2 | (row >> 2 & 1) | (row >> 3 & 1) << 1; }

// The walk over a sum, 64 steps of it at a time, for B indexes of a tensor [slab][rows][S] of cols / S slabs side by side.
// COLUMNS: the sum goes over the rows: B / 64 panels of 64 rows x 64 columns; else over the columns: one panel of B rows.  Base and S are
// whole chunks of eight values of two bytes.
template <int B, bool COLUMNS, int THREADS>
struct PanelWalk {
    static constexpr int PANELS = COLUMNS ? B / 64 : 1, ROWS = COLUMNS ? 64 : B, WAVES = THREADS / 64, APART = 8 * WAVES;
    static constexpr int PER = ROWS / APART;                // instructions of a wave to a panel, whose rows are APART apart
    static_assert(PER * APART == ROWS && WAVES % 2 == 0, "whole instructions per wave, one swizzle for all of a lane's rows");
    unsigned long long bytes;                               // of the tensor, from where the buffer begins
    unsigned voff[PANELS];                                  // of a lane's first load of each panel
    unsigned soff, row_bytes, slab_bytes;
    int rows_left, S, s0;
    bool even;              // by columns, or every 64 steps lie in one slab and all B rows exist: a lane's offset stays what it is

    // index0: the tile's first index; sum0: where the sum starts; thread: of the workgroup.  Returns where the buffer begins.
    constexpr __attribute__((always_inline)) unsigned long long begin(int rows, int S_, int cols, int index0, int sum0, int thread) {
        const int row = thread >> 3, chunk = (thread & 7) ^ panel_swz(row);
        S = S_;
        row_bytes = (unsigned)S * 2;
        slab_bytes = (unsigned)rows * row_bytes;
        const int first = COLUMNS ? index0 : sum0;          // the first column of all that this reads
        const int b0 = first / S;
        s0 = first - b0 * S;
        rows_left = rows - (COLUMNS ? sum0 : index0);
        const unsigned long long skip = (((unsigned long long)b0 * rows + (COLUMNS ? sum0 : index0)) * S) * 2;
        bytes = (unsigned long long)(cols / S) * rows * S * 2 - skip;
        even = COLUMNS || ((S % 64 == 0 || cols == S) && rows_left >= B);
        soff = COLUMNS ? 0 : s0 * 2;
        for (int i = 0; i < PANELS; i++) {
            if (COLUMNS) {
                const int s = s0 + i * 64 + chunk * 8, db = s / S;
                voff[i] = index0 + i * 64 + chunk * 8 < cols ? (((unsigned)db * rows + row) * S + (s - db * S)) * 2 : OUTSIDE;
            } else voff[i] = (unsigned)row * row_bytes + chunk * 16;
        }
        return skip;
    }
    // Whether the next 64 steps, of which `left` exist, are read at voff as it is; else at voffset(), load by load.
    constexpr __attribute__((always_inline)) bool plain(int left) const { return even && left >= 64; }
    constexpr __attribute__((always_inline)) unsigned voffset(int i, int j, int left, int thread) const {
        const int row = thread >> 3, chunk = (thread & 7) ^ panel_swz(row);
        if (COLUMNS) return row + j * APART < left ? voff[i] : OUTSIDE;
        unsigned v = voff[i];
        for (int s = s0 + chunk * 8; s >= S; s -= S) v += slab_bytes - row_bytes;
        return chunk * 8 < left && row + j * APART < rows_left ? v : OUTSIDE;
    }
    constexpr __attribute__((always_inline)) unsigned soffset(int j) const { return soff + j * APART * row_bytes; }
    // On to the next 64 steps.  Returns how far the buffer's beginning moves.
    constexpr __attribute__((always_inline)) unsigned long long advance() {
        unsigned long long move = 0;
        if (COLUMNS) {
            soff += 64 * row_bytes;
            if (soff >= 1u << 31) {             // rows of up to 2^23 bytes: what 32 bits hold ends after 512 of them
                move = soff;
                soff = 0;
            }
        } else {
            soff += 128;
            s0 += 64;
            if (s0 >= S) {
                const int n = s0 / S;
                s0 -= n * S;
                soff = s0 * 2;
                move = (unsigned long long)n * slab_bytes;
            }
        }
        if (move) bytes = bytes > move ? bytes - move : 0;
        return move;
    }
};
