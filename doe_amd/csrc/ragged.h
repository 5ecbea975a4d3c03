// ragged.h -- rows of many sequences behind each other (row_starts), the last of each at
// its sequence's last position.
#pragma once

#include "common.h"

namespace doe {

// Positions of sequence b that its row of the page table can hold and has in use.
__device__ __forceinline__ int held_positions(const int32_t *lens, int64_t room, int b) {
    const int n = lens[b];
    return n < 0 ? 0 : (n > room ? (int)room : n);
}
// The sequence and position of row `row` of a call (row_starts null: row b of sequence
// b); false where it is of none.  A position below 0 has no place.
__device__ __forceinline__ bool row_position(const int32_t *lens, int64_t room, int batch, const int32_t *row_starts, int64_t row,
                                             int &b, int &pos) {
    int lo = 0;
    int64_t behind = 0;  // rows of the sequence from this one on
    if (row_starts) {
        int hi = batch;  // the last b with row_starts[b] <= row
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (row_starts[mid] <= row) lo = mid;
            else hi = mid;
        }
        behind = row_starts[lo + 1] - row;
        if (row < row_starts[lo] || behind <= 0) return false;
    } else {
        lo = (int)row;
        behind = 1;
    }
    b = lo;
    pos = (int)(held_positions(lens, room, lo) - behind);
    return true;
}

}  // namespace doe
