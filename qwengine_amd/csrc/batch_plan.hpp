// How a batch decode is cut into key ranges, and the size of the scratch that follows from it (host code only, so that the
// sizes can be checked without a GPU).
#pragma once

#include <stddef.h>

#include <algorithm>

#include "qwattn.h"
#include "shapes.hpp"

namespace qwa {

constexpr int BT_WAVES = 4;   // waves of a workgroup; they take the 32-key tiles of its key range in turn
constexpr int BT_MAXRT = 3;   // 16-row MFMA tiles of a workgroup at most
constexpr int BT_STEP = 128;  // key ranges are multiples of this

// Key range [0, n_shared) for all rows together, and [n_shared, len) of every sequence by itself, each cut into ranges of
// fixed length so that the workgroups of a range fill the chip.
struct BatchPlan {
    int rt_shared, groups, ns_shared, len_shared;  // row tiles of a workgroup, row groups, ranges, positions of a range
    int rt_own, ns_own, len_own;
    int slots() const { return ns_shared + ns_own; }  // partial states of a row
};

inline void bt_cut(int positions, int units, int most, int* ns, int* len) {
    if (positions <= 0) {
        *ns = 0;
        *len = BT_STEP;
        return;
    }
    const int steps = (positions + BT_STEP - 1) / BT_STEP;
    const int want = std::min(std::min(most, steps), std::max(1, (512 + units - 1) / units));
    *len = (steps + want - 1) / want * BT_STEP;
    *ns = (positions + *len - 1) / *len;
}

inline BatchPlan batch_plan(int n, int nq, int n_shared, int max_len) {
    BatchPlan p;
    const int rows = n * nq * GRP, tiles = (rows + 15) / 16;
    p.rt_shared = std::min(tiles, BT_MAXRT);
    p.groups = (tiles + p.rt_shared - 1) / p.rt_shared;
    p.rt_own = (nq * GRP + 15) / 16;
    bt_cut(n_shared, p.groups * NKV, 128, &p.ns_shared, &p.len_shared);
    bt_cut(max_len - n_shared, n * NKV, 128, &p.ns_own, &p.len_own);
    return p;
}

// partial states: O [slot][row][256] and (m, l) [slot][row]
inline size_t batch_bytes(int n, int nq, int n_shared, int max_len) {
    const BatchPlan p = batch_plan(n, nq, n_shared, max_len);
    return (size_t)p.slots() * n * nq * NH * (HD + 2) * sizeof(float);
}

}  // namespace qwa
