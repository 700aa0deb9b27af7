// How a batch decode is cut into key ranges, and the size of the scratch that follows from it (host code only, so that the
// sizes can be checked without a GPU).
#pragma once

#include <stddef.h>

#include <algorithm>

#include "pf_plan.hpp"
#include "qwattn.h"
#include "shapes.hpp"

namespace qwa {

constexpr int BT_WAVES = 4;   // waves of a register workgroup; they take the tiles of its key range in turn
constexpr int BT_MAXRT = 2;   // 16-row MFMA tiles of such a workgroup at most
constexpr int BT_STEP = 128;  // its key ranges are multiples of this
constexpr int BT_FEW = 32;    // rows of a KV head up to which the shared positions are left to register workgroups

// Key range [0, n_shared) for all rows together, and [n_shared, len) of every sequence by itself, each cut so that the
// workgroups fill the chip.
//  register workgroups (k_bt_shared, k_bt_own): up to BT_MAXRT row tiles, key ranges of fixed length;
//  tile workgroups (k_bt_tiles): PF_ROWS rows, the shared PF_TILE-key tiles in nt ranges of about equal length.
struct BatchPlan {
    int blocks, nt;              // row blocks and key ranges of the tile workgroups (0: none)
    int ns_shared, len_shared;   // key ranges of register workgroups over the shared positions, and their length
    int rt_shared;
    int groups, rt_own;          // row groups of a sequence, and the row tiles of a group
    int ns_own, len_own;
    int slots() const { return ns_shared + ns_own; }  // fp32 partial states of a row
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
    BatchPlan p = {};
    const int rows = n * nq * GRP, own = nq * GRP;
    p.rt_shared = std::min((rows + 15) / 16, BT_MAXRT);
    p.rt_own = std::min((own + 15) / 16, BT_MAXRT);
    p.groups = (own + 16 * p.rt_own - 1) / (16 * p.rt_own);
    if (rows > BT_FEW && n_shared > 0) {
        const int tiles = (n_shared + PF_TILE - 1) / PF_TILE;
        p.blocks = (rows + PF_ROWS - 1) / PF_ROWS;
        p.nt = std::min(tiles, std::max(1, 256 / (p.blocks * NKV)));
        p.len_shared = BT_STEP;
    } else {
        bt_cut(n_shared, NKV, 128, &p.ns_shared, &p.len_shared);
    }
    bt_cut(max_len - n_shared, n * p.groups * NKV, 128, &p.ns_own, &p.len_own);
    return p;
}

// Partial states in the work buffer, each [slot][row] with row = token * NH + head: of the tile workgroups O / l as 16-bit
// fixed point [256] and (m, l, scale, -), of the register workgroups O as fp32 [256] and (m, l).
struct BatchWork {
    size_t tile_o, tile_ml, o, ml, bytes;  // byte offsets
};
inline BatchWork batch_work(const BatchPlan& p, int n, int nq) {
    const size_t rows = (size_t)n * nq * NH;
    BatchWork w;
    w.tile_o = 0;
    w.tile_ml = w.tile_o + p.nt * rows * HD * 2;
    w.o = w.tile_ml + p.nt * rows * 16;
    w.ml = w.o + p.slots() * rows * HD * 4;
    w.bytes = w.ml + p.slots() * rows * 8;
    if (w.bytes == 0) w.bytes = 16;
    return w;
}

}  // namespace qwa
