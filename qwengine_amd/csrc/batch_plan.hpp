// How a batch decode is cut into key ranges, and the size of the scratch that follows from it (host code only, so that the
// sizes can be checked without a GPU).
#pragma once

#include <stddef.h>

#include <algorithm>

#include "pf_plan.hpp"
#include "qwattn.h"
#include "shapes.hpp"

namespace qwa {

constexpr int BT_WAVES = 4;               // waves of a register workgroup; they take the tiles of its key range in turn
constexpr int BT_MAXRT = 2;               // 16-row MFMA tiles of such a workgroup at most
constexpr int BT_TWAVES = 8;              // waves of a tile workgroup (four convert V, four K)
constexpr int BT_TROWS = 16 * BT_TWAVES;  // its rows
// Register workgroups that the chip holds, two a CU.  Own positions of 24 sequences, us, 256 / 512 / 1024 workgroups (one a CU,
// two, two rounds): up to 16384 Q4_0 positions 81 / 71 / 83, 8000 Q8_0 59 / 60 / 63, 8000 F16 97 / 99 / 103.
constexpr int BT_FILL = 512;
// Positions of a step; key ranges are whole steps.  A tile for each wave (own positions, steps of 64 / 128 / 256, us: 32
// sequences of up to 700 Q8_0 positions 19.6 / 17.7 / 17.8, 5 x 7 queries of 513 F16 15.7 / 15.2 / 17.6, 5 of 5000 Q4_0 18.2 / 16.1
// / 16.1).
constexpr int BT_STEP = 128;
// Rows of a KV head up to which the shared positions are left to register workgroups: one pass of them.  Whole call, us,
// register / tile workgroups, 32768 shared positions: 18 rows Q4_0 40.5 / 47.5, Q8_0 41.7 / 47.7, F16 45.0 / 43.9; 30 rows 43.2 /
// 47.9, 44.7 / 48.0, 49.1 / 45.4; 36 rows 47.9 / 48.0, 50.9 / 48.5, 50.5 / 45.6; 60 rows 51.2 / 49.2, 53.5 / 50.9, 54.4 / 47.8.
// 4096: 30 rows 26.3 / 28.6, 27.6 / 28.7, 25.2 / 26.9; 60 rows 31.0 / 31.2, 31.0 / 29.9, 28.1 / 28.6.
constexpr int BT_FEW = 32;

// The shared positions [0, n_shared) are worked on for all rows together, the positions of its own [n_shared, len) for every
// sequence by itself.
//  tile workgroups (k_bt_tiles): BT_TROWS rows, the shared PF_TILE-key tiles in nt ranges of about equal length;
//  register workgroups over the shared positions (k_bt_shared): up to BT_MAXRT row tiles, key ranges of fixed length;
//  register workgroups over the own positions (k_bt_own): the steps of BT_STEP positions of all sequences in a row, cut
//  into wgs slices of equal length (the kernel knows the sequences' lengths, the plan only their bound), each worked on as
//  one segment per sequence that it meets.
struct BatchPlan {
    int blocks, nt;                // row blocks and key ranges of the tile workgroups (0: none)
    int groups_shared, rt_shared;  // passes of register workgroups over the batch's rows (1 where they run), their row tiles
    int ns_shared, len_shared;     // key ranges of register workgroups over the shared positions, and their length
    int groups, rt_own;            // row groups of a sequence, and the row tiles of a group
    int wgs;                       // slices of the own steps (0: no own positions)
};

inline BatchPlan batch_plan(int n, int nq, int n_shared, int max_len) {
    BatchPlan p = {};
    const int rows = n * nq * GRP, own = nq * GRP;
    p.rt_shared = rows <= 16 ? 1 : BT_MAXRT;
    p.groups_shared = (rows + 16 * p.rt_shared - 1) / (16 * p.rt_shared);
    p.rt_own = std::min((own + 15) / 16, BT_MAXRT);
    p.groups = (own + 16 * p.rt_own - 1) / (16 * p.rt_own);
    if (rows > BT_FEW && n_shared > 0) {
        const int tiles = (n_shared + PF_TILE - 1) / PF_TILE;
        p.blocks = (rows + BT_TROWS - 1) / BT_TROWS;
        p.nt = std::min(tiles, std::max(1, 256 / (p.blocks * NKV)));
    } else if (n_shared > 0) {
        static_assert(BT_FEW <= 16 * BT_MAXRT, "one pass");
        const int steps = (n_shared + BT_STEP - 1) / BT_STEP, most = std::min(steps, BT_FILL / NKV);
        p.len_shared = (steps + most - 1) / most * BT_STEP;
        p.ns_shared = (n_shared + p.len_shared - 1) / p.len_shared;
    }
    if (max_len > n_shared) {
        const long long steps = (long long)n * ((max_len - (n_shared & ~15) + BT_STEP - 1) / BT_STEP);
        p.wgs = (int)std::min<long long>(steps, std::max(1, BT_FILL / (NKV * p.groups)));
    }
    return p;
}

// Partial states in the work buffer: of the tile workgroups O / l as 16-bit fixed point [256] and (m, l, scale, -), of the
// register workgroups O as fp32 [256] and (m, l).  Those over the shared positions are [range][row] with row = token * NH +
// head.  Segment (slice w, batch row b) of the own positions has number w + b (both only grow along the steps, one of them
// with each segment): [KV head][segment][query * GRP + head of the group].  begin: the step at which each batch row begins,
// and the total.
struct BatchWork {
    size_t tile_o, tile_ml, o, ml, own_o, own_ml, begin, bytes;  // byte offsets
};
inline BatchWork batch_work(const BatchPlan& p, int n, int nq) {
    const size_t rows = (size_t)n * nq * NH, own = p.wgs ? (size_t)NKV * (p.wgs + n) * nq * GRP : 0;
    BatchWork w;
    w.tile_o = 0;
    w.tile_ml = w.tile_o + p.nt * rows * HD * 2;
    w.o = w.tile_ml + p.nt * rows * 16;
    w.ml = w.o + p.ns_shared * rows * HD * 4;
    w.own_o = w.ml + p.ns_shared * rows * 8;
    w.own_ml = w.own_o + own * HD * 4;
    w.begin = w.own_ml + own * 8;
    w.bytes = w.begin + 4 * ((size_t)n + 1);
    return w;
}

}  // namespace qwa
