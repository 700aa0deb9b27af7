// How the attention of a batch of chunks is cut, and the size of the scratch that follows from it (host code only, so that the
// sizes can be checked without a GPU).
#pragma once

#include <stddef.h>

#include <algorithm>

#include "pf_plan.hpp"
#include "qwattn.h"
#include "shapes.hpp"

namespace qwa {

constexpr int CH_PAIRS = 4;                 // pairs of waves of a workgroup: one takes scores, the other multiplies by V
constexpr int CH_ROWS = 32 * CH_PAIRS;      // rows (token, head of the group) of a workgroup
constexpr int CH_SLICES = 256 / NKV;        // workgroups of a KV head: one round of the chip's 256 CUs

// A chunk's rows are cut into blocks of CH_ROWS; a block walks the PF_TILE-key tiles from the first to the last that one of its
// rows sees.  The tiles of all blocks in a row, cut into `slices` equal parts, are the workgroups of a KV head.
// blocks, slices: bounds of what the device finds, which knows the chunks; rows: of a block that are stored.
struct ChunkPlan {
    int blocks, slices, rows;
};

inline ChunkPlan chunk_plan(int n, int rows, int max_len) {
    ChunkPlan p;
    // (a chunk has one partly filled block)
    p.blocks = (int)std::min<long long>((long long)GRP * rows, (long long)GRP * rows / CH_ROWS + n);
    p.slices = (int)std::min<long long>(CH_SLICES, (long long)p.blocks * ((max_len + PF_TILE - 1) / PF_TILE));
    p.rows = std::min(CH_ROWS, GRP * rows);
    return p;
}

// Work buffer: the blocks' descriptions, their number and that of their tiles; the partial states of the blocks that lie in
// several slices, two places a slice (its first block, if it began in an earlier one, and its last one): O as fp32 [256] and
// (m, l, sum for the log) a row.
struct ChunkWork {
    size_t blocks, head, o, ml, bytes;  // byte offsets
};
constexpr size_t CH_BLOCK_BYTES = 32;
inline ChunkWork chunk_work(const ChunkPlan& p) {
    const size_t parts = (size_t)NKV * p.slices * 2 * p.rows;
    ChunkWork w;
    w.o = 0;
    w.ml = w.o + parts * HD * 4;
    w.blocks = w.ml + parts * 16;
    w.head = w.blocks + p.blocks * CH_BLOCK_BYTES;
    w.bytes = w.head + 16;
    return w;
}

}  // namespace qwa
