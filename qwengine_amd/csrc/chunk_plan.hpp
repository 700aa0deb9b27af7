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

// Chunks of at least CH_IMG_BLOCKS blocks read their keys as images: tiles that k_ch_image has brought into the form of LDS once,
// instead of every block by itself.  An image is 35840 bytes, 1.1 times what its tile takes in an F16 cache, 2.1 times Q8_0, 3.9 times
// Q4_0.  There is room for CH_IMG_TILES tiles (of each KV head: 587 MB) or one sequence, whichever is more, as far as the rows
// allow, and chunks that find none left do without.  The bound is one for all types, about where the quantized ones break even;
// of F16, which has nothing to convert, chunks of 12 to 23 blocks lose up to a tenth by it.  One chunk at 8000 positions, whole
// call, us, with / without images:
//   blocks      6            8            10             12             16             24
//   F16     85.2 / 74.2  92.6 / 84.1  100.2 / 91.3   115.1 / 105.5  129.1 / 124.4  170.0 / 169.3
//   Q8_0    85.8 / 80.4  97.1 / 94.4  103.6 / 102.9  116.3 / 116.2  132.0 / 140.0  175.0 / 191.9
//   Q4_0    86.3 / 82.1  96.2 / 95.5  102.0 / 103.7  113.5 / 116.4  130.9 / 138.7  171.2 / 190.1
// Four chunks of 12 blocks 332 / 320, 343 / 358, 339 / 356; of 24 blocks 589 / 629, 629 / 711, 603 / 692.
constexpr int CH_IMG_BLOCKS = 12;
constexpr int CH_IMG_TILES = 4096;
struct ChunkImage {
    uint16_t k[PF_TILE * HD];
    uint16_t scales[PF_TILE * 8];
    int k_dead;                // halves without a place
    int k_pad[63];             // (these 256 bytes are copied as one)
    uint16_t vt[PF_TILE * HD];
    uint8_t odd_keys[8 * HD];  // of V values that are not finite
    int odd[4];                // which quarters of them hold any (1)
    int pad[60];               // (as are these)
};

// A chunk's rows are cut into blocks of CH_ROWS; a block walks the PF_TILE-key tiles from the first to the last that one of its
// rows sees.  What a KV head's workgroups walk are `slices` parts of the blocks' tiles (ch_cuts in attn_chunks.hip).
// blocks, slices, images (chunks that read images), tiles (of images), few: bounds of what the device finds, which knows the
// chunks; rows: of a block that are stored; join: whether any block may lie in several slices.
// Calls of few chunks and blocks, without images, need no plan from a kernel of its own (7 to 10 us): a wave of every workgroup
// makes it in 2, a lane a chunk, a lane a block.
constexpr int CH_OWN = 64;
// Chunks of up to CH_FEW rows (one or two tokens) are no blocks where blocks are cut: their keys' steps of CH_STEP positions in a
// row, cut into as many equal slices, follow a workgroup's tiles, and are walked by its waves a tile each (paged_walk.hpp): 499
// tokens and 23 decoded ones over 8192 Q4_0 positions 230 us, as blocks 317, of which a decoded token filled a twentieth.
constexpr int CH_FEW = 16, CH_FEW_ROWS = CH_FEW / GRP * GRP, CH_STEP = 256;
// What a block takes besides its tiles (Q's way into registers, O's way out), in tiles: the slices are cut from rows of both.
// (Six prompts of up to 1021 F16 tokens, of whose blocks some have 1 tile and some 32, the kernel: 0 / 4 / 6 / 8 / 11: 208 / 166 / 158
// / 148 / 149 us; a chunk of 1024 tokens at 32768 the same with each.)
constexpr int CH_EXTRA = 8;
// Tiles of the parts that a block is cut into at least.  Whole call, us, 2 / 3 / 4 / 5: two chunks of 20 tokens at 512 Q8_0 positions
// 35 / 32 / 31 / 31, at 320 28 with each, 100 tokens of 100 35 / 37 / 30 / 30.
constexpr int CH_LEAST = 4;
struct ChunkPlan {
    int blocks, slices, rows, images, tiles, few;  // few: chunks that may be of so few rows
    bool own, join;
};

inline ChunkPlan chunk_plan(int n, int rows, int max_len) {
    ChunkPlan p;
    const int most = (max_len + PF_TILE - 1) / PF_TILE;
    // (a chunk has one partly filled block)
    p.blocks = (int)std::min<long long>((long long)GRP * rows, (long long)GRP * rows / CH_ROWS + n);
    p.slices = (int)std::min<long long>(CH_SLICES, (long long)p.blocks * most);
    p.join = p.blocks > p.slices || most > CH_LEAST;  // (else every block stays whole)
    p.rows = std::min(CH_ROWS, GRP * rows);
    // (a chunk of CH_IMG_BLOCKS blocks has more than CH_IMG_BLOCKS - 1 full ones)
    p.images = std::min(n, (int)((long long)GRP * rows / (CH_ROWS * (CH_IMG_BLOCKS - 1))));
    p.tiles = (int)std::min<long long>((long long)p.images * most, std::max(most, CH_IMG_TILES));
    p.few = p.join ? std::min(n, rows) : 0;
    p.own = n <= CH_OWN && p.blocks <= CH_OWN && p.images == 0;
    return p;
}

// Work buffer: the blocks' descriptions, the list of chunks with images, the numbers of blocks, their tiles, chunks with images
// and those tiles; the images; the partial states of the blocks that lie in several slices, two places a slice (its first block,
// if it began in an earlier one, and its last one): O as fp32 [256] and (m, l, sum for the log) a row; the same of the chunks of few
// rows, a place for each pair of a slice and a chunk that meet (slice + number of the chunk).
struct ChunkWork {
    size_t images, o, ml, few_o, few_ml, blocks, list, head, bytes;  // byte offsets
};
constexpr size_t CH_BLOCK_BYTES = 48;
inline ChunkWork chunk_work(const ChunkPlan& p) {
    const size_t parts = (size_t)NKV * p.slices * 2 * p.rows;
    ChunkWork w;
    w.images = 0;
    w.o = w.images + (size_t)NKV * p.tiles * sizeof(ChunkImage);
    w.ml = w.o + parts * HD * 4;
    w.few_o = w.ml + parts * 16;
    const size_t few = p.few > 0 ? (size_t)NKV * (p.slices + p.few) * CH_FEW_ROWS : 0;
    w.few_ml = w.few_o + few * HD * 4;
    w.blocks = w.few_ml + few * 16;
    w.list = w.blocks + p.blocks * CH_BLOCK_BYTES;
    w.head = w.list + p.images * 16;
    w.bytes = w.head + 32;
    return w;
}

// The weights: blocks of CW_ROWS rows, tiles of CW_TILE keys.  A block's sums go to its sequence's weights if it is its
// chunk's only one, else to a place [KV head][max_len] of the work buffer, from which they are added up in order.
// parts: places (a chunk of several blocks has at most twice as many as it has full ones).
constexpr int CW_ROWS = 256, CW_TILE = 64;
struct WeightsPlan {
    int blocks, slices, parts;
    bool own;
};
inline WeightsPlan weights_plan(int n, int rows, int max_len) {
    WeightsPlan p;
    const long long full = (long long)GRP * rows / CW_ROWS;
    p.blocks = (int)std::min<long long>((long long)GRP * rows, full + n);
    p.slices = (int)std::min<long long>(CH_SLICES, (long long)p.blocks * ((max_len + CW_TILE - 1) / CW_TILE));
    p.parts = (int)std::min<long long>(p.blocks, 2 * full);
    p.own = n <= CH_OWN && p.blocks <= CH_OWN;
    return p;
}
struct WeightsWork {
    size_t parts, blocks, list, head, bytes;  // byte offsets
};
inline WeightsWork weights_work(const WeightsPlan& p, int max_len) {
    WeightsWork w;
    w.parts = 0;
    w.blocks = w.parts + ((size_t)p.parts * NKV * max_len * 4 + 15) / 16 * 16;
    w.list = w.blocks + p.blocks * CH_BLOCK_BYTES;
    w.head = w.list + (size_t)(p.parts / 2) * 16;
    w.bytes = w.head + 32;
    return w;
}

}  // namespace qwa
