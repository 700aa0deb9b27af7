// Attention of a batch of chunks of new tokens over a paged cache (gfx950).
//
// Batch row b has the tokens off[b] .. off[b + 1] - 1, the last c = off[b + 1] - off[b] positions of its sequence; token t of it
// sees positions [0, len - c + t].  For row r = (token, head):  out = sum_j p_j V_j / sum_j p_j * sigmoid(gate),
// p_j = exp(s_j), s_j = q_r . K_j / 16, and log sum_j p_j for who asks for it.
//  * A block is CH_ROWS consecutive rows (6 * token + head of the group) of a chunk; its keys are walked in 32-key tiles.  The
//    tiles of all blocks are cut into slices of about the same time, a workgroup each: a long sequence's tokens and a prompt of a
//    thousand load the chip alike.  A block that lies in several slices leaves partial states, which k_ch_join joins in the
//    slices' order; the others are finished where they are.
//  * A workgroup has two waves a SIMD, with a role each.  The score waves keep Q (32 rows: hi and lo part, 128 registers), bring K
//    into LDS and leave tile i's exponents there: S^T = K Q^T against the rows' references.  The value waves keep O (32 rows, 128
//    registers), bring V into LDS, take the exponentials of tile i - 1 and add V^T P^T.  So each fragment of K and V that is read
//    from LDS meets 32 rows, which one wave with both Q and O has no registers for, and one wave's arithmetic runs beside the
//    other's MFMAs.
//  * Chunks of one or two tokens leave most of a block empty.  Where sequences are cut, they are worked on behind the tiles: a wave
//    a tile, its bytes straight into registers (paged_walk.hpp).
//  * Chunks of many blocks would convert each tile once a block: k_ch_image does it for them once, and the waves copy the images
//    into LDS, two tiles ahead.
//  * Scores are exact up to fp32 accumulation (K as its codes, Q / 16 as the sum of two fp16 parts), as the batched decode's are;
//    the arithmetic of a tile, of V that is not finite and of the probabilities' range is paged_tiles.hpp's.
// Roundings below 32 bits: the dequantized V (d * code) and the probabilities are fp16, half a step 2^-11 of the value, because the
// matrix instructions take fp16.  Exact ones would need a second product for the low parts, or, of V, one with P * d for each
// block of 32 dims; as they are, errors against 64 bits are 2.1e-4 of the norm over F16, which is the output's own rounding, and
// 2.6e-4 to 3.1e-4 over the quantized types.  The sum of a row's probabilities is that of the rounded ones, which P V applies, but
// the log of the sum is taken of the unrounded.  The output is fp16.
#include <algorithm>
#include <type_traits>

#include "chunk_plan.hpp"
#include "launch.hpp"
#include "paged_walk.hpp"

namespace qwa {

// a block: its chunk's first row and number of tokens, the sequence's length and number (< 0: unknown, len 0), the block's number
// in the chunk, its first tile in the row of all tiles, its tiles, the positions that its last row sees, the chunk's first image,
// or the block's place for its sums (-1: none)
struct alignas(16) ChunkBlock {
    int row0, count, len, seq;
    int blk, begin, tiles, end;
    int place, pad[3];
};
static_assert(sizeof(ChunkBlock) == CH_BLOCK_BYTES, "work buffer");

// what the plan is made from
struct ChunkSource {
    qwa_kv_pages p;
    const int* seqs;
    const int* off;
    int n, rows, max_len;
    int few;  // chunks of up to so many rows are listed by themselves
};

struct ChunkArgs {
    ChunkSource src;
    bool own;                // every workgroup makes the plan itself
    const float* q;
    const float* gate;
    uint16_t* out16;
    float* lse;              // [rows][24] or none
    ChunkBlock* blocks;
    const int4* list;        // chunks with images: sequence, length, first image, images
    int* head;               // numbers of blocks, their tiles, chunks with images, images, chunks of few rows, their steps, and
                             // the longest block's tiles
    ChunkImage* images;      // [tile][KV head]
    float* part_o;           // [KV head][slice][2][rows][256]
    float4* part_ml;         // [KV head][slice][2][rows]
    float* few_o;            // [KV head][slice + chunk of few rows][CH_FEW_ROWS][256]
    float4* few_ml;
    int slices, prows, few;
};

size_t prefill_batch_work_bytes(int n, int rows, int max_len) { return chunk_work(chunk_plan(n, rows, max_len)).bytes; }

// sum and largest over the workgroup's threads before this one, and over all
template <int T>
__device__ __forceinline__ int ch_scan(int v, int* s_wave, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();  // s_wave may still be read
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        const int y = s_wave[w];
        if (w < wave) before += y;
        all += y;
    }
    *total = all;
    return before + x - v;
}

// The blocks of all chunks, by one workgroup: thread b has chunk b.  A chunk of rows outside [0, rows], or that begins before an
// earlier one's end, has none.  For the weights (other sizes of blocks and tiles) only the last chunk of a sequence counts, and
// chunks of several blocks get places for their sums (list: sequence, length, tokens, first place) instead of images (sequence,
// length, first image, images).  The chunks of few rows follow the blocks: their `begin` and `tiles` count steps.
template <bool WEIGHTS, int CH_PT>
__global__ void __launch_bounds__(CH_PT) k_ch_plan(ChunkSource src, int most, int most_list, int room,
                                                   ChunkBlock* __restrict__ blocks, int4* __restrict__ list,
                                                   int* __restrict__ head) {
    constexpr int ROWS = WEIGHTS ? CW_ROWS : CH_ROWS, TILE = WEIGHTS ? CW_TILE : PF_TILE;
    const qwa_kv_pages& p = src.p;
    const int* __restrict__ seqs = src.seqs;
    const int* __restrict__ off = src.off;
    const int n = src.n, rows = src.rows, max_len = src.max_len;
    __shared__ int s_wave[CH_PT / 64];
    __shared__ int s_end[CH_PT], s_first[CH_PT], s_count[CH_PT], s_len[CH_PT], s_seq[CH_PT], s_blk[CH_PT], s_place[CH_PT];
    const int t = threadIdx.x, lane = t & 63;
    int first = 0, end = 0;
    if (t < n) {
        first = off[t];
        end = off[t + 1];
        if (first < 0 || end > rows || end < first) end = first = 0;
    }
    // the furthest end of the chunks before this one
    int far = end > first ? end : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(far, o, 64);
        if (lane >= o) far = max(far, y);
    }
    s_end[t] = far;
    __syncthreads();
    int before = lane > 0 ? s_end[t - 1] : 0;
    for (int w = 0; w < t >> 6; w++) before = max(before, s_end[64 * w + 63]);
    int count = end > first && before <= first ? end - first : 0;
    const int seq = t < n ? (seqs ? seqs[t] : t) : -1;
    const bool known = seq >= 0 && seq < p.n_seq;
    s_first[t] = first;
    s_len[t] = known && count > 0 ? min(max(p.len[seq], 0), max_len) : 0;
    s_seq[t] = known ? seq : -1;
    s_count[t] = count;
    if (WEIGHTS) {
        __syncthreads();
        if (!known) count = 0;
        if (seqs && count > 0)
            for (int j = t + 1; j < n; j++)
                if (s_seq[j] == seq && s_count[j] > 0) count = 0;
        __syncthreads();
        s_count[t] = count;
    }
    const bool few = !WEIGHTS && count > 0 && GRP * count <= src.few;
    const int mine = few ? 0 : (GRP * count + ROWS - 1) / ROWS;
    int nb, all, listed, used;
    s_blk[t] = ch_scan<CH_PT>(mine, s_wave, &nb);
    nb = min(nb, most);  // (never more: the chunks' rows are disjoint)
    // images, or places, as long as there is room for them (of places there always is)
    const int want = WEIGHTS ? (mine > 1 ? mine : 0) : mine >= CH_IMG_BLOCKS ? (s_len[t] + PF_TILE - 1) / PF_TILE : 0;
    const int place = ch_scan<CH_PT>(min(want, room + 1), s_wave, &all);
    const bool has = want > 0 && place + want <= room;
    const int entry = ch_scan<CH_PT>(has, s_wave, &listed);
    ch_scan<CH_PT>(has ? want : 0, s_wave, &used);
    s_place[t] = has && entry < most_list ? place : -1;
    if (s_place[t] >= 0)
        list[entry] = WEIGHTS ? make_int4(s_seq[t], s_len[t], count, place) : make_int4(s_seq[t], s_len[t], place, want);
    __syncthreads();
    int tiles = 0, longest = 0;
    for (int j0 = 0; j0 < nb; j0 += CH_PT) {
        const int j = j0 + t;
        ChunkBlock x = {};
        if (j < nb) {
            int lo = 0, hi = n;  // the last chunk whose first block is at most j: an empty one shares that with the next
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_blk[mid] <= j) lo = mid;
                else hi = mid;
            }
            x.row0 = s_first[lo];
            x.count = s_count[lo];
            x.len = s_len[lo];
            x.seq = s_seq[lo];
            x.blk = j - s_blk[lo];
            const int last = min((x.blk + 1) * ROWS, GRP * x.count) - 1;
            x.end = max(0, x.len - x.count + last / GRP + 1);
            x.tiles = max(1, (x.end + TILE - 1) / TILE);  // (rows that see nothing are written too)
            x.place = s_place[lo] < 0 ? -1 : s_place[lo] + (WEIGHTS ? x.blk : 0);
        }
        x.begin = tiles + ch_scan<CH_PT>(x.tiles, s_wave, &all);
        tiles += all;
        if (j < nb) {
            blocks[j] = x;
            longest = max(longest, x.tiles);
        }
    }
    if (!WEIGHTS) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) longest = max(longest, __shfl_xor(longest, o, 64));
        __syncthreads();
        if (lane == 0) s_wave[t >> 6] = longest;
        __syncthreads();
        for (int w = 0; w < CH_PT / 64; w++) longest = max(longest, s_wave[w]);
    }
    int n_few = 0, steps = 0;
    if (!WEIGHTS && src.few > 0) {
        const int j = ch_scan<CH_PT>(few, s_wave, &n_few);
        ChunkBlock x = {};
        x.row0 = first;
        x.count = count;
        x.len = x.end = s_len[t];
        x.seq = s_seq[t];
        x.tiles = few ? max(1, (x.len + CH_STEP - 1) / CH_STEP) : 0;
        x.place = -1;
        x.begin = ch_scan<CH_PT>(x.tiles, s_wave, &steps);
        if (few && nb + j < most) blocks[nb + j] = x;  // (always)
    }
    if (t == 0) {
        head[0] = nb;
        head[1] = tiles;
        head[2] = min(listed, most_list);
        head[3] = used;
        head[4] = n_few;
        head[5] = steps;
        head[6] = longest;
    }
}

// (a thread a chunk; fewer waves wait less at its barriers: 24 chunks 7.0 us with 128 threads, 9.4 with 1024.  With many blocks it
// goes through more rounds, 25 instead of 4 for 128 chunks of 512 tokens, which is 8 us of a call of 1770; 128 chunks of 8 tokens
// 54.4 / 56.6, of 64 170.9 / 170.6)
constexpr int CH_PLAN_FEW = 128;
template <bool WEIGHTS>
void launch_plan(const ChunkSource& src, int most, int most_list, int room, ChunkBlock* blocks, int4* list, int* head,
                 hipStream_t st) {
    if (src.n <= CH_PLAN_FEW)
        hipLaunchKernelGGL((k_ch_plan<WEIGHTS, CH_PLAN_FEW>), dim3(1), dim3(CH_PLAN_FEW), 0, st, src, most, most_list, room, blocks,
                           list, head);
    else
        hipLaunchKernelGGL((k_ch_plan<WEIGHTS, QWA_PAGES_MAXN>), dim3(1), dim3(QWA_PAGES_MAXN), 0, st, src, most, most_list, room,
                           blocks, list, head);
}

// The same of up to CH_OWN chunks and blocks, by one wave, in LDS; places without a bound.
struct OwnPlan {
    ChunkBlock blocks[CH_OWN];
    int4 list[CH_OWN];
    int head[7];
};
template <bool WEIGHTS>
__device__ __forceinline__ void ch_own_plan(OwnPlan& plan, const ChunkSource& src) {
    static_assert(CH_OWN == 64, "a lane a chunk, a lane a block");
    constexpr int ROWS = WEIGHTS ? CW_ROWS : CH_ROWS, TILE = WEIGHTS ? CW_TILE : PF_TILE;
    if (threadIdx.x < 64) {
        const int t = threadIdx.x;
        auto before = [&](int x) {  // sum over the lanes before
            int y = x;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int z = __shfl_up(y, o, 64);
                if (t >= o) y += z;
            }
            return y - x;
        };
        int first = t < src.n ? src.off[t] : 0, end = t < src.n ? src.off[t + 1] : 0;
        int seq = t < src.n ? (src.seqs ? src.seqs[t] : t) : -1;
        const bool known = seq >= 0 && seq < src.p.n_seq;
        const int all = src.p.len[known ? seq : 0];
        if (first < 0 || end > src.rows || end < first) end = first = 0;
        int far = end > first ? end : 0;  // (an empty chunk has no end)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(far, o, 64);
            if (t >= o) far = max(far, y);
        }
        far = __shfl_up(far, 1, 64);
        int count = end > first && (t == 0 || far <= first) ? end - first : 0;
        if (!known) seq = -1;
        if (WEIGHTS) {
            if (!known) count = 0;
            if (src.seqs) {
                const int had = count;
                for (int j = 1; j < src.n; j++) {
                    const int oc = __builtin_amdgcn_readlane(had, j), os = __builtin_amdgcn_readlane(seq, j);
                    if (j > t && oc > 0 && os == seq) count = 0;
                }
            }
        }
        const int len = known && count > 0 ? min(max(all, 0), src.max_len) : 0;
        const bool few = !WEIGHTS && count > 0 && GRP * count <= src.few;
        const int mine = few ? 0 : (GRP * count + ROWS - 1) / ROWS, blk0 = before(mine);
        const int want = WEIGHTS && mine > 1 ? mine : 0, place = before(want), entry = before(want > 0);
        if (want > 0) plan.list[entry] = make_int4(seq, len, count, place);
        const int nb = min(__builtin_amdgcn_readlane(blk0 + mine, 63), CH_OWN);
        int lo = 0;  // block t's chunk
        for (int j = 0; j < src.n; j++) {
            const int b0 = __builtin_amdgcn_readlane(blk0, j);
            if (t >= b0 && t < b0 + __builtin_amdgcn_readlane(mine, j)) lo = j;
        }
        ChunkBlock x = {};
        x.row0 = __shfl(first, lo, 64);
        x.count = __shfl(count, lo, 64);
        x.len = __shfl(len, lo, 64);
        x.seq = __shfl(seq, lo, 64);
        x.blk = t - __shfl(blk0, lo, 64);
        const int last = min((x.blk + 1) * ROWS, GRP * x.count) - 1;
        x.end = max(0, x.len - x.count + last / GRP + 1);
        x.tiles = t < nb ? max(1, (x.end + TILE - 1) / TILE) : 0;
        const int pl = __shfl(place, lo, 64), many = __shfl(want, lo, 64);
        x.place = many > 0 ? pl + x.blk : -1;
        x.begin = before(x.tiles);
        if (t < nb) plan.blocks[t] = x;
        int longest = x.tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) longest = max(longest, __shfl_xor(longest, o, 64));
        int n_few = 0, steps = 0;
        if (!WEIGHTS && src.few > 0) {
            const int j = before(few);
            ChunkBlock y = {};
            y.row0 = first;
            y.count = count;
            y.len = y.end = len;
            y.seq = seq;
            y.tiles = few ? max(1, (len + CH_STEP - 1) / CH_STEP) : 0;
            y.place = -1;
            y.begin = before(y.tiles);
            if (few && nb + j < CH_OWN) plan.blocks[nb + j] = y;  // (always)
            n_few = j + few;
            steps = y.begin + y.tiles;
        }
        if (t == 63) {
            plan.head[0] = nb;
            plan.head[1] = x.begin + x.tiles;
            plan.head[2] = entry + (want > 0);
            plan.head[3] = 0;
            plan.head[4] = n_few;
            plan.head[5] = steps;
            plan.head[6] = longest;
        }
    }
    __syncthreads();
}

// How the tiles are cut: the same for every workgroup of a call.  Where that keeps the longest slice about as short (few blocks),
// each block by itself, into parts of up to `part` tiles: a workgroup has one part.  Otherwise the row of all tiles, of which a
// block has the places extra * (j + 1) + its tiles' numbers, and `extra` before those, into slices of the same length.
struct ChunkCuts {
    int extra, row, slices, part;  // part: 0 if the row is cut
    __device__ __forceinline__ int cut(int w) const { return (int)((long long)w * row / slices); }
    // the block of slice w, and its parts before that: a lane a block (wave-uniform; -1: none)
    __device__ __forceinline__ int block(const ChunkBlock* blocks, int nb, int w, int* before) const {
        const int lane = threadIdx.x & 63, parts = lane < nb ? (blocks[lane].tiles + part - 1) / part : 0;
        int upto = parts;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(upto, o, 64);
            if (lane >= o) upto += y;
        }
        const unsigned long long has = __ballot(lane < nb && upto - parts <= w && w < upto);
        const int j = has ? __builtin_ctzll(has) : -1;
        *before = __builtin_amdgcn_readlane(upto - parts, j < 0 ? 0 : j);
        return j;
    }
};
__device__ __forceinline__ ChunkCuts ch_cuts(int slices, int nb, int tiles, int longest) {
    ChunkCuts c = {0, tiles, min(slices, tiles), 0};
    if (tiles == 0) return c;
    if (nb <= slices) {
        static_assert(CH_SLICES <= 64, "a lane a block");
        const int spare = slices - nb;  // (sum of the parts <= nb + tiles / part <= slices)
        const int part = spare > 0 ? min(longest, max(CH_LEAST, (tiles + spare - 1) / spare)) : longest;
        if (part <= tiles / slices + CH_EXTRA) c.part = part;
    }
    if (c.part == 0) {
        c.extra = CH_EXTRA;
        c.row = tiles + CH_EXTRA * nb;
        c.slices = slices;
    }
    return c;
}
// steps, or tiles of the weights
__device__ __forceinline__ ChunkCuts ch_cuts(int slices, int tiles) { return ChunkCuts{0, tiles, min(slices, tiles), 0}; }

// the block that holds place s, found by the whole workgroup
__device__ __forceinline__ int ch_find(const ChunkBlock* blocks, int nb, int extra, int s, int* s_found) {
    for (int j = threadIdx.x; j < nb; j += blockDim.x) {
        const int begin = blocks[j].begin + extra * j;
        if (begin <= s && s < begin + extra + blocks[j].tiles) *s_found = j;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*s_found);
}

// a block's description in scalar registers
__device__ __forceinline__ ChunkBlock ch_block(const ChunkBlock& c) {
    auto uni = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    return ChunkBlock{uni(c.row0), uni(c.count), uni(c.len), uni(c.seq), uni(c.blk), uni(c.begin), uni(c.tiles), uni(c.end),
                      uni(c.place)};
}

// The images: a workgroup of 512 threads converts a tile of one KV head, half of them K, half V, from registers to memory.  What it
// writes bounds it: 33792 Q8_0 positions (151 MB of images) 37 us.
constexpr int CH_IMG_WGS = 2048;
template <int KVT>
__global__ void __launch_bounds__(512) k_ch_image(ChunkArgs a, qwa_kv_layer kv, qwa_kv_pages p) {
    constexpr int VB = value_bytes(KVT);
    const int t = threadIdx.x, n = a.head[2], units = a.head[3] * NKV;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int tile = unit / NKV, g = unit % NKV;
        int lo = 0, hi = n;  // the last chunk whose first image is at most this
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (a.list[mid].z <= tile) lo = mid;
            else hi = mid;
        }
        const int4 c = a.list[lo];
        const int k0 = (tile - c.z) * PF_TILE, end = c.y;
        const int* __restrict__ table = p.table + (size_t)max(c.x, 0) * p.ld;
        int at[2];
#pragma unroll
        for (int h = 0; h < 2; h++) at[h] = __builtin_amdgcn_readfirstlane(bt_place(p, table, k0 + 16 * h, end));
        const size_t head = (size_t)g * kv.capacity;
        ChunkImage& img = a.images[(size_t)tile * NKV + g];
        const int dead = (at[0] < 0) | (at[1] < 0) << 1, left = end - k0;
        BtRaw<KVT> raw;
        if (wave < 4) {
            const int rows[2] = {at[0] < 0 ? 16 : min(left, 16), at[1] < 0 ? 16 : min(left - 16, 16)};
            bt_load_v<KVT>(raw, kv.v + head * VB, KVT == QWA_KV_F16 ? nullptr : kv.vs + head * 8, at, rows, t);
            static_assert(offsetof(ChunkImage, odd) - offsetof(ChunkImage, odd_keys) == offsetof(BtOdd, tile), "BtOdd");
            BtOdd& odd = *reinterpret_cast<BtOdd*>(img.odd_keys);
            if ((t & 63) == 0) odd.tile[wave] = 0;  // (the wave's own, before it may be set)
            if (t == 0) img.k_dead = dead;
            bt_store_v<KVT>(raw, reinterpret_cast<_Float16*>(img.vt), odd, t, (uint32_t)dead, 1);
        } else {
            const int h = (wave >> 1) & 1;
            bt_load_k<KVT>(raw, kv.k + head * VB, KVT == QWA_KV_F16 ? nullptr : kv.ks + head * 8, at[h],
                           min(max(left - 16 * h, 0), 16), t);
            bt_store_k<KVT>(raw, reinterpret_cast<_Float16*>(img.k), img.scales, t);
        }
    }
}

constexpr int CH_KD = 2;    // K steps read ahead of their MFMAs
constexpr int CH_VD = 6;    // V fragments in flight

// sigmoid by the reciprocal instruction (1 ulp; the output is rounded to fp16): the division's steps are a third of what the rows'
// ends took
__device__ __forceinline__ float ch_sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + fast_exp2(-PF_LOG2E * x)); }
__device__ __forceinline__ uint2 ch_gated(float4 v, float4 g) {
    return make_uint2((uint32_t)f2h_bits(v.x * ch_sigmoid(g.x)) | ((uint32_t)f2h_bits(v.y * ch_sigmoid(g.y)) << 16),
                      (uint32_t)f2h_bits(v.z * ch_sigmoid(g.z)) | ((uint32_t)f2h_bits(v.w * ch_sigmoid(g.w)) << 16));
}
constexpr int CH_RING = 3;  // tiles in LDS: the one read, and two on their way

template <int KVT>
struct ChunkLds {
    _Float16 k[CH_RING][PF_TILE * HD];
    _Float16 vt[CH_RING][PF_TILE * HD];
    uint16_t scales[CH_RING][PF_TILE * 8];  // of K
    BtOdd odd[2];                           // of V that was not an image
    int odd_flags[CH_RING][64];             // of an image: its odd
    int k_flags[CH_RING][64];               // and k_dead
    float cr[2][CH_PAIRS][2][16];           // what O is multiplied by before a tile's P V
    int moved[2][CH_PAIRS];                 // ... if any of it is not 1
    float m[CH_PAIRS][2][16];               // a finished segment's references
    union {
        f4 s[2][2][2][64];                  // a tile's exponents: [tile & 1][row tile][half of the keys][lane]
        float4 x[16 * HD / 8];              // half of a row tile's O on its way out
    } pair[CH_PAIRS];
    uint2 q[CH_PAIRS][16 * HD / 8];         // half of a row tile's Q, one part, on its way into operands
};

// A segment: the tiles [tb, tb + nt) of a block that a workgroup walks.
struct ChunkSegment {
    ChunkBlock c;
    int tb, nt, nrows, wrow0;  // rows of the chunk; the wave's first
    int base;                  // tiles that the workgroup has walked before: tile i has place (base + i) of the rings in LDS
};

// Q / 16 of a wave's 32 rows as the B operand, hi and lo part: rows are read in runs of 512 bytes, their fp16 pieces go to unit
// (4 s + lg, row ^ (4 s + lg) % 16) of the wave's part of LDS and come back as the lane's fragments s.
template <int KVT>
__device__ __forceinline__ void ch_load_q(h8 (&qb)[2][2][8], const float* __restrict__ q, const ChunkBlock& c, int wrow0,
                                          int nrows, int g, uint2* lds_q, int lane) {
    const int i16 = lane & 15, lg = lane >> 4, l5 = lane & 31, half = l5 & 1, u = l5 >> 1;
    uint8_t* const area = reinterpret_cast<uint8_t*>(lds_q);
    float4 x[2][8];
    auto load = [&](int r) {  // round r = 2 * row tile + half of the dims
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const int row = min(wrow0 + 16 * (r >> 1) + 2 * k + (lane >> 5), nrows - 1);
            x[r & 1][k] = *reinterpret_cast<const float4*>(
                q + ((size_t)(c.row0 + row / GRP) * NH + g * GRP + row % GRP) * HD + 128 * (r & 1) + 4 * l5);
        }
    };
    load(0);
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int rt = r >> 1;
        if (r < 3) load(r + 1);
        __builtin_amdgcn_sched_barrier(0);  // (registers: one round ahead)
#pragma unroll
        for (int part = 0; part < 2; part++) {
            auto piece = [&](float v, float f) { return part ? q_lo(v * f) : q_hi(v * f); };
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int row = 2 * k + (lane >> 5);
                const float f = wrow0 + 16 * rt + row < nrows ? 0.0625f : 0.0f;
                uint32_t w0 = h2_bits(h2{piece(x[r & 1][k].x, f), piece(x[r & 1][k].y, f)});
                uint32_t w1 = h2_bits(h2{piece(x[r & 1][k].z, f), piece(x[r & 1][k].w, f)});
                if constexpr (KVT == QWA_KV_Q4_0) {
                    // the operand's order [0, 4, 1, 5, 2, 6, 3, 7]: the even lane makes the first two words, the odd one the rest
                    const uint32_t mine = half ? w1 : w0;
                    const uint32_t other = __builtin_amdgcn_update_dpp(0, half ? w0 : w1, 0xB1, 0xF, 0xF, true);
                    const uint32_t lo = half ? other : mine, hi = half ? mine : other;
                    w0 = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
                    w1 = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
                }
                *reinterpret_cast<uint2*>(area + 16 * (16 * u + (row ^ u)) + 8 * half) = make_uint2(w0, w1);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the area is the wave's own)
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int s = 0; s < 4; s++)
                qb[rt][part][4 * (r & 1) + s] =
                    *reinterpret_cast<const h8*>(area + 16 * (16 * (4 * s + lg) + (i16 ^ (4 * s + lg))));
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// S^T = K Q^T of a tile: lane (row i16 of row tile rt) gets keys 16 kt + 4 lg + e.  The K fragments of a step are read while the
// step before multiplies; a row tile's products are scaled while the other's are on their way.
template <int KVT>
__device__ __forceinline__ void ch_scores(f4 (&sc)[2][2], const h8 (&qb)[2][2][8], const _Float16* Ks, const _Float16* Sc, int i16,
                                          int lg) {
    constexpr bool SC = KVT != QWA_KV_F16;
    f4 T[2][2];
    h4 ks[CH_KD + 1][2];
    h8 kf[CH_KD + 1][2];
    auto scale = [&](int st, int rt) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++) {
#pragma unroll
            for (int e = 0; e < 4; e++) sc[rt][kt][e] = fmaf((float)ks[st % (CH_KD + 1)][kt][e], T[rt][kt][e], sc[rt][kt][e]);
            // (the sums stay where they are: put off past the last block, they kept all products, and spilled)
            asm volatile("" : "+v"(sc[rt][kt]));
        }
    };
    auto read = [&](int st) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++) kf[st % (CH_KD + 1)][kt] = lds_h8(Ks + 8 * (32 * (4 * st + lg) + 16 * kt + (i16 ^ (2 * st))));
        if constexpr (SC)
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
                ks[st % (CH_KD + 1)][kt] = *reinterpret_cast<const h4*>(Sc + 8 * (16 * kt + 4 * (st >> 1) + lg) + 4 * (st & 1));
    };
    auto multiply = [&](int st, int rt) {
#pragma unroll
        for (int part = 1; part >= 0; part--)
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (SC) T[rt][kt] = mfma16(kf[st % (CH_KD + 1)][kt], qb[rt][part][st], part ? zero : T[rt][kt]);
                else sc[rt][kt] = mfma16(kf[st % (CH_KD + 1)][kt], qb[rt][part][st], sc[rt][kt]);
            }
    };
#pragma unroll
    for (int rt = 0; rt < 2; rt++)
#pragma unroll
        for (int kt = 0; kt < 2; kt++) sc[rt][kt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int st = 0; st < CH_KD; st++) read(st);
#pragma unroll
    for (int st = 0; st < 8; st++) {
        // (two of the eight multiplications by scales behind each MFMA: they run while it does)
        auto mix = [&](bool scales) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                if (scales) __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
            }
        };
        __builtin_amdgcn_sched_barrier(0);
        multiply(st, 0);
        if (SC && st > 0) scale(st - 1, 1);
        mix(SC && st > 0);
        __builtin_amdgcn_sched_barrier(0);
        if (st + CH_KD < 8) read(st + CH_KD);  // (into the places of step st - 1)
        __builtin_amdgcn_sched_barrier(0);
        multiply(st, 1);
        if (SC) scale(st, 0);
        mix(SC);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (SC) scale(7, 1);
}

// The pool positions of a tile's groups of 16 keys, 64 tiles ahead: lane l has those of tile l.
template <int G>
struct ChunkPlaces {
    int ahead[G], tile = 0;
    __device__ __forceinline__ void next(int (&at)[G], const qwa_kv_pages& p, const int* __restrict__ table, int tb, int end,
                                         int lane) {
        if ((tile & 63) == 0)
#pragma unroll
            for (int h = 0; h < G; h++) ahead[h] = bt_place(p, table, 16 * (G * (tb + tile + lane) + h), end);
#pragma unroll
        for (int h = 0; h < G; h++) at[h] = __builtin_amdgcn_readlane(ahead[h], tile & 63);
        tile++;
    }
};

// a wave's part of 16 KB on their way into LDS, without registers
__device__ __forceinline__ void ch_copy(const void* lds, const void* src, int wave, int lane) {
#pragma unroll
    for (int c = 0; c < 16 / CH_PAIRS; c++) {
        const int i = wave + CH_PAIRS * c;
        dma_sv<16>(lds_addr(lds) + 1024 * i, src, (uint32_t)(1024 * i + 16 * lane));
    }
}

// The score waves' segment.  Between barriers i and i + 1: K of tile i + 1 from registers (or tile i + 2 of the images) into LDS,
// scores of tile i.
template <int KVT, bool IMG>
__device__ __forceinline__ void ch_score_walk(ChunkLds<KVT>& lds, const ChunkArgs& a, const qwa_kv_layer& kv,
                                              const qwa_kv_pages& p, const ChunkSegment& sg, int g, int pair, int t) {
    constexpr bool SC = KVT != QWA_KV_F16;
    const int lane = t & 63;
    const int* __restrict__ table = p.table + (size_t)max(sg.c.seq, 0) * p.ld;
    const size_t head = (size_t)g * kv.capacity;
    const uint8_t* const kh = kv.k + head * value_bytes(KVT);
    const uint16_t* const ksh = SC ? kv.ks + head * 8 : nullptr;
    const ChunkImage* const img = a.images + (size_t)(max(sg.c.place, 0) + sg.tb) * NKV + g;
    // positions that this lane's rows see, the fewest that one of the wave's does
    int vis[2], vmin = 0x7fffffff;
#pragma unroll
    for (int rt = 0; rt < 2; rt++) {
        const int r = sg.wrow0 + 16 * rt + (lane & 15);
        vis[rt] = r < sg.nrows ? sg.c.len - sg.c.count + r / GRP + 1 : 0;
        if (r < sg.nrows) vmin = min(vmin, vis[rt]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) vmin = min(vmin, __shfl_xor(vmin, o, 64));
    vmin = __builtin_amdgcn_readfirstlane(vmin);
    float m[2] = {-INFINITY, -INFINITY};  // the rows' references
    uint32_t dead = 0;  // halves without a place, two bits a tile from tile i on
    BtRaw<KVT> rk[2];
    ChunkPlaces<2> places;
    auto load = [&](BtRaw<KVT>& rk, int i, int ahead) {
        int at[2];
        places.next(at, p, table, sg.tb, sg.c.end, lane);
        dead |= (uint32_t)((at[0] < 0) | (at[1] < 0) << 1) << (2 * ahead);
        const int h = pair >> 1, left = sg.c.end - (sg.tb + i) * PF_TILE - 16 * h;
        bt_load_k<KVT>(rk, kh, ksh, h ? at[1] : at[0], min(max(left, 0), 16), t);
    };
    auto slot = [&](int i) { return (sg.base + i) % CH_RING; };
    auto copy = [&](int i) {
        const ChunkImage& x = img[(size_t)i * NKV];
        ch_copy(lds.k[slot(i)], x.k, pair, lane);
        if (SC && pair < 2) dma_sv<4>(lds_addr(lds.scales[slot(i)]) + 256 * pair, x.scales, (uint32_t)(256 * pair + 4 * lane));
        if (pair == 2) dma_sv<4>(lds_addr(lds.k_flags[slot(i)]), &x.k_dead, (uint32_t)(4 * lane));
    };
    auto landed = [&](bool last) {  // all copies (but the last one, if there is another on its way)
        if (last) wait_vmcnt<0>();
        else if ((SC && pair < 2) || pair == 2) wait_vmcnt<16 / CH_PAIRS + 1>();
        else wait_vmcnt<16 / CH_PAIRS>();
    };
    if constexpr (!IMG) {
        load(rk[0], 0, 0);
        if (sg.nt > 1) load(rk[1], 1, 1);
    }
    h8 qb[2][2][8];
    ch_load_q<KVT>(qb, a.q, sg.c, sg.wrow0, sg.nrows, g, lds.q[pair], lane);
    if constexpr (IMG) {
        wait_vmcnt<0>();  // from here on vmcnt counts only the copies
        copy(0);
        if (sg.nt > 1) copy(1);
        landed(sg.nt <= 1);
    } else {
        bt_store_k<KVT>(rk[0], lds.k[slot(0)], lds.scales[slot(0)], t);
        if (sg.nt > 2) load(rk[0], 2, 2);
    }
    __syncthreads();
    auto step = [&](int i, BtRaw<KVT>& rk) __attribute__((always_inline)) {
        if constexpr (IMG) {
            if (i + 2 < sg.nt) copy(i + 2);
        } else {
            if (i + 1 < sg.nt) bt_store_k<KVT>(rk, lds.k[slot(i + 1)], lds.scales[slot(i + 1)], t);
            if (i + 3 < sg.nt) load(rk, i + 3, 3);
        }
        if (sg.wrow0 < sg.nrows) {
            // (an opaque copy of the lane: the LDS addresses, kept across the tiles, spilled)
            int ol = lane;
            asm volatile("" : "+v"(ol));
            f4 sc[2][2];
            ch_scores<KVT>(sc, qb, lds.k[slot(i)], reinterpret_cast<const _Float16*>(lds.scales[slot(i)]), ol & 15, ol >> 4);
            if constexpr (!SC) {
                mfma_settle(sc[0][0], sc[0][1]);
                mfma_settle(sc[1][0], sc[1][1]);
            }
            const int k0 = (sg.tb + i) * PF_TILE, b = i & 1;
            const int gone = IMG ? __builtin_amdgcn_readfirstlane(lds.k_flags[slot(i)][0]) : (int)(dead & 3);
            if (k0 + PF_TILE > vmin || gone != 0) {
#pragma unroll
                for (int rt = 0; rt < 2; rt++)
#pragma unroll
                    for (int kt = 0; kt < 2; kt++)
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            sc[rt][kt][e] = k0 + 16 * kt + 4 * (ol >> 4) + e < vis[rt] && !((gone >> kt) & 1) ? sc[rt][kt][e]
                                                                                                              : -INFINITY;
            }
            float cr[2];
#pragma unroll
            for (int rt = 0; rt < 2; rt++) {
                float mx = max3f(max3f(-INFINITY, sc[rt][0][0], sc[rt][0][1]), sc[rt][0][2], sc[rt][0][3]);
                mx = rows_max(max3f(max3f(mx, sc[rt][1][0], sc[rt][1][1]), sc[rt][1][2], sc[rt][1][3]));
                const float mx2 = mx * PF_LOG2E, mn = mx2 > m[rt] + BT_HEAD ? mx2 - BT_RAISE : m[rt];
                cr[rt] = mn == m[rt] ? 1.0f : fast_exp2(m[rt] - mn);
                const float ref = mn == -INFINITY ? 0.0f : mn;  // a row that saw nothing keeps l = 0, O = 0
                m[rt] = mn;
#pragma unroll
                for (int kt = 0; kt < 2; kt++) {
                    f4 x;
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = fmaf(sc[rt][kt][e], PF_LOG2E, -ref);
                    lds.pair[pair].s[b][rt][kt][ol] = x;
                }
            }
            const bool any = __any(cr[0] != 1.0f || cr[1] != 1.0f);
            if (any)
#pragma unroll
                for (int rt = 0; rt < 2; rt++) lds.cr[b][pair][rt][ol & 15] = cr[rt];
            if (ol == 0) lds.moved[b][pair] = any;
            if (i + 1 == sg.nt)
#pragma unroll
                for (int rt = 0; rt < 2; rt++) lds.m[pair][rt][ol & 15] = m[rt];
        }
        dead >>= 2;
        if constexpr (IMG) landed(i + 2 >= sg.nt);
        __syncthreads();
    };
    if constexpr (IMG) {
        for (int i = 0; i < sg.nt; i++) step(i, rk[0]);
    } else {  // (the bytes of two tiles on their way: those of one were waited for where a workgroup is alone with its rows)
        for (int i = 0; i < sg.nt; i += 2) {
            step(i, rk[1]);
            if (i + 1 < sg.nt) step(i + 1, rk[0]);
        }
    }
}

// The value waves' segment.  Between barriers i and i + 1: V of tile i from registers (or tile i + 1 of the images) into LDS,
// exponentials and P V of tile i - 1; behind the last barrier the last tile's, and the rows' results.
template <int KVT, bool IMG, bool LSE>
__device__ __forceinline__ void ch_value_walk(ChunkLds<KVT>& lds, const ChunkArgs& a, const qwa_kv_layer& kv,
                                              const qwa_kv_pages& p, const ChunkSegment& sg, int g, int pair, size_t part, int t) {
    constexpr bool SC = KVT != QWA_KV_F16;
    const int lane = t & 63, i16 = lane & 15, lg = lane >> 4;
    const int* __restrict__ table = p.table + (size_t)max(sg.c.seq, 0) * p.ld;
    const size_t head = (size_t)g * kv.capacity;
    const uint8_t* const vh = kv.v + head * value_bytes(KVT);
    const uint16_t* const vsh = SC ? kv.vs + head * 8 : nullptr;
    const ChunkImage* const img = a.images + (size_t)(max(sg.c.place, 0) + sg.tb) * NKV + g;
    const bool rows_here = sg.wrow0 < sg.nrows;
    int vis[2];  // positions that this lane's rows see
#pragma unroll
    for (int rt = 0; rt < 2; rt++) {
        const int r = sg.wrow0 + 16 * rt + i16;
        vis[rt] = r < sg.nrows ? sg.c.len - sg.c.count + r / GRP + 1 : 0;
    }
    BtRaw<KVT> rv[2];
    ChunkPlaces<2> places;
    uint32_t dead = 0;  // halves without a place, two bits a tile: tile i - 1, tile i, ...
    auto load = [&](BtRaw<KVT>& rv, int i) {
        int at[2];
        places.next(at, p, table, sg.tb, sg.c.end, lane);
        const int left = sg.c.end - (sg.tb + i) * PF_TILE;
        const int rows[2] = {at[0] < 0 ? 16 : min(left, 16), at[1] < 0 ? 16 : min(left - 16, 16)};
        bt_load_v<KVT>(rv, vh, vsh, at, rows, t);
        return (uint32_t)((at[0] < 0) | (at[1] < 0) << 1);
    };
    auto slot = [&](int i) { return (sg.base + i) % CH_RING; };
    auto copy = [&](int i) {
        const ChunkImage& x = img[(size_t)i * NKV];
        ch_copy(lds.vt[slot(i)], x.vt, pair, lane);
        if (pair == 0) dma_sv<4>(lds_addr(lds.odd_flags[slot(i)]), x.odd, (uint32_t)(4 * lane));
    };
    auto landed = [&](bool last) {
        if (last) wait_vmcnt<0>();
        else if (pair == 0) wait_vmcnt<16 / CH_PAIRS + 1>();
        else wait_vmcnt<16 / CH_PAIRS>();
    };
    f4 o[2][16];
    float l[2], lx[2];
#pragma unroll
    for (int rt = 0; rt < 2; rt++) {
        l[rt] = lx[rt] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < 16; dt++) o[rt][dt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if constexpr (IMG) {
        wait_vmcnt<0>();  // from here on vmcnt counts only the copies
        copy(0);
    } else {
        dead = load(rv[0], 0) << 2;
        if (sg.nt > 1) dead |= load(rv[1], 1) << 4;
    }
    __syncthreads();
    auto step = [&](int i, BtRaw<KVT>& rv) __attribute__((always_inline)) {
        // (opaque copies: LDS addresses kept across the tiles took the registers of O)
        int ol = lane;
        asm volatile("" : "+v"(ol));
        const int oi = ol & 15, og = ol >> 4;
        if constexpr (IMG) {
            if (i + 1 < sg.nt) copy(i + 1);
        } else {
            if (i < sg.nt)
                bt_store_v<KVT>(rv, lds.vt[slot(i)], lds.odd[(sg.base + i) & 1], 64 * pair + ol, (dead >> 2) & 3, sg.base + i);
            if (i + 2 < sg.nt) dead |= load(rv, i + 2) << 6;
        }
        if (i > 0 && rows_here) {
            const int b = (i - 1) & 1, k0 = (sg.tb + i - 1) * PF_TILE;
            f4 sc[2][2];
#pragma unroll
            for (int rt = 0; rt < 2; rt++)
#pragma unroll
                for (int kt = 0; kt < 2; kt++) sc[rt][kt] = lds.pair[pair].s[b][rt][kt][ol];
            const int4 odd =
                *reinterpret_cast<const int4*>(IMG ? lds.odd_flags[slot(i - 1)] : lds.odd[(sg.base + i - 1) & 1].tile);
            const bool moved = __builtin_amdgcn_readfirstlane(lds.moved[b][pair]) != 0;
            float cr[2] = {1.0f, 1.0f};
            if (moved)
#pragma unroll
                for (int rt = 0; rt < 2; rt++) cr[rt] = lds.cr[b][pair][rt][oi];
            // the V fragments' reads begin while the exponentials are taken
            const _Float16* vrow = lds.vt[slot(i - 1)] + 8 * (256 * og + oi);
            h8 vf[CH_VD];
#pragma unroll
            for (int dt = 0; dt < CH_VD - 1; dt++) vf[dt] = lds_h8(vrow + 8 * 16 * dt);
            h8 pb[2];
#pragma unroll
            for (int rt = 0; rt < 2; rt++) {
                float rx = 0.0f, rs = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float x = fast_exp2(sc[rt][e >> 2][e & 3]);
                    pb[rt][e] = (_Float16)x;
                    if (LSE) rx += x;
                }
                // the sum of the rounded probabilities, the weights that P V applies
                const h2 one2 = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
                for (int e = 0; e < 8; e += 2) rs = __builtin_amdgcn_fdot2(h2{pb[rt][e], pb[rt][e + 1]}, one2, rs, false);
                l[rt] = l[rt] * cr[rt] + rs;
                if (LSE) lx[rt] = lx[rt] * cr[rt] + rx;
            }
            if (moved) {
#pragma unroll
                for (int rt = 0; rt < 2; rt++)
#pragma unroll
                    for (int dt = 0; dt < 16; dt++) o[rt][dt] *= cr[rt];
            }
            // O^T += V^T P^T
#pragma unroll
            for (int dt = 0; dt < 16; dt++) {
                if (dt + CH_VD - 1 < 16) vf[(dt + CH_VD - 1) % CH_VD] = lds_h8(vrow + 8 * 16 * (dt + CH_VD - 1));
#pragma unroll
                for (int rt = 0; rt < 2; rt++) o[rt][dt] = mfma16(vf[dt % CH_VD], pb[rt], o[rt][dt]);
            }
            // a dim is NaN in the rows that see a value of it that is not finite
            const int mark = IMG ? 1 : sg.base + i - 1;
            if (__builtin_amdgcn_readfirstlane(odd.x == mark || odd.y == mark || odd.z == mark || odd.w == mark)) {
                const int of[4] = {odd.x, odd.y, odd.z, odd.w};
                const uint8_t* const keys_of = IMG ? img[(size_t)(i - 1) * NKV].odd_keys : lds.odd[(sg.base + i - 1) & 1].keys;
                uint32_t seen[2][2] = {};
#pragma unroll
                for (int rt = 0; rt < 2; rt++)
#pragma unroll
                    for (int k = 0; k < PF_TILE; k++) {
                        const int cb = k / 4 % 4, h = k / 16;
                        if (of[cb] == mark && k0 + k < vis[rt])  // (halves without a place are zeros)
                            seen[rt][cb / 2] |= 1u << (8 * (2 * (cb & 1) + h) + k % 4);
                    }
#pragma unroll
                for (int dt = 0; dt < 16; dt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int dim = 8 * (16 * (dt & 1) + 4 * og + e) + (dt >> 1);
                        const uint2 keys = *reinterpret_cast<const uint2*>(keys_of + 8 * dim);
#pragma unroll
                        for (int rt = 0; rt < 2; rt++)
                            o[rt][dt][e] = ((keys.x & seen[rt][0]) | (keys.y & seen[rt][1])) != 0 ? NAN : o[rt][dt][e];
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (IMG) wait_vmcnt<0>();
            }
        }
        dead >>= 2;
        if (i < sg.nt) {
            // (V of tile i, sent before that of tile i + 1)
            if constexpr (IMG) landed(i + 1 >= sg.nt);
            __syncthreads();
        }
    };
    if constexpr (IMG) {
        for (int i = 0; i <= sg.nt; i++) step(i, rv[0]);
    } else {
        for (int i = 0; i <= sg.nt; i += 2) {
            step(i, rv[0]);
            if (i < sg.nt) step(i + 1, rv[1]);
        }
    }
    if (!rows_here) return;
    // O by way of LDS, half of a row tile's dims at a time, so that rows are written as they lie in memory
    const bool whole = sg.nt == sg.c.tiles;
    float4* const area = lds.pair[pair].x;
    const int u = lane & 31;
    float4 gv[2][8];
    auto place = [&](int r, int k) {  // output row k of round r = 2 * row tile + half of the dims
        const int row = min(sg.wrow0 + 16 * (r >> 1) + 2 * k + (lane >> 5), sg.nrows - 1);
        return ((size_t)(sg.c.row0 + row / GRP) * NH + g * GRP + row % GRP) * HD + 128 * (r & 1) + 4 * u;
    };
    auto gates = [&](int r) {
#pragma unroll
        for (int k = 0; k < 8; k++) gv[r & 1][k] = *reinterpret_cast<const float4*>(a.gate + place(r, k));
    };
    if (whole) gates(0);
#pragma unroll
    for (int rt = 0; rt < 2; rt++) {
        const float lt = rows_sum(l[rt]), lxt = LSE ? rows_sum(lx[rt]) : 0.0f, m = lds.m[pair][rt][i16];
        const float il = whole ? (lt == 0.0f ? 0.0f : 1.0f / lt) : 1.0f;
        const int r0 = sg.wrow0 + 16 * rt + i16;
        if (lg == 0 && r0 < sg.nrows) {
            if (!whole) a.part_ml[part + r0 - CH_ROWS * sg.c.blk] = make_float4(m, lt, lxt, 0.0f);
            else if (LSE)
                a.lse[(size_t)(sg.c.row0 + r0 / GRP) * NH + g * GRP + r0 % GRP] =
                    lxt == 0.0f ? -INFINITY : (m + __log2f(lxt)) * 0.6931471805599453f;
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 2 * rt + e;
            if (whole && r < 3) gates(r + 1);
            // o[rt][2 k + e][j] is dim 8 x + k, x = 16 e + 4 lg + j: unit 2 (4 lg + j) + k / 4 of the half
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    area[32 * i16 + ((2 * (4 * lg + j) + h) ^ (i16 & 7))] =
                        make_float4(o[rt][8 * h + e][j] * il, o[rt][8 * h + 2 + e][j] * il, o[rt][8 * h + 4 + e][j] * il,
                                    o[rt][8 * h + 6 + e][j] * il);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the area is the wave's own)
            __builtin_amdgcn_wave_barrier();
            float4 v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int xr = 2 * k + (lane >> 5);
                v[k] = area[32 * xr + (u ^ (xr & 7))];
            }
            const int row0 = sg.wrow0 + 16 * rt + (lane >> 5);
            if (whole) {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint2 w = ch_gated(v[k], gv[r & 1][k]);
                    if (row0 + 2 * k < sg.nrows) *reinterpret_cast<uint2*>(a.out16 + place(r, k)) = w;
                }
            } else {
                float* const dst = a.part_o + (part + row0 - CH_ROWS * sg.c.blk) * HD + 128 * e + 4 * u;
#pragma unroll
                for (int k = 0; k < 8; k++)
                    if (row0 + 2 * k < sg.nrows) *reinterpret_cast<float4*>(dst + 2 * k * HD) = v[k];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

// a chunk of few rows, for bt_walk: its state goes to place `rec` on
struct FewSegment : BtRange {
    int first, count, len;
    size_t rec;
};
template <bool LSE>
struct FewRows {
    static constexpr int WAVES = 2 * CH_PAIRS;
    static constexpr bool SUM = LSE;
    using SEGMENT = FewSegment;
    const ChunkArgs& a;
    __device__ __forceinline__ int seen(const SEGMENT& s, int tok) const { return s.len - s.count + tok + 1; }
    __device__ __forceinline__ const float* q(const SEGMENT& s, int tok) const { return a.q + (size_t)(s.first + tok) * NH * HD; }
    __device__ __forceinline__ size_t place(const SEGMENT& s, int r) const { return s.rec + r; }
    __device__ __forceinline__ void sums(const SEGMENT&, size_t place, float m, float l, float x) const {
        a.few_ml[place] = make_float4(m, l, x, 0.0f);
    }
    __device__ __forceinline__ float* o(const SEGMENT&, size_t place) const { return a.few_o + place * HD; }
};

template <int KVT, bool LSE>
struct ChunkShared {
    union {
        ChunkLds<KVT> tiles;
        BtLds<KVT, 1, FewRows<LSE>::WAVES, LSE> walk;
    };
    int found;
    OwnPlan plan;
};

// 1024 tokens over 32768 Q8_0 positions 1200 to 1260 us, 0.70 PFLOP/s, 1.05 with the second part of Q (large products of the
// library 1.21); 1.65 us a tile.  Of a SIMD's cycles 49% are MFMAs and 39% issue VALU instructions, LDS is busy for 31% and without
// conflicts; the value waves are the longer chain: copies' issue and exponents 1200 cycles, exponentials 900, P V 750 and 500
// between them, of 3400 to 3800 a tile.  Without the images' copies a tile took 1.4 us, the copies alone 1.2 (7.3 TB/s of images,
// which the L2s miss: a head's workgroups are spread over the positions).  A segment costs about 8 tiles besides: Q's way in and,
// longer, O's way out with the gates.  Six prompts of up to 1021 F16 tokens, 136 to 152 us, move 0.36 GB of Q, gates, outputs and
// states meanwhile.  Measured and not kept, none with a difference: Q three loads ahead, the next block's description in LDS, rows'
// addresses without divisions, the exponents' reads before the copies, the score waves at a higher priority; slower: raw tiles for
// long chunks (1450), the value waves at a higher priority (1365).
template <int KVT, bool LSE>
__global__ void __launch_bounds__(128 * CH_PAIRS) __attribute__((amdgpu_waves_per_eu(2, 2)))
k_ch_tiles(ChunkArgs a, qwa_kv_layer kv, qwa_kv_pages p) {
    __shared__ __attribute__((aligned(16))) ChunkShared<KVT, LSE> shared;
    ChunkLds<KVT>& lds = shared.tiles;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int pair = wave & (CH_PAIRS - 1);
    // workgroups 8 apart run on one XCD: each has consecutive slices of one head, whose tiles its L2 then holds
    int unit = blockIdx.x;
    if (gridDim.x % 8 == 0) unit = (int)(gridDim.x / 8) * (blockIdx.x & 7) + (blockIdx.x >> 3);
    const ChunkBlock* blocks = a.blocks;
    const int* head = a.head;
    if (a.own) {
        ch_own_plan<false>(shared.plan, a.src);
        blocks = shared.plan.blocks;
        head = shared.plan.head;
        if (blockIdx.x == 0) {  // for the join
            const int words = (head[0] + head[4]) * (int)(sizeof(ChunkBlock) / 4);
            for (int i = threadIdx.x; i < words; i += blockDim.x)
                reinterpret_cast<int*>(a.blocks)[i] = reinterpret_cast<const int*>(blocks)[i];
            if (threadIdx.x < 7) a.head[threadIdx.x] = head[threadIdx.x];
        }
    }
    const int nb = __builtin_amdgcn_readfirstlane(head[0]), tiles = __builtin_amdgcn_readfirstlane(head[1]);
    const int g = unit / a.slices, w = unit % a.slices;
    int s = 0, s_end = 0, j = 0;
    if (threadIdx.x < 8) lds.odd[threadIdx.x >> 2].tile[threadIdx.x & 3] = -1;
    const ChunkCuts tile_cuts = ch_cuts(a.slices, nb, tiles, __builtin_amdgcn_readfirstlane(head[6]));
    if (tile_cuts.part > 0) {
        int before;
        j = tile_cuts.block(blocks, nb, w, &before);
        if (j >= 0) {
            const ChunkBlock c = ch_block(blocks[j]);
            const int parts = (c.tiles + tile_cuts.part - 1) / tile_cuts.part;
            s = c.begin + (w - before) * c.tiles / parts;
            s_end = c.begin + (w - before + 1) * c.tiles / parts;
        }
        __syncthreads();
    } else if (w < tile_cuts.slices) {
        s = tile_cuts.cut(w);
        s_end = tile_cuts.cut(w + 1);
        j = ch_find(blocks, nb, tile_cuts.extra, s, &shared.found);
    }
    const int s_begin = s;
    int walked = 0;
    // The segments; the roles meet at a segment's barriers, one and one a tile.  Behind the last one the score waves go on to the
    // next segment's Q and K while the value waves finish: what these still read there (V and flags of the last tile, its
    // scores, which the pair's own O follows) is written by nobody before the next barrier.
    while (s < s_end) {
        // (an opaque copy of the thread: addresses kept across the segments took registers of the loop over tiles)
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        ChunkSegment sg;
        sg.c = ch_block(blocks[j]);
        const int first = sg.c.begin + tile_cuts.extra * (j + 1), stop = min(s_end, first + sg.c.tiles), from = s;
        s = stop;
        j++;
        sg.base = walked;
        sg.tb = max(from - first, 0);
        sg.nt = stop - first - sg.tb;
        if (sg.nt <= 0) continue;  // (the slice ends before the block's first tile)
        walked += sg.nt;
        sg.nrows = GRP * sg.c.count;
        sg.wrow0 = CH_ROWS * sg.c.blk + 32 * pair;
        const size_t part = (((size_t)g * a.slices + w) * 2 + (from == s_begin ? 0 : 1)) * a.prows;
        if (wave < CH_PAIRS) {
            if (sg.c.place >= 0) ch_score_walk<KVT, true>(lds, a, kv, p, sg, g, pair, t);
            else ch_score_walk<KVT, false>(lds, a, kv, p, sg, g, pair, t);
        } else {
            if (sg.c.place >= 0) ch_value_walk<KVT, true, LSE>(lds, a, kv, p, sg, g, pair, part, t);
            else ch_value_walk<KVT, false, LSE>(lds, a, kv, p, sg, g, pair, part, t);
        }
    }
    const int n_few = a.few > 0 ? __builtin_amdgcn_readfirstlane(head[4]) : 0;
    if (n_few == 0) return;
    // the chunks of few rows
    const int steps = __builtin_amdgcn_readfirstlane(head[5]);
    const ChunkCuts cuts = ch_cuts(a.slices, steps);
    if (w >= cuts.slices) return;
    s = cuts.cut(w);
    s_end = cuts.cut(w + 1);
    __syncthreads();  // (of the tiles' LDS nothing is read any more)
    j = ch_find(blocks + nb, n_few, 0, s, &shared.found);
    auto segment = [&] {
        const ChunkBlock c = ch_block(blocks[nb + j]);
        const int k0 = (s - c.begin) * CH_STEP, stop = min(s_end, c.begin + c.tiles);
        const FewSegment x = {{p.table + (size_t)max(c.seq, 0) * p.ld, 0, GRP * c.count, k0, min((stop - c.begin) * CH_STEP, c.end), 0},
                              c.row0, c.count, c.len, ((size_t)g * (a.slices + a.few) + w + j) * CH_FEW_ROWS};
        s = stop;
        return x;
    };
    bt_walk<KVT, 1>(shared.walk, FewRows<LSE>{a}, kv, p, g, segment(), [&](FewSegment& seg) {
        if (s >= s_end) return false;
        j++;
        seg = segment();
        return true;
    });
}

// A row's output from its states of slices w0 .. w1, in that order: 4 dims a lane.
template <bool LSE, class PLACE>
__device__ __forceinline__ void ch_join_row(const ChunkArgs& a, const float* o, const float4* sums, size_t out, int w0, int w1,
                                            int lane, PLACE place) {
    const float4 gv = *reinterpret_cast<const float4*>(a.gate + out * HD + 4 * lane);
    float M = -INFINITY, L = 0.0f, X = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int w = w0; w <= w1; w += 8) {
        float4 ml[8], x[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const size_t at = place(min(w + u, w1));
            ml[u] = sums[at];
            x[u] = *reinterpret_cast<const float4*>(o + at * HD + 4 * lane);
        }
#pragma unroll
        for (int u = 0; u < 8; u++) {
            if (w + u > w1) break;
            const float Mn = fmaxf(M, ml[u].x);
            const float f0 = M == Mn ? 1.0f : fast_exp2(M - Mn);
            // a state that saw nothing weighs nothing; one of NaN scores (l is NaN) makes the row NaN
            const float f = ml[u].y == 0.0f ? 0.0f : fast_exp2(ml[u].x - Mn);
            M = Mn;
            L = fmaf(L, f0, f * ml[u].y);
            if (LSE) X = fmaf(X, f0, f * ml[u].z);
            acc.x = fmaf(acc.x, f0, f * x[u].x);
            acc.y = fmaf(acc.y, f0, f * x[u].y);
            acc.z = fmaf(acc.z, f0, f * x[u].z);
            acc.w = fmaf(acc.w, f0, f * x[u].w);
        }
    }
    const float il = L == 0.0f ? 0.0f : 1.0f / L;
    *reinterpret_cast<uint2*>(a.out16 + out * HD + 4 * lane) =
        ch_gated(make_float4(acc.x * il, acc.y * il, acc.z * il, acc.w * il), gv);
    if (LSE && lane == 0) a.lse[out] = X == 0.0f ? -INFINITY : (M + __log2f(X)) * 0.6931471805599453f;
}

// Joins the states of the blocks that lie in several slices, in the slices' order: workgroup (cut between two slices, part of the
// rows; KV head) has the block that the cut lies in, if it is the first cut in it; a wave a row.  The workgroups behind those have
// a chunk of few rows each.  The states' bytes bound it: 64 MB 18 to 21 us; two blocks of three parts 7.4.
constexpr int CH_JR = 16;  // rows of a workgroup
template <bool LSE>
__global__ void __launch_bounds__(256) k_ch_join(ChunkArgs a, int parts) {
    __shared__ int found;
    const ChunkBlock* const blocks = a.blocks;
    const int* const head = a.head;
    const int g = blockIdx.y, cut = blockIdx.x / parts + 1, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (cut >= a.slices) {
        const int j = (int)blockIdx.x - (a.slices - 1) * parts;
        if (j >= head[4]) return;
        const ChunkBlock c = blocks[head[0] + j];
        const int steps = head[5], slices = ch_cuts(a.slices, steps).slices;
        auto slice = [&](int s) { return (int)(((long long)(s + 1) * slices - 1) / steps); };  // that holds step s
        const int w0 = slice(c.begin), w1 = slice(c.begin + c.tiles - 1);
        const size_t rec = (size_t)g * (a.slices + a.few) + j;
        for (int r = wave; r < GRP * c.count; r += 4)
            ch_join_row<LSE>(a, a.few_o, a.few_ml, (size_t)(c.row0 + r / GRP) * NH + g * GRP + r % GRP, w0, w1, lane,
                             [&](int w) { return (rec + w) * CH_FEW_ROWS + r; });
        return;
    }
    const ChunkCuts cuts = ch_cuts(a.slices, head[0], head[1], head[6]);
    const int part = blockIdx.x % parts;
    auto rows = [&](const ChunkBlock& c, int w0, int w1, auto place) {
        for (int r = CH_JR * part + wave; r < CH_JR * (part + 1); r += 4) {
            const int row = CH_ROWS * c.blk + r;
            if (row >= GRP * c.count) return;
            ch_join_row<LSE>(a, a.part_o, a.part_ml, (size_t)(c.row0 + row / GRP) * NH + g * GRP + row % GRP, w0, w1, lane,
                             [&](int w) { return (((size_t)g * a.slices + w) * 2 + place(w)) * a.prows + r; });
        }
    };
    if (cuts.part > 0) {  // blocks in slices of their own (where one is cut there are fewer blocks than slices)
        const int j = cut - 1;
        if (j >= head[0]) return;
        const ChunkBlock c = blocks[j];
        const int n = (c.tiles + cuts.part - 1) / cuts.part;
        if (n == 1) return;
        int w0 = 0;  // the parts of the blocks before it
        for (int i = lane; i < j; i += 64) w0 += (blocks[i].tiles + cuts.part - 1) / cuts.part;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) w0 += __shfl_xor(w0, o, 64);
        w0 = __builtin_amdgcn_readfirstlane(w0);
        rows(c, w0, w0 + n - 1, [](int) { return 0; });
        return;
    }
    if (cut >= cuts.slices) return;
    const int s = cuts.cut(cut), s_before = cuts.cut(cut - 1);
    const int j = ch_find(blocks, head[0], cuts.extra, s, &found);
    const ChunkBlock c = blocks[j];
    // the cut lies before the block's first tile, or an earlier one lies behind that
    const int begin = c.begin + cuts.extra * j, first = begin + cuts.extra;
    if (s <= first || s_before > first) return;
    // its slices: cut - 1 up to the one that holds its last tile
    const int last = first + c.tiles - 1;
    int w1 = cut;
    while (w1 + 1 < cuts.slices && cuts.cut(w1 + 1) <= last) w1++;
    rows(c, cut - 1, w1, [&](int w) { return w == cut - 1 && begin > s_before ? 1 : 0; });
}

hipError_t launch_prefill_batch(const float* q, const float* gate, const qwa_kv_layer& kv, int kvt, const qwa_kv_pages& p,
                                const int* seqs, const int* off, int n, int rows, int max_len, uint16_t* out16, float* lse,
                                void* work, hipStream_t st) {
    const ChunkPlan pl = chunk_plan(n, rows, max_len);
    const ChunkWork w = chunk_work(pl);
    uint8_t* base = static_cast<uint8_t*>(work);
    ChunkBlock* blocks = reinterpret_cast<ChunkBlock*>(base + w.blocks);
    int* head = reinterpret_cast<int*>(base + w.head);
    int4* list = reinterpret_cast<int4*>(base + w.list);
    const ChunkSource src{p, seqs, off, n, rows, max_len, pl.few > 0 ? CH_FEW : 0};
    const ChunkArgs a{src, pl.own, q, gate, out16, lse, blocks, list, head, reinterpret_cast<ChunkImage*>(base + w.images),
                      reinterpret_cast<float*>(base + w.o), reinterpret_cast<float4*>(base + w.ml),
                      reinterpret_cast<float*>(base + w.few_o), reinterpret_cast<float4*>(base + w.few_ml), pl.slices, pl.rows,
                      pl.few};
    if (!pl.own)
        launch_plan<false>(src, pl.blocks, pl.images, pl.tiles, blocks, list, head, st);
    if (pl.tiles > 0) {
        const dim3 ig((unsigned)std::min(pl.tiles * NKV, CH_IMG_WGS));
        switch (kvt) {
            case QWA_KV_F16: hipLaunchKernelGGL(k_ch_image<QWA_KV_F16>, ig, dim3(512), 0, st, a, kv, p); break;
            case QWA_KV_Q8_0: hipLaunchKernelGGL(k_ch_image<QWA_KV_Q8_0>, ig, dim3(512), 0, st, a, kv, p); break;
            default: hipLaunchKernelGGL(k_ch_image<QWA_KV_Q4_0>, ig, dim3(512), 0, st, a, kv, p); break;
        }
    }
    const dim3 grid(pl.slices * NKV), block(128 * CH_PAIRS);
#define QWA_CH(T)                                                                              \
    case T:                                                                                    \
        if (lse) hipLaunchKernelGGL((k_ch_tiles<T, true>), grid, block, 0, st, a, kv, p);      \
        else hipLaunchKernelGGL((k_ch_tiles<T, false>), grid, block, 0, st, a, kv, p);         \
        break
    switch (kvt) {
        QWA_CH(QWA_KV_F16);
        QWA_CH(QWA_KV_Q8_0);
        default: QWA_CH(QWA_KV_Q4_0);
    }
#undef QWA_CH
    if (pl.join) {
        const int parts = (pl.rows + CH_JR - 1) / CH_JR;
        const dim3 jg((pl.slices - 1) * parts + pl.few, NKV);
        if (lse) hipLaunchKernelGGL(k_ch_join<true>, jg, dim3(256), 0, st, a, parts);
        else hipLaunchKernelGGL(k_ch_join<false>, jg, dim3(256), 0, st, a, parts);
    }
    return hipGetLastError();
}

// ---- the weights: for position j of a sequence and KV head g, the sum over the chunk's rows (token, head of g) that see it of
// exp(s_j - lse), added to what it had (the chunk's own positions begin with it).
struct WeightsArgs {
    ChunkSource src;
    bool own;                  // every workgroup makes the plan itself
    const float* q;
    const float* lse;          // [rows][24]
    float* mass;               // [sequence][KV head][ld * page]
    const ChunkBlock* blocks;
    const int4* list;          // chunks of several blocks: sequence, length, tokens, first place
    const int* head;           // numbers of blocks, their tiles, such chunks, places
    float* parts;              // [place][KV head][max_len]
    int slices, max_len;
};

size_t weights_batch_work_bytes(int n, int rows, int max_len) {
    return weights_work(weights_plan(n, rows, max_len), max_len).bytes;
}

constexpr int CW_WAVES = CW_ROWS / 32;
template <int KVT>
struct WeightsLds {
    _Float16 k[2][CW_TILE * HD];
    uint16_t scales[2][CW_TILE * 8];
    int dead[2];                       // of the tile, groups of 16 keys without a place
    float sum[2][CW_WAVES][CW_TILE];   // of the waves' rows, by key
    uint2 q[CW_WAVES][16 * HD / 8];
    int found;
    OwnPlan plan;
};

// A workgroup walks the 64-key tiles of a slice as k_ch_tiles does, with K alone: all waves convert it, then each takes the scores
// of its 32 rows, and the sums over them; the workgroup's sum of a tile is written while the next one is multiplied.  1000 tokens
// over 16384 Q4_0 positions 460 to 520 us, 0.43 PFLOP/s, 0.85 with both parts of Q: of a SIMD's cycles 39% are MFMAs and 54% issue
// VALU instructions (a block scale's product for each score and 32 dims, exponentials, sums over rows, and K's conversion, which
// each of its 24 blocks does for itself), which its two waves, at the same step of a tile, rarely overlap; <Q8_0> keeps 15 registers
// in scratch, <Q4_0> 8.  A token in each of 16 sequences of 6000 to 16000 positions: F16 108 us, 367 MB at 3.4 TB/s, Q8_0 117,
// Q4_0 109.  What the three types have in common there is a tile's chain: conversion, a barrier, scores by two of eight waves.
template <int KVT>
__global__ void __launch_bounds__(64 * CW_WAVES) __attribute__((amdgpu_waves_per_eu(2, 2)))
k_cw_tiles(WeightsArgs a, qwa_kv_layer kv, qwa_kv_pages p) {
    __shared__ __attribute__((aligned(16))) WeightsLds<KVT> lds;
    constexpr bool SC = KVT != QWA_KV_F16;
    constexpr int G = CW_TILE / 16;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    int unit = blockIdx.x;
    if (gridDim.x % 8 == 0) unit = (int)(gridDim.x / 8) * (blockIdx.x & 7) + (blockIdx.x >> 3);
    const int g = unit / a.slices, w = unit % a.slices;
    const ChunkBlock* blocks = a.blocks;
    const int* head_of = a.head;
    if (a.own) {
        ch_own_plan<true>(lds.plan, a.src);
        blocks = lds.plan.blocks;
        head_of = lds.plan.head;
    }
    const int nb = __builtin_amdgcn_readfirstlane(head_of[0]), tiles = __builtin_amdgcn_readfirstlane(head_of[1]);
    const ChunkCuts cuts = ch_cuts(a.slices, tiles);
    if (w >= cuts.slices) return;
    int s = cuts.cut(w);
    const int s_end = cuts.cut(w + 1);
    int j = ch_find(blocks, nb, 0, s, &lds.found);
    const size_t head = (size_t)g * kv.capacity;
    const uint8_t* const kh = kv.k + head * value_bytes(KVT);
    const uint16_t* const ksh = SC ? kv.ks + head * 8 : nullptr;
    while (s < s_end) {
        // (an opaque copy of the thread: addresses kept across the segments took registers of the loop over tiles)
        int t = threadIdx.x;
        asm volatile("" : "+v"(t));
        const int lane = t & 63, i16 = lane & 15;
        const ChunkBlock c = ch_block(blocks[j]);
        const int tb = s - c.begin, nt = min(s_end, c.begin + c.tiles) - s;
        const int nrows = GRP * c.count;
        // (a block of one wave's rows: two waves have them, and half of the keys each; 16 tokens over 6000 to 16000 F16 positions
        // 109 us instead of 136)
        const bool few = nrows <= 32;
        const int wrow0 = few ? 0 : CW_ROWS * c.blk + 32 * wave;
        const bool rows_here = few ? wave < 2 : wrow0 < nrows;
        const int* __restrict__ table = p.table + (size_t)max(c.seq, 0) * p.ld;
        int vis[2], vmin = 0x7fffffff;  // (0 with a row that there is not: what it has is left out like a hidden position)
        float lse[2];
#pragma unroll
        for (int rt = 0; rt < 2; rt++) {
            const int r = wrow0 + 16 * rt + i16;
            vis[rt] = r < nrows ? c.len - c.count + r / GRP + 1 : 0;
            vmin = min(vmin, vis[rt]);
            lse[rt] = r < nrows ? a.lse[(size_t)(c.row0 + r / GRP) * NH + g * GRP + r % GRP] : 0.0f;
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) vmin = min(vmin, __shfl_xor(vmin, o, 64));
        vmin = __builtin_amdgcn_readfirstlane(vmin);
        BtRaw<KVT> rk[2];
        ChunkPlaces<G> places;
        int dead_next = 0;  // groups without a place, four bits a tile, of the next tile to be stored first
        const int grp = __builtin_amdgcn_readfirstlane(t >> 7);  // the thread's group of 16 keys
        auto load = [&](BtRaw<KVT>& rk, int i, int ahead) {
            int at[G];
            places.next(at, p, table, tb, c.end, lane);
            const int mine = grp == 0 ? at[0] : grp == 1 ? at[1] : grp == 2 ? at[2] : at[3];
            dead_next |= ((at[0] < 0) | (at[1] < 0) << 1 | (at[2] < 0) << 2 | (at[3] < 0) << 3) << (G * ahead);
            bt_load_k<KVT>(rk, kh, ksh, mine, min(max(c.end - (tb + i) * CW_TILE - 16 * grp, 0), 16), t);
        };
        auto store = [&](BtRaw<KVT>& rk, int i) {
            const int b = i & 1, h = t >> 8;
            bt_store_k<KVT>(rk, lds.k[b] + PF_TILE * HD * h, lds.scales[b] + PF_TILE * 8 * h, t);
            if (t == 0) lds.dead[b] = dead_next & ((1 << G) - 1);
            dead_next >>= G;
        };
        // The sums of tile i: to the block's place, or to the sequence's weights, whose old values are read a tile ahead.  The
        // last wave does it: of chunks of few tokens it is one that has no rows.
        const bool writes = wave == CW_WAVES - 1;
        float* const mass = a.mass + ((size_t)max(c.seq, 0) * NKV + g) * ((size_t)p.ld * p.page);
        // (What no token sees is left as it is, a position without a place too; k_cw_join looks at the pages itself.)
        float old = 0.0f;
        bool unseen = false;
        auto fetch = [&](int i) {
            const int key = (tb + i) * CW_TILE + lane;
            if (!writes || c.place >= 0) return;
            old = key < c.len - c.count ? mass[key] : 0.0f;
            unseen = (lds.dead[i & 1] >> (lane >> 4)) & 1;
        };
        auto write = [&](int i) {
            const int key = (tb + i) * CW_TILE + lane;
            if (!writes || key >= c.end || unseen) return;
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < CW_WAVES; k++) v += lds.sum[i & 1][k][lane];
            if (c.place >= 0) a.parts[((size_t)c.place * NKV + g) * a.max_len + key] = v;
            else mass[key] = old + v;
        };
        load(rk[0], 0, 0);
        if (nt > 1) load(rk[1], 1, 1);
        h8 qb[2][2][8];
        ch_load_q<KVT>(qb, a.q, c, wrow0, nrows, g, lds.q[wave], lane);
        store(rk[0], 0);
        if (nt > 2) load(rk[0], 2, 1);
        __syncthreads();
        auto step = [&](int i, BtRaw<KVT>& rk) __attribute__((always_inline)) {
            const int k0 = (tb + i) * CW_TILE, b = i & 1;
            if (i > 0) write(i - 1);
            fetch(i);
            if (i + 1 < nt) store(rk, i + 1);
            if (i + 3 < nt) load(rk, i + 3, 1);
            int ol = lane;  // (opaque: LDS addresses kept across the tiles)
            asm volatile("" : "+v"(ol));
            const int oi = ol & 15, og = ol >> 4;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                f4 sum[2] = {};
                if (rows_here && (!few || h == wave)) {
                    f4 sc[2][2];
                    ch_scores<KVT>(sc, qb, lds.k[b] + PF_TILE * HD * h,
                                   reinterpret_cast<const _Float16*>(lds.scales[b] + PF_TILE * 8 * h), oi, og);
                    const int dead = __builtin_amdgcn_readfirstlane(lds.dead[b]) >> (2 * h);
                    const bool masked = k0 + CW_TILE > vmin || dead != 0;
#pragma unroll
                    for (int rt = 0; rt < 2; rt++)
#pragma unroll
                        for (int kt = 0; kt < 2; kt++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                float x = (sc[rt][kt][e] - lse[rt]) * PF_LOG2E;
                                if (masked)
                                    x = k0 + 32 * h + 16 * kt + 4 * og + e < vis[rt] && !((dead >> kt) & 1) ? x : -INFINITY;
                                sum[kt][e] += fast_exp2(x);
                            }
                }
                // over the 16 rows of the lanes
#pragma unroll
                for (int kt = 0; kt < 2; kt++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        float x = sum[kt][e];
                        x += row_move<0xB1>(x);
                        x += row_move<0x4E>(x);
                        x += row_move<0x141>(x);
                        x += row_move<0x140>(x);
                        sum[kt][e] = x;
                    }
                    if (oi == 0)
                        *reinterpret_cast<f4*>(&lds.sum[b][wave][32 * h + 16 * kt + 4 * og]) = sum[kt];
                }
            }
            __syncthreads();
        };
        for (int i = 0; i < nt; i += 2) {
            step(i, rk[1]);
            if (i + 1 < nt) step(i + 1, rk[0]);
        }
        write(nt - 1);
        // (the next segment's first sums are written behind its first barrier)
        s += nt;
        j++;
    }
}

// The weights of chunks of several blocks: the blocks' sums in order (24 blocks of 17384 positions, 6.7 MB, 16 us).
__global__ void __launch_bounds__(256) k_cw_join(WeightsArgs a, size_t ld_pos) {
    __shared__ OwnPlan plan;
    if (a.own) ch_own_plan<true>(plan, a.src);
    const int g = blockIdx.y, n = a.own ? plan.head[2] : a.head[2];
    for (int k = blockIdx.z; k < n; k += gridDim.z) {
        const int4 c = a.own ? plan.list[k] : a.list[k];
        const int nb = (GRP * c.z + CW_ROWS - 1) / CW_ROWS;
        for (int key = blockIdx.x * 256 + threadIdx.x; key < c.y; key += gridDim.x * 256) {
            // the first block that sees the position: the first whose last row does
            const int r = GRP * max(0, key - (c.y - c.z)), b0 = r / CW_ROWS;
            float v = 0.0f;
            for (int b = b0; b < nb; b++) v += a.parts[((size_t)(c.w + b) * NKV + g) * a.max_len + key];
            float* const m = a.mass + ((size_t)c.x * NKV + g) * ld_pos + key;
            if (bt_place(a.src.p, a.src.p.table + (size_t)c.x * a.src.p.ld, key & ~15, c.y) >= 0)
                *m = key < c.y - c.z ? *m + v : v;
        }
    }
}

hipError_t launch_weights_batch(const float* q, const float* lse, const qwa_kv_layer& kv, int kvt, const qwa_kv_pages& p,
                                const int* seqs, const int* off, int n, int rows, int max_len, float* mass, void* work,
                                hipStream_t st) {
    const WeightsPlan pl = weights_plan(n, rows, max_len);
    const WeightsWork w = weights_work(pl, max_len);
    uint8_t* base = static_cast<uint8_t*>(work);
    ChunkBlock* blocks = reinterpret_cast<ChunkBlock*>(base + w.blocks);
    int4* list = reinterpret_cast<int4*>(base + w.list);
    int* head = reinterpret_cast<int*>(base + w.head);
    const ChunkSource src{p, seqs, off, n, rows, max_len, 0};
    const WeightsArgs a{src, pl.own, q, lse, mass, blocks, list, head, reinterpret_cast<float*>(base + w.parts), pl.slices, max_len};
    if (!pl.own)
        launch_plan<true>(src, pl.blocks, pl.parts / 2, pl.parts, blocks, list, head, st);
    const dim3 grid(pl.slices * NKV), block(64 * CW_WAVES);
    switch (kvt) {
        case QWA_KV_F16: hipLaunchKernelGGL(k_cw_tiles<QWA_KV_F16>, grid, block, 0, st, a, kv, p); break;
        case QWA_KV_Q8_0: hipLaunchKernelGGL(k_cw_tiles<QWA_KV_Q8_0>, grid, block, 0, st, a, kv, p); break;
        default: hipLaunchKernelGGL(k_cw_tiles<QWA_KV_Q4_0>, grid, block, 0, st, a, kv, p); break;
    }
    if (pl.parts > 0) {
        const dim3 jg((unsigned)std::min(64, (max_len + 255) / 256), NKV, (unsigned)std::min(pl.parts / 2, 16));
        hipLaunchKernelGGL(k_cw_join, jg, dim3(256), 0, st, a, (size_t)p.ld * p.page);
    }
    return hipGetLastError();
}

}  // namespace qwa
