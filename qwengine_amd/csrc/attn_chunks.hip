// Attention of a batch of chunks of new tokens over a paged cache (gfx950).
//
// Batch row b has the tokens off[b] .. off[b + 1] - 1, the last c = off[b + 1] - off[b] positions of its sequence; token t of it
// sees positions [0, len - c + t].  For row r = (token, head):  out = sum_j p_j V_j / sum_j p_j * sigmoid(gate),
// p_j = exp(s_j), s_j = q_r . K_j / 16, and log sum_j p_j for who asks for it.
//  * A block is CH_ROWS consecutive rows (6 * token + head of the group) of a chunk; its keys are walked in 32-key tiles.  The tiles
//    of all blocks in a row are cut into equal slices, a workgroup each: a long sequence's decoded token and a prompt of
//    a thousand load the chip alike.  A block that lies in several slices leaves partial states, which k_ch_join joins in the
//    slices' order; the others are finished where they are.
//  * A workgroup has two waves a SIMD, with a role each.  The score waves keep Q (32 rows: hi and lo part, 128 registers), take
//    S^T = K Q^T of tile i, the exponentials, and leave P in LDS.  The value waves keep O (32 rows, 128 registers), add V^T P^T of
//    tile i - 1, and bring the next tiles from the cache into LDS.  So each fragment of K and V that is read from LDS meets 32
//    rows, which one wave with both Q and O has no registers for, and the exponentials of one wave run beside the other's MFMAs.
//  * Scores are exact up to fp32 accumulation (K as its codes, Q / 16 as the sum of two fp16 parts), as the batched decode's are;
//    the arithmetic of a tile, of V that is not finite and of the probabilities' range is paged_tiles.hpp's.
// Roundings below 32 bits: the dequantized V (d * code) and the probabilities are fp16, half a step 2^-11 of the value; the sum of a
// row's probabilities is that of the rounded ones, which P V applies, but the log of the sum is taken of the unrounded.  The
// output is fp16.
#include <type_traits>

#include "chunk_plan.hpp"
#include "launch.hpp"
#include "paged_tiles.hpp"

namespace qwa {

// a block: its chunk's first row and number of tokens, the sequence's length and number (< 0: unknown, len 0), the block's number in
// the chunk, its first tile in the row of all tiles, its tiles
struct alignas(16) ChunkBlock {
    int row0, count, len, seq;
    int blk, begin, tiles, end;  // end: positions that its last row sees
};
static_assert(sizeof(ChunkBlock) == CH_BLOCK_BYTES, "work buffer");

struct ChunkArgs {
    const float* q;
    const float* gate;
    uint16_t* out16;
    float* lse;              // [rows][24] or none
    const ChunkBlock* blocks;
    const int* head;         // number of blocks, number of tiles
    float* part_o;           // [KV head][slice][2][rows][256]
    float4* part_ml;         // [KV head][slice][2][rows]
    int slices, prows;
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
// earlier one's end, has none.
constexpr int CH_PT = QWA_PAGES_MAXN;
__global__ void __launch_bounds__(CH_PT) k_ch_plan(qwa_kv_pages p, const int* __restrict__ seqs, const int* __restrict__ off, int n,
                                                   int rows, int max_len, int most, ChunkBlock* __restrict__ blocks,
                                                   int* __restrict__ head) {
    __shared__ int s_wave[CH_PT / 64];
    __shared__ int s_end[CH_PT], s_first[CH_PT], s_count[CH_PT], s_len[CH_PT], s_seq[CH_PT], s_blk[CH_PT + 1];
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
    const int count = end > first && before <= first ? end - first : 0;
    const int seq = t < n ? (seqs ? seqs[t] : t) : -1;
    const bool known = seq >= 0 && seq < p.n_seq;
    s_first[t] = first;
    s_count[t] = count;
    s_len[t] = known && count > 0 ? min(max(p.len[seq], 0), max_len) : 0;
    s_seq[t] = known ? seq : -1;
    int nb;
    const int mine = (GRP * count + CH_ROWS - 1) / CH_ROWS;
    s_blk[t] = ch_scan<CH_PT>(mine, s_wave, &nb);
    if (t == CH_PT - 1) s_blk[CH_PT] = nb;
    __syncthreads();
    nb = min(nb, most);  // (never more: the chunks' rows are disjoint)
    int tiles = 0;
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
            const int last = min((x.blk + 1) * CH_ROWS, GRP * x.count) - 1;
            x.end = max(0, x.len - x.count + last / GRP + 1);
            x.tiles = max(1, (x.end + PF_TILE - 1) / PF_TILE);  // (rows that see nothing are written too)
        }
        int all;
        x.begin = tiles + ch_scan<CH_PT>(x.tiles, s_wave, &all);
        tiles += all;
        if (j < nb) blocks[j] = x;
    }
    if (t == 0) {
        head[0] = nb;
        head[1] = tiles;
    }
}

// slices that hold tiles: the same number for every workgroup of a call
__device__ __forceinline__ int ch_slices(const ChunkArgs& a, int tiles) { return min(a.slices, tiles); }
__device__ __forceinline__ int ch_cut(int w, int tiles, int slices) { return (int)((long long)w * tiles / slices); }

// the block that holds tile s, found by the whole workgroup
__device__ __forceinline__ int ch_find(const ChunkArgs& a, int nb, int s, int* s_found) {
    for (int j = threadIdx.x; j < nb; j += blockDim.x) {
        const int begin = a.blocks[j].begin;
        if (begin <= s && s < begin + a.blocks[j].tiles) *s_found = j;
    }
    __syncthreads();
    return __builtin_amdgcn_readfirstlane(*s_found);
}

constexpr int CH_VD = 3;  // V fragments in flight

template <int KVT>
struct ChunkLds {
    _Float16 k[2][PF_TILE * HD];
    _Float16 vt[2][PF_TILE * HD];
    uint16_t scales[2][KVT == QWA_KV_F16 ? 8 : PF_TILE * 8];  // of K
    BtOdd odd[2];                                             // of V
    int dead[4];                                              // by tile: halves without a place
    h8 p[2][CH_PAIRS][2][64];                                 // P^T of a tile, as operands
    float cr[2][CH_PAIRS][2][16];                             // what O is multiplied by before it, where it is
    int moved[2][CH_PAIRS];                                   // ... anything but 1
    float4 ml[CH_PAIRS][2][16];                               // of a finished segment: m, l, the log's sum
    union {
        uint2 q[CH_PAIRS][16 * HD / 4];                       // a row tile's Q, one part, on its way into operands
        float4 x[CH_PAIRS][16 * HD / 8];                      // half of a row tile's O on its way out
    };
    int found;
};

template <int KVT, bool LSE>
__global__ void __launch_bounds__(128 * CH_PAIRS) __attribute__((amdgpu_waves_per_eu(2, 2)))
k_ch_tiles(ChunkArgs a, qwa_kv_layer kv, qwa_kv_pages p) {
    __shared__ __attribute__((aligned(16))) ChunkLds<KVT> lds;
    constexpr bool SC = KVT != QWA_KV_F16;
    const int t = threadIdx.x, lane = t & 63, i16 = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int pair = wave & (CH_PAIRS - 1);
    // workgroups 8 apart run on one XCD: each has consecutive slices of one head, whose tiles its L2 then holds
    int unit = blockIdx.x;
    if (gridDim.x % 8 == 0) unit = (int)(gridDim.x / 8) * (blockIdx.x & 7) + (blockIdx.x >> 3);
    const int g = unit / a.slices, w = unit % a.slices;
    const int nb = a.head[0], tiles = a.head[1];
    const int slices = ch_slices(a, tiles);
    if (w >= slices) return;
    int s = ch_cut(w, tiles, slices);
    const int s_begin = s, s_end = ch_cut(w + 1, tiles, slices);
    int j = ch_find(a, nb, s, &lds.found);
    const size_t head = (size_t)g * kv.capacity;
    const uint8_t* const kh = kv.k + head * value_bytes(KVT);
    const uint8_t* const vh = kv.v + head * value_bytes(KVT);
    const uint16_t* const ksh = SC ? kv.ks + head * 8 : nullptr;
    const uint16_t* const vsh = SC ? kv.vs + head * 8 : nullptr;

    auto walk = [&](auto role) __attribute__((always_inline)) {
        constexpr bool VALUES = decltype(role)::value;
        while (s < s_end) {
            const ChunkBlock c = a.blocks[j];
            const int tb = s - c.begin, nt = min(s_end, c.begin + c.tiles) - s;
            const int end = __builtin_amdgcn_readfirstlane(c.end), nrows = __builtin_amdgcn_readfirstlane(GRP * c.count);
            const int wrow0 = __builtin_amdgcn_readfirstlane(CH_ROWS * c.blk) + 32 * pair;
            const bool rows_here = wrow0 < nrows;
            int vis[2];  // positions that this lane's rows see
#pragma unroll
            for (int rt = 0; rt < 2; rt++) {
                const int r = wrow0 + 16 * rt + i16;
                vis[rt] = r < nrows ? c.len - c.count + r / GRP + 1 : 0;
            }
            if constexpr (VALUES) {
                const int* __restrict__ table = p.table + (size_t)max(c.seq, 0) * p.ld;
                BtRaw<KVT> rk, rv;
                // the pool positions of the tiles' halves, 64 tiles ahead: lane l has those of tile l
                int ahead[2], at[2], tile = 0;
                auto place = [&]() {
                    if ((tile & 63) == 0)
#pragma unroll
                        for (int h = 0; h < 2; h++) ahead[h] = bt_place(p, table, (tb + tile + lane) * PF_TILE + 16 * h, end);
#pragma unroll
                    for (int h = 0; h < 2; h++) at[h] = __builtin_amdgcn_readlane(ahead[h], tile & 63);
                    tile++;
                };
                auto bits = [&]() { return (uint32_t)((at[0] < 0) | (at[1] < 0) << 1); };
                auto load_k = [&](int i) {
                    const int h = pair >> 1, left = end - (tb + i) * PF_TILE - 16 * h;
                    bt_load_k<KVT>(rk, kh, ksh, h ? at[1] : at[0], min(max(left, 0), 16), t);
                };
                auto load_v = [&](int i) {
                    const int left = end - (tb + i) * PF_TILE;
                    const int rows[2] = {at[0] < 0 ? 16 : min(left, 16), at[1] < 0 ? 16 : min(left - 16, 16)};
                    bt_load_v<KVT>(rv, vh, vsh, at, rows, t);
                };
                auto store_k = [&](int i, uint32_t dead) {
                    bt_store_k<KVT>(rk, lds.k[i & 1], lds.scales[i & 1], t);
                    if (wave == CH_PAIRS && lane == 0) lds.dead[i & 3] = (int)dead;
                };
                f4 o[2][16];
#pragma unroll
                for (int rt = 0; rt < 2; rt++)
#pragma unroll
                    for (int dt = 0; dt < 16; dt++) o[rt][dt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
                place();
                load_k(0);
                load_v(0);
                uint32_t dead_v = bits(), dead_k = dead_v;
                if (wave == CH_PAIRS && lane < 8) lds.odd[lane >> 2].tile[lane & 3] = -1;
                store_k(0, dead_k);
                if (nt > 1) {
                    place();
                    load_k(1);
                    dead_k = bits();
                }
                __syncthreads();
                for (int i = 0; i <= nt; i++) {
                    // K of tile i + 1 and V of tile i into LDS, then their successors' loads
                    if (i + 1 < nt) store_k(i + 1, dead_k);
                    if (i < nt) bt_store_v<KVT>(rv, lds.vt[i & 1], lds.odd[i & 1], t, dead_v, i);
                    if (i + 1 < nt) {
                        load_v(i + 1);
                        dead_v = dead_k;
                    }
                    if (i + 2 < nt) {
                        place();
                        load_k(i + 2);
                        dead_k = bits();
                    }
                    if (i > 0 && rows_here) {
                        const int b = (i - 1) & 1;
                        if (__builtin_amdgcn_readfirstlane(lds.moved[b][pair])) {
#pragma unroll
                            for (int rt = 0; rt < 2; rt++) {
                                const float f = lds.cr[b][pair][rt][i16];
#pragma unroll
                                for (int dt = 0; dt < 16; dt++) o[rt][dt] *= f;
                            }
                        }
                        h8 pb[2];
#pragma unroll
                        for (int rt = 0; rt < 2; rt++) pb[rt] = lds.p[b][pair][rt][lane];
                        // O^T += V^T P^T
                        const _Float16* vrow = lds.vt[b] + 8 * (256 * lg + i16);
                        h8 vf[CH_VD];
#pragma unroll
                        for (int dt = 0; dt < CH_VD - 1; dt++) vf[dt] = lds_h8(vrow + 8 * 16 * dt);
#pragma unroll
                        for (int dt = 0; dt < 16; dt++) {
                            if (dt + CH_VD - 1 < 16) vf[(dt + CH_VD - 1) % CH_VD] = lds_h8(vrow + 8 * 16 * (dt + CH_VD - 1));
#pragma unroll
                            for (int rt = 0; rt < 2; rt++) o[rt][dt] = mfma16(vf[dt % CH_VD], pb[rt], o[rt][dt]);
                        }
                        // a dim is NaN in the rows that see a value of it that is not finite
                        const int4 of4 = *reinterpret_cast<const int4*>(lds.odd[b].tile);
                        if (__builtin_amdgcn_readfirstlane(of4.x == i - 1 || of4.y == i - 1 || of4.z == i - 1 || of4.w == i - 1)) {
                            const int of[4] = {of4.x, of4.y, of4.z, of4.w};
                            const int k0 = (tb + i - 1) * PF_TILE, dead = lds.dead[(i - 1) & 3];
                            uint32_t seen[2][2] = {};
#pragma unroll
                            for (int rt = 0; rt < 2; rt++)
#pragma unroll
                                for (int k = 0; k < PF_TILE; k++) {
                                    const int cb = k / 4 % 4, h = k / 16;
                                    if (of[cb] == i - 1 && k0 + k < vis[rt] && !((dead >> h) & 1))
                                        seen[rt][cb / 2] |= 1u << (8 * (2 * (cb & 1) + h) + k % 4);
                                }
#pragma unroll
                            for (int dt = 0; dt < 16; dt++) {
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const int dim = 8 * (16 * (dt & 1) + 4 * lg + e) + (dt >> 1);
                                    const uint2 keys = *reinterpret_cast<const uint2*>(&lds.odd[b].keys[8 * dim]);
#pragma unroll
                                    for (int rt = 0; rt < 2; rt++)
                                        o[rt][dt][e] =
                                            ((keys.x & seen[rt][0]) | (keys.y & seen[rt][1])) != 0 ? NAN : o[rt][dt][e];
                                }
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                    }
                    if (i < nt) __syncthreads();
                }
                // O by way of LDS, half of the dims at a time, so that rows are written as they lie in memory
                const bool whole = nt == c.tiles;
                const size_t part = (((size_t)g * a.slices + w) * 2 + (s == s_begin ? 0 : 1)) * a.prows;
                if (rows_here) {
                    float4* const area = lds.x[pair];
#pragma unroll
                    for (int rt = 0; rt < 2; rt++)
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            // o[rt][2 k + e][j] is dim 8 x + k, x = 16 e + 4 lg + j: unit 2 (4 lg + j) + k / 4 of the half
#pragma unroll
                            for (int jj = 0; jj < 4; jj++)
#pragma unroll
                                for (int h = 0; h < 2; h++)
                                    area[32 * i16 + ((2 * (4 * lg + jj) + h) ^ (i16 & 7))] =
                                        make_float4(o[rt][8 * h + e][jj], o[rt][8 * h + 2 + e][jj], o[rt][8 * h + 4 + e][jj],
                                                    o[rt][8 * h + 6 + e][jj]);
                            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the area is the wave's own)
                            __builtin_amdgcn_wave_barrier();
#pragma unroll
                            for (int k = 0; k < 8; k++) {
                                const int xr = 2 * k + (lane >> 5), u = lane & 31, r = wrow0 + 16 * rt + xr;
                                const float4 v = area[32 * xr + (u ^ (xr & 7))];
                                if (r < nrows) {
                                    const int dim = 128 * e + 4 * u;
                                    if (whole) {
                                        const size_t at0 = ((size_t)(c.row0 + r / GRP) * NH + g * GRP + r % GRP) * HD + dim;
                                        const float l = lds.ml[pair][rt][xr].y, il = l == 0.0f ? 0.0f : 1.0f / l;
                                        const float4 gv = *reinterpret_cast<const float4*>(a.gate + at0);
                                        *reinterpret_cast<uint2*>(a.out16 + at0) =
                                            make_uint2((uint32_t)f2h_bits(v.x * il * sigmoid(gv.x)) |
                                                           ((uint32_t)f2h_bits(v.y * il * sigmoid(gv.y)) << 16),
                                                       (uint32_t)f2h_bits(v.z * il * sigmoid(gv.z)) |
                                                           ((uint32_t)f2h_bits(v.w * il * sigmoid(gv.w)) << 16));
                                    } else {
                                        *reinterpret_cast<float4*>(a.part_o + (part + r - CH_ROWS * c.blk) * HD + dim) = v;
                                    }
                                }
                            }
                            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                            __builtin_amdgcn_wave_barrier();
                        }
#pragma unroll
                    for (int rt = 0; rt < 2; rt++) {
                        const int r = wrow0 + 16 * rt + i16;
                        if (lg == 0 && r < nrows) {
                            const float4 ml = lds.ml[pair][rt][i16];
                            if (!whole) a.part_ml[part + r - CH_ROWS * c.blk] = ml;
                            else if (LSE)
                                a.lse[(size_t)(c.row0 + r / GRP) * NH + g * GRP + r % GRP] =
                                    ml.z == 0.0f ? -INFINITY : (ml.x + __log2f(ml.z)) * 0.6931471805599453f;
                        }
                    }
                }
                __syncthreads();
            } else {
                // Q / 16 as the B operand, hi and lo part: a row is read as one kilobyte, its fp16 pieces go to unit (s, lg,
                // row ^ (4 s + lg) % 16) of the wave's part of LDS and come back as the lane's fragments s
                h8 qb[2][2][8];
#pragma unroll
                for (int rt = 0; rt < 2; rt++) {
                    float4 x[16];
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const int rk = min(wrow0 + 16 * rt + k, nrows - 1);
                        x[k] = *reinterpret_cast<const float4*>(
                            a.q + ((size_t)(c.row0 + rk / GRP) * NH + g * GRP + rk % GRP) * HD + 4 * lane);
                    }
                    uint8_t* const area = reinterpret_cast<uint8_t*>(lds.q[pair]);
                    const int u = lane >> 1, half = lane & 1;  // piece u = 4 s + lg, dims 4 half .. 4 half + 3 of it
#pragma unroll
                    for (int part = 0; part < 2; part++) {
                        auto piece = [&](float v, float f) { return part ? q_lo(v * f) : q_hi(v * f); };
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            const float f = wrow0 + 16 * rt + k < nrows ? 0.0625f : 0.0f;
                            uint32_t w0 = h2_bits(h2{piece(x[k].x, f), piece(x[k].y, f)});
                            uint32_t w1 = h2_bits(h2{piece(x[k].z, f), piece(x[k].w, f)});
                            if constexpr (KVT == QWA_KV_Q4_0) {
                                // the operand's order [0, 4, 1, 5, 2, 6, 3, 7]: the even lane makes the first two words, the odd
                                // one the rest
                                const uint32_t mine = half ? w1 : w0;
                                const uint32_t other = __builtin_amdgcn_update_dpp(0, half ? w0 : w1, 0xB1, 0xF, 0xF, true);
                                const uint32_t lo = half ? other : mine, hi = half ? mine : other;
                                w0 = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
                                w1 = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
                            }
                            *reinterpret_cast<uint2*>(area + 16 * (16 * u + (k ^ (u & 15))) + 8 * half) = make_uint2(w0, w1);
                        }
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the area is the wave's own)
                        __builtin_amdgcn_wave_barrier();
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            qb[rt][part][k] =
                                *reinterpret_cast<const h8*>(area + 16 * (16 * (4 * k + lg) + (i16 ^ ((4 * k + lg) & 15))));
                        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                        __builtin_amdgcn_wave_barrier();
                    }
                }
                int vmin = 0x7fffffff;
#pragma unroll
                for (int rt = 0; rt < 2; rt++)
                    if (wrow0 + 16 * rt + i16 < nrows) vmin = min(vmin, vis[rt]);
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) vmin = min(vmin, __shfl_xor(vmin, o, 64));
                vmin = __builtin_amdgcn_readfirstlane(vmin);
                float m[2], l[2], lx[2];
#pragma unroll
                for (int rt = 0; rt < 2; rt++) {
                    m[rt] = -INFINITY;
                    l[rt] = lx[rt] = 0.0f;
                }
                __syncthreads();
                for (int i = 0; i < nt; i++) {
                    if (rows_here) {
                        const int k0 = (tb + i) * PF_TILE, b = i & 1;
                        const _Float16* Ks = lds.k[b];
                        const _Float16* Sc = reinterpret_cast<const _Float16*>(lds.scales[b]);
                        // S^T = K Q^T: lane (row i16 of row tile rt) gets keys k0 + 16 kt + 4 lg + e; the K fragments of a step
                        // are read while the step before multiplies, whose product is scaled while the next one is on its way
                        f4 sc[2][2] = {}, T[2][2][2];
                        h8 ks[2];  // scales of blocks s - 1 and s, s even, or s and s + 1
                        auto scale = [&](int st, int rt, int kt) {
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                sc[rt][kt][e] = fmaf((float)ks[kt][4 * (st & 1) + e], T[st & 1][rt][kt][e], sc[rt][kt][e]);
                        };
                        auto kfrag = [&](int st, int kt) {
                            return lds_h8(Ks + 8 * (32 * (4 * st + lg) + 16 * kt + (i16 ^ (2 * st))));
                        };
                        h8 kf[2][2];
#pragma unroll
                        for (int kt = 0; kt < 2; kt++) kf[0][kt] = kfrag(0, kt);
#pragma unroll
                        for (int st = 0; st < 8; st++) {
                            if (st + 1 < 8)
#pragma unroll
                                for (int kt = 0; kt < 2; kt++) kf[(st + 1) & 1][kt] = kfrag(st + 1, kt);
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int part = 1; part >= 0; part--)
#pragma unroll
                                for (int rt = 0; rt < 2; rt++)
#pragma unroll
                                    for (int kt = 0; kt < 2; kt++) {
                                        const h8 k8 = kf[st & 1][kt];
                                        if constexpr (SC) {
                                            const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                                            T[st & 1][rt][kt] = mfma16(k8, qb[rt][part][st], part ? zero : T[st & 1][rt][kt]);
                                        } else {
                                            sc[rt][kt] = mfma16(k8, qb[rt][part][st], sc[rt][kt]);
                                        }
                                    }
                            if constexpr (SC) {
                                if (st > 0)
#pragma unroll
                                    for (int rt = 0; rt < 2; rt++) {
                                        scale(st - 1, rt, 0);
                                        scale(st - 1, rt, 1);
                                    }
                                if (st % 2 == 0)
#pragma unroll
                                    for (int kt = 0; kt < 2; kt++) ks[kt] = lds_h8(Sc + 8 * (16 * kt + 2 * st + lg));
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        if constexpr (SC) {
#pragma unroll
                            for (int rt = 0; rt < 2; rt++) {
                                scale(7, rt, 0);
                                scale(7, rt, 1);
                            }
                        } else {
                            mfma_settle(sc[0][0], sc[0][1]);
                            mfma_settle(sc[1][0], sc[1][1]);
                        }
                        const int dead = __builtin_amdgcn_readfirstlane(lds.dead[i & 3]);
                        bool moved = false;
                        float cr[2];
#pragma unroll
                        for (int rt = 0; rt < 2; rt++) {
                            if (k0 + PF_TILE > vmin || dead != 0) {
#pragma unroll
                                for (int kt = 0; kt < 2; kt++)
#pragma unroll
                                    for (int e = 0; e < 4; e++)
                                        sc[rt][kt][e] = k0 + 16 * kt + 4 * lg + e < vis[rt] && !((dead >> kt) & 1)
                                                            ? sc[rt][kt][e] : -INFINITY;
                            }
                            float mx = max3f(max3f(-INFINITY, sc[rt][0][0], sc[rt][0][1]), sc[rt][0][2], sc[rt][0][3]);
                            mx = rows_max(max3f(max3f(mx, sc[rt][1][0], sc[rt][1][1]), sc[rt][1][2], sc[rt][1][3]));
                            const float mx2 = mx * PF_LOG2E, mn = mx2 > m[rt] + BT_HEAD ? mx2 - BT_RAISE : m[rt];
                            cr[rt] = mn == m[rt] ? 1.0f : fast_exp2(m[rt] - mn);
                            const float ref = mn == -INFINITY ? 0.0f : mn;  // a row that saw nothing keeps l = 0, O = 0
                            m[rt] = mn;
                            moved |= cr[rt] != 1.0f;
                            h8 pb;
                            float rx = 0.0f;
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                const float x = fast_exp2(fmaf(sc[rt][e >> 2][e & 3], PF_LOG2E, -ref));
                                pb[e] = (_Float16)x;
                                if (LSE) rx += x;
                            }
                            lds.p[b][pair][rt][lane] = pb;
                            // the sum of the rounded probabilities, the weights that P V applies
                            const h2 one2 = {(_Float16)1.0f, (_Float16)1.0f};
                            float rs = 0.0f;
#pragma unroll
                            for (int e = 0; e < 8; e += 2) rs = __builtin_amdgcn_fdot2(h2{pb[e], pb[e + 1]}, one2, rs, false);
                            l[rt] = l[rt] * cr[rt] + rs;
                            if (LSE) lx[rt] = lx[rt] * cr[rt] + rx;
                        }
                        const bool any = __any(moved);
                        if (any)
#pragma unroll
                            for (int rt = 0; rt < 2; rt++) lds.cr[b][pair][rt][i16] = cr[rt];
                        if (lane == 0) lds.moved[b][pair] = any;
                        if (i + 1 == nt) {
#pragma unroll
                            for (int rt = 0; rt < 2; rt++) {
                                const float4 ml = make_float4(m[rt], rows_sum(l[rt]), LSE ? rows_sum(lx[rt]) : 0.0f, 0.0f);
                                if (lg == 0) lds.ml[pair][rt][i16] = ml;
                            }
                        }
                    }
                    __syncthreads();
                }
                __syncthreads();
            }
            s += nt;
            j++;
        }
    };
    if (wave < CH_PAIRS) walk(std::false_type{});
    else walk(std::true_type{});
}

// Joins the states of the blocks that lie in several slices, in the slices' order: workgroup (cut between two slices, KV head,
// part of the rows) has the block that the cut lies in, if it is the first cut in it; a wave a row, 4 dims a lane.
constexpr int CH_JR = 16;  // rows of a workgroup
template <bool LSE>
__global__ void __launch_bounds__(256) k_ch_join(ChunkArgs a) {
    __shared__ int found;
    const int tiles = a.head[1], slices = ch_slices(a, tiles);
    const int g = blockIdx.y, cut = blockIdx.x + 1;
    if (cut >= slices) return;
    const int s = ch_cut(cut, tiles, slices), s_before = ch_cut(cut - 1, tiles, slices);
    const int j = ch_find(a, a.head[0], s, &found);
    const ChunkBlock c = a.blocks[j];
    if (c.begin == s || c.begin < s_before) return;  // the cut lies between two blocks, or an earlier one lies in this
    // its slices: cut - 1 up to the one that holds its last tile
    const int last = c.begin + c.tiles - 1;
    int w1 = cut;
    while (w1 + 1 < slices && ch_cut(w1 + 1, tiles, slices) <= last) w1++;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto place = [&](int w) {
        return (((size_t)g * a.slices + w) * 2 + (w == cut - 1 && c.begin != s_before ? 1 : 0)) * a.prows;
    };
    for (int r = CH_JR * blockIdx.z + wave; r < CH_JR * ((int)blockIdx.z + 1); r += 4) {
        const int row = CH_ROWS * c.blk + r;
        if (row >= GRP * c.count) return;
        const size_t out = (size_t)(c.row0 + row / GRP) * NH + g * GRP + row % GRP;
        const float4 gv = *reinterpret_cast<const float4*>(a.gate + out * HD + 4 * lane);
        float M = -INFINITY, L = 0.0f, X = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w0 = cut - 1; w0 <= w1; w0 += 4) {
            float4 ml[4], x[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const size_t at = place(min(w0 + u, w1)) + r;
                ml[u] = a.part_ml[at];
                x[u] = *reinterpret_cast<const float4*>(a.part_o + at * HD + 4 * lane);
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (w0 + u > w1) break;
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
            make_uint2((uint32_t)f2h_bits(acc.x * il * sigmoid(gv.x)) | ((uint32_t)f2h_bits(acc.y * il * sigmoid(gv.y)) << 16),
                       (uint32_t)f2h_bits(acc.z * il * sigmoid(gv.z)) | ((uint32_t)f2h_bits(acc.w * il * sigmoid(gv.w)) << 16));
        if (LSE && lane == 0) a.lse[out] = X == 0.0f ? -INFINITY : (M + __log2f(X)) * 0.6931471805599453f;
    }
}

hipError_t launch_prefill_batch(const float* q, const float* gate, const qwa_kv_layer& kv, int kvt, const qwa_kv_pages& p,
                                const int* seqs, const int* off, int n, int rows, int max_len, uint16_t* out16, float* lse,
                                void* work, hipStream_t st) {
    const ChunkPlan pl = chunk_plan(n, rows, max_len);
    const ChunkWork w = chunk_work(pl);
    uint8_t* base = static_cast<uint8_t*>(work);
    ChunkBlock* blocks = reinterpret_cast<ChunkBlock*>(base + w.blocks);
    int* head = reinterpret_cast<int*>(base + w.head);
    const ChunkArgs a{q, gate, out16, lse, blocks, head, reinterpret_cast<float*>(base + w.o),
                      reinterpret_cast<float4*>(base + w.ml), pl.slices, pl.rows};
    hipLaunchKernelGGL(k_ch_plan, dim3(1), dim3(CH_PT), 0, st, p, seqs, off, n, rows, max_len, pl.blocks, blocks, head);
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
    if (pl.slices > 1) {
        const dim3 jg(pl.slices - 1, NKV, (pl.rows + CH_JR - 1) / CH_JR);
        if (lse) hipLaunchKernelGGL(k_ch_join<true>, jg, dim3(256), 0, st, a);
        else hipLaunchKernelGGL(k_ch_join<false>, jg, dim3(256), 0, st, a);
    }
    return hipGetLastError();
}

}  // namespace qwa
