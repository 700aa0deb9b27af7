// Decode attention of a batch of sequences over a paged cache, the shared prefix read once (gfx950).
//
// For row r = (token, head) with q_r, and its keys K_j, V_j:  out = sum_j exp(s_j - m) V_j / sum_j exp(s_j - m) *
// sigmoid(gate), s_j = q_r . K_j / 16.  The sum splits over any partition of the keys into partial states (m, l, O), so the
// positions that all sequences share are worked on for the rows of all sequences together, in ranges of fixed length, those
// of its own for each sequence by itself, in equal slices of all sequences' positions (batch_plan.hpp), and k_bt_combine joins a
// row's states in a fixed order.
//  * Register workgroups (k_bt_own, and k_bt_shared for the shared positions of few rows) have one KV head and up to
//    BT_MAXRT 16-row tiles (row 6 * token + head of that KV head); their waves take the tiles of the key range in turn, each
//    with its own running maximum, sum and O, and merge at the end through LDS.
//  * Tile workgroups (k_bt_tiles, the shared positions of more rows) have BT_TROWS rows, 16 a wave: each tile is dequantized
//    once into LDS, by way of registers, and every wave multiplies its rows with it.
//  * Pages are multiples of 16 positions and tiles start at multiples of 16, so each 16 keys lie in one page.  A wave looks
//    the pages of its next 64 tiles up at once, a lane a tile.
//  * S^T = K Q^T and O^T += V^T P^T on fp16 MFMA with fp32 accumulation.  K enters as its exact codes, 32 dims (a block of the
//    cache) an MFMA, whose fp32 product is multiplied by the key's block scale, and Q / 16 as the sum of two fp16 parts: scores
//    are exact up to fp32 accumulation, as the one-sequence decode's are.  (With Q / 16 and d * code rounded to fp16, keys eight
//    times as large as the others moved an output by 4e-3 to 6e-3.)  In a register workgroup a lane loads 64 dims of one key and
//    16 dims of the keys whose probabilities it holds straight into registers and converts there; the next tile's K loads go
//    out when the scores are done, its V loads when P V is.
// A batch of one call has the same bits again; another batch, or another cut, sums a row's states in another order.
// Roundings below 32 bits: the dequantized V (d * code) and the probabilities are fp16 (half a step: 2^-11 of the value, random
// in sign, as in the prefill: P V then has one MFMA per 32 keys and 16 dims; for the probabilities' range see BT_RAISE), a tile
// workgroup's O / l is 16-bit fixed point (half a step: 2^-16 of the row's largest, attn_tiles.hpp), the output is fp16.
#include <type_traits>

#include "batch_plan.hpp"
#include "launch.hpp"
#include "paged_walk.hpp"

namespace qwa {

constexpr int BT_KD = 1;  // K steps read ahead of their MFMAs
constexpr int BT_VD = 3;  // V fragments in flight
size_t batch_work_bytes(int n, int nq, int n_shared, int max_len) {
    return batch_work(batch_plan(n, nq, n_shared, max_len), n, nq).bytes;
}

struct BatchArgs {
    const float* q;
    const int* seqs;
    PfPartO* tile_o;    // partial states (BatchWork): of the tile workgroups [range][row][256],
    PfPartMl* tile_ml;  // [range][row]
    float* part_o;      // of the register workgroups over the shared positions [range][row][256],
    float2* part_ml;    // [range][row]
    float* own_o;       // and over the own positions [KV head][segment][query row][256],
    float2* own_ml;     // [KV head][segment][query row]
    int* begin;         // first step of each batch row's own positions, and their total [n + 1]
    int n, nq, n_shared, max_len, wgs;
};

// positions of batch row b, 0 for an unknown sequence.  A longer sequence counts as one of max_len positions, for its queries'
// limits as for the key ranges.
__device__ __forceinline__ int bt_seq(const BatchArgs& a, int b) { return a.seqs ? a.seqs[b] : b; }
__device__ __forceinline__ int bt_len(const BatchArgs& a, const qwa_kv_pages& p, int b) {
    const int s = bt_seq(a, b);
    return s >= 0 && s < p.n_seq ? min(max(p.len[s], 0), a.max_len) : 0;
}
// the same of rows b, b + step, ..., 0 past the batch; N loads on their way at once
template <int N>
__device__ __forceinline__ void bt_lens(const BatchArgs& a, const qwa_kv_pages& p, int b, int step, int* len) {
    int s[N], m[N];
#pragma unroll
    for (int j = 0; j < N; j++) s[j] = bt_seq(a, min(b + step * j, a.n - 1));
#pragma unroll
    for (int j = 0; j < N; j++) m[j] = p.len[min(max(s[j], 0), p.n_seq - 1)];
#pragma unroll
    for (int j = 0; j < N; j++) len[j] = b + step * j < a.n && s[j] >= 0 && s[j] < p.n_seq ? min(max(m[j], 0), a.max_len) : 0;
}
constexpr int BT_LENS = 4;

// the longest batch row, the first of those (wave-uniform)
__device__ __forceinline__ int bt_longest(const BatchArgs& a, const qwa_kv_pages& p, int lane) {
    int m = -1, b = 0;
    for (int j0 = lane; j0 < a.n; j0 += 64 * BT_LENS) {
        int x[BT_LENS];
        bt_lens<BT_LENS>(a, p, j0, 64, x);
#pragma unroll
        for (int k = 0; k < BT_LENS; k++)
            if (x[k] > m && j0 + 64 * k < a.n) m = x[k], b = j0 + 64 * k;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int om = __shfl_xor(m, o, 64), ob = __shfl_xor(b, o, 64);
        if (om > m || (om == m && ob < b)) m = om, b = ob;
    }
    return __builtin_amdgcn_readfirstlane(b);
}

// the rows of a batch, for bt_walk; the state of a row goes to place rstep * token + head of po, pml
struct BatchSegment : BtRange {
    float* po;
    float2* pml;
    int rstep;
};
struct BatchRows {
    static constexpr int WAVES = BT_WAVES;
    static constexpr bool SUM = false;
    using SEGMENT = BatchSegment;
    const BatchArgs& a;
    const qwa_kv_pages& p;
    __device__ __forceinline__ int seen(const SEGMENT&, int tok) const {
        return bt_len(a, p, tok / a.nq) - a.nq + tok % a.nq + 1;
    }
    __device__ __forceinline__ const float* q(const SEGMENT&, int tok) const { return a.q + (size_t)tok * NH * HD; }
    __device__ __forceinline__ size_t place(const SEGMENT& s, int r) const { return (size_t)s.rstep * (r / GRP) + r % GRP; }
    __device__ __forceinline__ void sums(const SEGMENT& s, size_t place, float m, float l, float) const {
        s.pml[place] = make_float2(m, l);
    }
    __device__ __forceinline__ float* o(const SEGMENT& s, size_t place) const { return s.po + place * HD; }
};
template <int KVT, int RT>
using BatchLds = BtLds<KVT, RT, BT_WAVES, false>;

// the shared positions, for up to BT_FEW rows of a KV head: workgroup = (key range, KV head)
template <int KVT, int RT>
__global__ void __launch_bounds__(64 * BT_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
k_bt_shared(BatchArgs a, qwa_kv_layer kv, qwa_kv_pages p, int len) {
    __shared__ BatchLds<KVT, RT> lds;
    const int g = blockIdx.x % NKV, sp = blockIdx.x / NKV;
    const int b = bt_longest(a, p, threadIdx.x & 63);
    const int k1 = min(min((sp + 1) * len, a.n_shared), bt_len(a, p, b));
    const int seq = bt_seq(a, b);
    const int* table = p.table + (seq >= 0 && seq < p.n_seq ? (size_t)seq * p.ld : 0);
    const size_t rec = (size_t)sp * a.n * a.nq * NH + g * GRP;
    bt_walk<KVT, RT>(lds, BatchRows{a, p}, kv, p, g,
                     {{table, 0, a.n * a.nq * GRP, sp * len, k1, 0}, a.part_o + rec * HD, a.part_ml + rec, NH},
                     [](BatchSegment&) { return false; });
}

// steps of batch row b's own positions (they begin at the multiple of 16 at or before n_shared)
__device__ __forceinline__ int bt_steps_of(const BatchArgs& a, int m) {
    return m > a.n_shared ? (m - (a.n_shared & ~15) + BT_STEP - 1) / BT_STEP : 0;
}

// the own positions: workgroup = (slice of the steps, KV head, row group), one segment per sequence that the slice meets.
// Equal slices, since a cut by sequences leaves the chip to the longest one (24 of up to 16384 positions: 108 instead of 89 us,
// in an early form).  About 6 us of latency (finding the slice, page numbers, first bytes, joining the waves) around a stream of the
// cache's bytes: 24 sequences of 267 000 Q4_0 positions together 71 us (4.3 TB/s; VALU instructions, most of them unpacking,
// take 56% of the issue cycles), of 131 000 Q8_0 ones 60 us (4.7 TB/s), F16 99 us (5.4 TB/s, where a large copy reads and writes
// 5.15).  The next segment's first tile is sent before this one's waves are joined (2 to 3 us of 65).  Not faster: a second tile
// on its way (registers for it are there), three waves a SIMD (spills).  Of several row tiles (more than two queries) a tile
// has 16 keys, since 32 spill: 8 x 8 queries over 12000 own Q4_0 positions 63 us.  <F16, 2> keeps 15 registers in scratch, none of
// them in the loop over tiles.
template <int KVT, int RT>
__global__ void __launch_bounds__(64 * BT_WAVES) __attribute__((amdgpu_waves_per_eu(2)))
k_bt_own(BatchArgs a, qwa_kv_layer kv, qwa_kv_pages p, int groups) {
    __shared__ BatchLds<KVT, RT> lds;
    // the groups of one (slice, head) read the same keys: workgroups 8 apart, which one XCD runs
    const int u = blockIdx.x / (8 * groups) * 8 + blockIdx.x % 8, grp = blockIdx.x / 8 % groups;
    const int g = u % NKV, w = u / NKV, lane = threadIdx.x & 63;
    if (w >= a.wgs) return;
    // where the batch rows begin: every wave sums the steps of n / 64 rows a lane
    const int per = (a.n + 63) / 64;
    auto scan = [&](int x) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(x, o, 64);
            if (lane >= o) x += y;
        }
        return x;
    };
    int mine = 0;
    for (int j0 = 0; j0 < per; j0 += BT_LENS) {
        int m[BT_LENS];
        bt_lens<BT_LENS>(a, p, lane * per + j0, 1, m);
#pragma unroll
        for (int k = 0; k < BT_LENS; k++) mine += j0 + k < per ? bt_steps_of(a, m[k]) : 0;
    }
    const int upto = scan(mine);
    const int total = __builtin_amdgcn_readlane(upto, 63);
    if (blockIdx.x == 0 && threadIdx.x < 64) {
        int s = upto - mine;
        for (int j0 = 0; j0 < per; j0 += BT_LENS) {
            int m[BT_LENS];
            bt_lens<BT_LENS>(a, p, lane * per + j0, 1, m);
#pragma unroll
            for (int k = 0; k < BT_LENS; k++)
                if (j0 + k < per && lane * per + j0 + k < a.n) {
                    a.begin[lane * per + j0 + k] = s;
                    s += bt_steps_of(a, m[k]);
                }
        }
        if (lane == 0) a.begin[a.n] = total;
    }
    const int slices = min(a.wgs, total);  // (none is empty)
    if (w >= slices) return;
    // (BT_FILL slices of QWA_PAGES_MAXN * MAX_POS / BT_STEP steps: the products fit 32 bits, whose divisions are much shorter)
    static_assert((long long)BT_FILL * QWA_PAGES_MAXN * (MAX_POS / BT_STEP) < 1LL << 32, "32-bit slices");
    int s = (int)((uint32_t)w * (uint32_t)total / (uint32_t)slices);
    const int end = (int)((uint32_t)(w + 1) * (uint32_t)total / (uint32_t)slices);
    // the batch row that holds step s: the lane whose rows do, then one of those, a lane each
    const int at = __builtin_ctzll(__ballot(upto > s));
    int b = at, first = __builtin_amdgcn_readlane(upto - mine, at), m = __builtin_amdgcn_readlane(mine, at);
    if (per > 1) {
        int x;
        bt_lens<1>(a, p, at * per + lane, 1, &x);
        x = lane < per ? bt_steps_of(a, x) : 0;
        const int within = scan(x), row = __builtin_ctzll(__ballot(first + within > s));
        b = at * per + row;
        first += __builtin_amdgcn_readlane(within - x, row);
        m = __builtin_amdgcn_readlane(x, row);
    }
    // the lengths and sequences of the 64 rows from b on, a lane each (read a segment at a time they were a round trip each)
    int row0 = b, lens, seqs;
    auto look = [&]() {
        row0 = b;
        bt_lens<1>(a, p, b + lane, 1, &lens);
        seqs = bt_seq(a, min(b + lane, a.n - 1));
    };
    look();
    const int base = a.n_shared & ~15;
    int stop = s;
    // the segment of batch row b, from step s on
    auto segment = [&]() {
        stop = min(end, first + m);
        const int k0 = base + (s - first) * BT_STEP;
        const int k1 = min(base + (stop - first) * BT_STEP, __builtin_amdgcn_readlane(lens, b - row0));
        const size_t rec = ((size_t)g * (a.wgs + a.n) + w + b) * a.nq * GRP;
        // (row r = 6 * token + head has place r - 6 nq b of the segment)
        const ptrdiff_t place = (ptrdiff_t)rec - (ptrdiff_t)b * a.nq * GRP;
        return BatchSegment{{p.table + (size_t)__builtin_amdgcn_readlane(seqs, b - row0) * p.ld, b * a.nq * GRP + grp * 16 * RT,
                         (b + 1) * a.nq * GRP, k0, k1, a.n_shared}, a.own_o + place * HD, a.own_ml + place, GRP};
    };
    bt_walk<KVT, RT>(lds, BatchRows{a, p}, kv, p, g, segment(), [&](BatchSegment& seg) {
        s = stop;
        if (s >= end) return false;
        do {
            first += m;
            if (++b - row0 >= 64) look();
            m = bt_steps_of(a, __builtin_amdgcn_readlane(lens, b - row0));
        } while (m == 0);
        seg = segment();
        return true;
    });
}

// The shared positions for BT_TROWS rows: workgroup = (row block, tile range, KV head).  The 8 waves have 16 rows each, two a
// SIMD, of which one converts V at the start of an iteration and the other K at its end, so the MFMAs of one run while the
// other converts, takes exponentials or waits for LDS.  128 sequences over 32768 positions: Q4_0 209 us, 0.74 PFLOP/s with the
// second part of Q (large products of the library reach 1.17), Q8_0 218, F16 202; 2.0 us a tile.  No unit bounds it: of a
// SIMD's cycles 45% issue VALU instructions and 30% are MFMAs, LDS is busy for 37% and 5% of conflicts.  Two waves do not
// cover each other's waits, and three a SIMD have 168 registers each, of which O and both parts of Q leave 40.  (12 waves with
// the low parts of Q in LDS spill 18 to 89 of them; whole call, 12 / 8 waves: Q4_0 240 to 256 / 245 us, Q8_0 256 to 265 / 229, F16
// 226 to 239 / 215, 32 sequences over 8192 Q8_0 58 / 52.5.  Block scales by lane broadcasts instead of from LDS: 12 us more.
// K and V fragments read further ahead: no difference.)
template <int KVT>
__global__ void __launch_bounds__(64 * BT_TWAVES) __attribute__((amdgpu_waves_per_eu(BT_TWAVES / 4, BT_TWAVES / 4)))
k_bt_tiles(BatchArgs a, qwa_kv_layer kv, qwa_kv_pages p, int blocks, int ns) {
    constexpr int XCH = 16 * 64 * 8;  // bytes of a wave's exchange of its rows' state
    __shared__ __attribute__((aligned(16))) union {
        struct {
            _Float16 k[2][PF_TILE * HD];
            _Float16 vt[2][PF_TILE * HD];
            uint16_t scales[2][KVT == QWA_KV_F16 ? 8 : PF_TILE * 8];  // of K
            BtOdd odd[2];
        } tile;
        uint2 xch[BT_TWAVES][XCH / 8];
    } lds;
    static_assert(sizeof(lds.xch) <= sizeof(lds.tile.k) + sizeof(lds.tile.vt), "what lies behind the tiles is not exchanged");
    auto& s_k = lds.tile.k;
    auto& s_vt = lds.tile.vt;
    const int t = threadIdx.x, lane = t & 63, i16 = lane & 15, lg = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // workgroups 8 apart run on one XCD: those of a (KV head, range) pair read the same tiles
    int pair = blockIdx.x / blocks, blk = blockIdx.x % blocks;
    if (NKV * ns % 8 == 0) {
        pair = NKV * ns / 8 * (blockIdx.x & 7) + (blockIdx.x >> 3) / blocks;
        blk = (blockIdx.x >> 3) % blocks;
    }
    const int g = pair % NKV, sp = pair / NKV;
    const int longest = bt_longest(a, p, lane);
    const int end = min(a.n_shared, bt_len(a, p, longest));
    const int seq = bt_seq(a, longest);
    const int* __restrict__ table = p.table + (seq >= 0 && seq < p.n_seq ? (size_t)seq * p.ld : 0);
    const int all = (a.n_shared + PF_TILE - 1) / PF_TILE;
    const int tb = sp * all / ns, te = (sp + 1) * all / ns;
    const int nt = min(te, (end + PF_TILE - 1) / PF_TILE) - tb;  // (a batch shorter than its shared part: fewer, or none)
    const int nrows = a.n * a.nq * GRP, wrow0 = blk * BT_TROWS + 16 * wave;
    const size_t head = (size_t)g * kv.capacity;

    // The pool positions of the tiles' halves, 64 tiles ahead: lane l has those of tile l.  dead: which halves of tiles i,
    // i + 1 have none, two bits a tile.
    int ahead[2], tile = 0;
    uint32_t dead = 0;
    auto place = [&](int* at) {
        if ((tile & 63) == 0)
#pragma unroll
            for (int h = 0; h < 2; h++) ahead[h] = bt_place(p, table, (tb + tile + lane) * PF_TILE + 16 * h, end);
#pragma unroll
        for (int h = 0; h < 2; h++) at[h] = __builtin_amdgcn_readlane(ahead[h], tile & 63);
        tile++;
    };
    const uint8_t* const kh = kv.k + head * value_bytes(KVT);
    const uint8_t* const vh = kv.v + head * value_bytes(KVT);
    const uint16_t* const ksh = KVT == QWA_KV_F16 ? nullptr : kv.ks + head * 8;
    const uint16_t* const vsh = KVT == QWA_KV_F16 ? nullptr : kv.vs + head * 8;

    constexpr bool SC = KVT != QWA_KV_F16;
    h8 qb[2][8];  // hi and lo part of Q / 16
    f4 o[16];
    float m = -INFINITY, l = 0.0f;
    const int r = wrow0 + i16, tok = r / GRP;
    const bool valid = r < nrows;
    const int vis = valid ? min(bt_len(a, p, tok / a.nq) - a.nq + tok % a.nq + 1, end) : 0;
    int vmin = valid ? vis : 0x7fffffff;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) vmin = min(vmin, __shfl_xor(vmin, o, 64));
    vmin = __builtin_amdgcn_readfirstlane(vmin);
    // ROLE 0: a wave that converts V, 1: K.  (In one loop for both, the registers that the roles share make a wave wait for its
    // loads as soon as they are sent.)
    auto walk = [&](auto role) __attribute__((always_inline)) {
        constexpr int ROLE = decltype(role)::value;
        BtRaw<KVT> raw;
        // looks up tile i, the next one, and sends its loads
        auto load = [&](int i) {
            int at[2];
            place(at);
            const int left = end - (tb + i) * PF_TILE;
            const int rows[2] = {at[0] < 0 ? 16 : min(left, 16), at[1] < 0 ? 16 : min(left - 16, 16)};
            const uint32_t bits = (uint32_t)((at[0] < 0) | (at[1] < 0) << 1);
            if constexpr (ROLE == 0) bt_load_v<KVT>(raw, vh, vsh, at, rows, t);
            else bt_load_k<KVT>(raw, kh, ksh, wave < 6 ? at[0] : at[1], wave < 6 ? rows[0] : rows[1], t);
            return bits;
        };
        auto store = [&](int i, uint32_t bits) {
            const int b = i & 1;
            if constexpr (ROLE == 0) bt_store_v<KVT>(raw, s_vt[b], lds.tile.odd[b], t, bits, i);
            else bt_store_k<KVT>(raw, s_k[b], lds.tile.scales[b], t);
        };
        if (nt > 0) dead = load(0);
        if (t < 8) lds.tile.odd[t >> 2].tile[t & 3] = -1;  // (behind the part of LDS that the exchange uses)

        // Q / 16 as the B operand, by way of the wave's part of the exchange, first the hi parts, then the lo parts: a row is
        // read as one kilobyte (fragment by fragment, 16 rows at once, the loads took 7 us), its fp16 pieces go to unit (s, lg,
        // row ^ (4 s + lg) % 16) and come back as the lane's fragments s
        {
            float4 x[16];
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const int rj = min(wrow0 + j, nrows - 1);
                x[j] = *reinterpret_cast<const float4*>(a.q + ((size_t)(rj / GRP) * NH + g * GRP + rj % GRP) * HD + 4 * lane);
            }
            uint8_t* const area = reinterpret_cast<uint8_t*>(lds.xch[wave]);
            const int c = lane >> 1, half = lane & 1;  // piece c = 4 s + lg, dims 4 half .. 4 half + 3 of it
#pragma unroll
            for (int part = 0; part < 2; part++) {
                auto piece = [&](float v, float f) { return part ? q_lo(v * f) : q_hi(v * f); };
#pragma unroll
                for (int j = 0; j < 16; j++) {
                    const float f = wrow0 + j < nrows ? 0.0625f : 0.0f;
                    uint32_t w0 = h2_bits(h2{piece(x[j].x, f), piece(x[j].y, f)});
                    uint32_t w1 = h2_bits(h2{piece(x[j].z, f), piece(x[j].w, f)});
                    if constexpr (KVT == QWA_KV_Q4_0) {
                        // the operand's order [0, 4, 1, 5, 2, 6, 3, 7]: the even lane makes the first two words, the odd one
                        // the rest
                        const uint32_t mine = half ? w1 : w0;
                        const uint32_t other = __builtin_amdgcn_update_dpp(0, half ? w0 : w1, 0xB1, 0xF, 0xF, true);
                        const uint32_t lo = half ? other : mine, hi = half ? mine : other;  // dims k, k + 1 and k + 4, k + 5
                        w0 = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
                        w1 = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
                    }
                    *reinterpret_cast<uint2*>(area + 16 * (16 * c + (j ^ (c & 15))) + 8 * half) = make_uint2(w0, w1);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the area is the wave's own)
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int s = 0; s < 8; s++)
                    qb[part][s] = *reinterpret_cast<const h8*>(area + 16 * (16 * (4 * s + lg) + (i16 ^ ((4 * s + lg) & 15))));
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
        }
        __syncthreads();  // the fragments are in registers; the tiles lie in the same LDS

#pragma unroll
        for (int dt = 0; dt < 16; dt++) o[dt] = f4{0.0f, 0.0f, 0.0f, 0.0f};

        if (nt > 0) {
            // tile 0 converted, tile 1's bytes on their way
            store(0, dead);
            if (nt > 1) dead |= load(1) << 2;
            __syncthreads();
            const bool rows_here = wrow0 < nrows;
            // tile i + 1 into the other buffer (free since the last barrier), then tile i + 2's loads
            auto convert = [&](int i) {
                if (i + 1 < nt) store(i + 1, (dead >> 2) & 3);
                if (i + 2 < nt) dead |= load(i + 2) << 4;
            };
            for (int i = 0; i < nt; i++) {
                const int k0 = (tb + i) * PF_TILE;
                const _Float16* Ks = s_k[i & 1];
                const _Float16* Vt = s_vt[i & 1];
                const _Float16* Sc = reinterpret_cast<const _Float16*>(lds.tile.scales[i & 1]);
                if constexpr (ROLE == 0) convert(i);
                if (rows_here) {
                    // S^T = K Q^T: lane (row i16) gets keys k0 + 16 kt + 4 lg + j; the K fragments of a step are read while
                    // the step before multiplies, whose product is scaled while the next one is on its way
                    f4 sc[2] = {}, T[2][2];
                    h8 ks[2];  // scales of blocks s - 1 and s, s even, or s and s + 1
                    auto scale = [&](int s, int kt) {
#pragma unroll
                        for (int j = 0; j < 4; j++) sc[kt][j] = fmaf((float)ks[kt][4 * (s & 1) + j], T[s & 1][kt][j], sc[kt][j]);
                    };
                    auto kfrag = [&](int s, int kt) {
                        return lds_h8(Ks + 8 * (32 * (4 * s + lg) + 16 * kt + (i16 ^ (2 * s))));
                    };
                    h8 kf[BT_KD + 1][2];
#pragma unroll
                    for (int s = 0; s < BT_KD; s++)
#pragma unroll
                        for (int kt = 0; kt < 2; kt++) kf[s][kt] = kfrag(s, kt);
#pragma unroll
                    for (int s = 0; s < 8; s++) {
                        if (s + BT_KD < 8)
#pragma unroll
                            for (int kt = 0; kt < 2; kt++) kf[(s + BT_KD) % (BT_KD + 1)][kt] = kfrag(s + BT_KD, kt);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int part = 1; part >= 0; part--)
#pragma unroll
                            for (int kt = 0; kt < 2; kt++) {
                                const h8 k8 = kf[s % (BT_KD + 1)][kt];
                                if constexpr (SC) {
                                    const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                                    T[s & 1][kt] = mfma16(k8, qb[part][s], part ? zero : T[s & 1][kt]);
                                } else {
                                    sc[kt] = mfma16(k8, qb[part][s], sc[kt]);
                                }
                            }
                        if constexpr (SC) {
                            if (s > 0) {
                                scale(s - 1, 0);
                                scale(s - 1, 1);
                            }
                            if (s % 2 == 0)
#pragma unroll
                                for (int kt = 0; kt < 2; kt++) ks[kt] = lds_h8(Sc + 8 * (16 * kt + 2 * s + lg));
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    if constexpr (SC) {
                        scale(7, 0);
                        scale(7, 1);
                    } else {
                        mfma_settle(sc[0], sc[1]);
                    }
                    if (k0 + PF_TILE > vmin || (dead & 3) != 0) {
#pragma unroll
                        for (int kt = 0; kt < 2; kt++)
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                sc[kt][j] = k0 + 16 * kt + 4 * lg + j < vis && !((dead >> kt) & 1) ? sc[kt][j] : -INFINITY;
                    }
                    float mx = max3f(max3f(-INFINITY, sc[0][0], sc[0][1]), sc[0][2], sc[0][3]);
                    mx = rows_max(max3f(max3f(mx, sc[1][0], sc[1][1]), sc[1][2], sc[1][3]));
                    const float mx2 = mx * PF_LOG2E, mn = mx2 > m + BT_HEAD ? mx2 - BT_RAISE : m;
                    const float cr = mn == m ? 1.0f : fast_exp2(m - mn);
                    const float ref = mn == -INFINITY ? 0.0f : mn;
                    m = mn;
                    // the V fragments' reads begin while the exponentials are taken
                    const _Float16* vrow = Vt + 8 * (256 * lg + i16);
                    h8 vf[BT_VD];
#pragma unroll
                    for (int dt = 0; dt < BT_VD - 1; dt++) vf[dt] = lds_h8(vrow + 8 * 16 * dt);
                    h8 pb;
#pragma unroll
                    for (int j = 0; j < 8; j++) pb[j] = (_Float16)fast_exp2(fmaf(sc[j >> 2][j & 3], PF_LOG2E, -ref));
                    // the sum of the rounded probabilities, the weights that P V applies
                    const h2 one2 = {(_Float16)1.0f, (_Float16)1.0f};
                    float rs = 0.0f;
#pragma unroll
                    for (int j = 0; j < 8; j += 2) rs = __builtin_amdgcn_fdot2(h2{pb[j], pb[j + 1]}, one2, rs, false);
                    l = l * cr + rs;
                    if (__any(cr != 1.0f)) {
#pragma unroll
                        for (int dt = 0; dt < 16; dt++) o[dt] *= cr;
                    }
                    // O^T += V^T P^T
#pragma unroll
                    for (int dt = 0; dt < 16; dt++) {
                        if (dt + BT_VD - 1 < 16) vf[(dt + BT_VD - 1) % BT_VD] = lds_h8(vrow + 8 * 16 * (dt + BT_VD - 1));
                        o[dt] = mfma16(vf[dt % BT_VD], pb, o[dt]);
                    }
                    // a dim is NaN in the rows that see a value of it that is not finite
                    const int4 w = *reinterpret_cast<const int4*>(lds.tile.odd[i & 1].tile);
                    if (__builtin_amdgcn_readfirstlane(w.x == i || w.y == i || w.z == i || w.w == i)) {
                        const int of[4] = {w.x, w.y, w.z, w.w};
                        uint32_t seen[2] = {0, 0};
#pragma unroll
                        for (int k = 0; k < PF_TILE; k++) {
                            const int cb = k / 4 % 4, h = k / 16;
                            if (of[cb] == i && k0 + k < vis && !((dead >> h) & 1))
                                seen[cb / 2] |= 1u << (8 * (2 * (cb & 1) + h) + k % 4);
                        }
#pragma unroll
                        for (int dt = 0; dt < 16; dt++) {
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const int dim = 8 * (16 * (dt & 1) + 4 * lg + j) + (dt >> 1);
                                const uint2 keys = *reinterpret_cast<const uint2*>(&lds.tile.odd[i & 1].keys[8 * dim]);
                                o[dt][j] = ((keys.x & seen[0]) | (keys.y & seen[1])) != 0 ? NAN : o[dt][j];
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
                if constexpr (ROLE != 0) convert(i);
                dead >>= 2;
                __syncthreads();
            }
        }
    };
    if (wave < 4) walk(std::integral_constant<int, 0>{});
    else walk(std::integral_constant<int, 1>{});

    // partial state: o[2 k + e][j] is dim 8 x + k of row i16, x = 16 e + 4 lg + j; through LDS, so that a store instruction
    // writes two whole 512-byte rows
    uint2* const xch = lds.xch[wave];
    __syncthreads();
    const float lt = rows_sum(l);
    const float il = lt == 0.0f ? 0.0f : 1.0f / lt;  // (a row that saw nothing: l = 0 and O = 0)
    float amax = 0.0f;  // (maximum, unlike fmaxf, keeps a NaN)
#pragma unroll
    for (int dt = 0; dt < 16; dt++)
#pragma unroll
        for (int j = 0; j < 4; j++) amax = __builtin_elementwise_maximum(amax, fabsf(o[dt][j]));
    amax = lt == 0.0f ? 0.0f : rows_max(amax < INFINITY ? amax : INFINITY) * il;
    const float f = amax > 1e-30f ? il / amax : 0.0f;
    const size_t range = (size_t)sp * a.n * a.nq * NH + g * GRP;
    // (a row whose O is not finite has no fixed-point form: its scale makes every value NaN)
    const float scale = amax < INFINITY ? (f != 0.0f ? amax * (1.0f / 32767.0f) : 0.0f) : NAN;
    if (valid && lg == 0) a.tile_ml[range + (size_t)tok * NH + r % GRP] = make_float4(m, lt, scale, 0.0f);
    auto pack = [&](float x, float y) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_i16(x * f, y * f));
    };
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int e = q & 1, k = 4 * (q >> 1);  // dims 8 x + k .. + 3: 8-byte unit 2 x + k / 4
            xch[64 * i16 + ((2 * (16 * e + 4 * lg + j) + k / 4) ^ (4 * i16))] =
                make_uint2(pack(o[2 * k + e][j], o[2 * k + 2 + e][j]), pack(o[2 * k + 4 + e][j], o[2 * k + 6 + e][j]));
        }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (the area is the wave's own)
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const int xr = 2 * k + (lane >> 5), ro = wrow0 + xr;
        const uint4 w = *reinterpret_cast<const uint4*>(&xch[64 * xr + ((2 * (lane & 31)) ^ (4 * xr))]);
        if (ro < nrows)
            *reinterpret_cast<uint4*>(a.tile_o + (range + (size_t)(ro / GRP) * NH + ro % GRP) * (HD / 4) + 2 * (lane & 31)) = w;
    }
}

// Joins a row's partial states in a fixed order, gates, rounds: WPR waves per row (token * NH + head), 4 dims per lane.  The
// weights 2^(m - M) come one state a lane, 64 at a time; wave k of a row reads the states' rows k, k + WPR, ..., eight at
// a time.
// The states' bytes and a chain of dependent loads bound it: 768 rows of 32 fixed-point and 5 fp32 states 7.1 us (17 MB).
template <int WPR>
__global__ void __launch_bounds__(256) k_bt_combine(BatchArgs a, const float* __restrict__ gate, int nt, int ns_shared,
                                                    uint16_t* __restrict__ out16, qwa_act_q8 oq, int do_q) {
    __shared__ float4 s_o[WPR > 1 ? 4 : 1][64];
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), part = wave % WPR, lane = threadIdx.x & 63;
    const int row = blockIdx.x * (4 / WPR) + wave / WPR;
    const int nrows = a.n * a.nq * NH;
    if (row >= nrows) return;  // (all waves of a row, and with WPR = 4 of a workgroup)
    const int tok = row / NH, b = tok / a.nq, h = row % NH;
    const float4 gv = *reinterpret_cast<const float4*>(gate + (size_t)row * HD + 4 * lane);
    // the batch row's segments: those of the slices from its first step's to its last one's
    int segs = 0;
    size_t seg0 = 0;
    if (a.wgs > 0) {
        const uint32_t s0 = a.begin[b], s1 = a.begin[b + 1], total = a.begin[a.n];
        if (s1 > s0) {
            const uint32_t slices = min((uint32_t)a.wgs, total);
            const int w0 = (int)(((s0 + 1) * slices - 1) / total), w1 = (int)((s1 * slices - 1) / total);
            segs = w1 - w0 + 1;
            seg0 = ((size_t)(h / GRP) * (a.wgs + a.n) + w0 + b) * a.nq * GRP + (tok % a.nq) * GRP + h % GRP;
        }
    }
    float M = -INFINITY, L = 0.0f;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // adds `count` states: ml(s) their (m, l, factor of the stored values), x(s) the lane's four values
    constexpr int U = 8;
    auto add = [&](int count, auto ml_of, auto x_of) {
        for (int s0 = 0; s0 < count; s0 += 64) {
            const int most = min(64, count - s0);
            float4 x[U];
            // (with few states only those: a load of one again costs as much as the first; 57600 rows of 4 states 73 -> 54 us)
            if (most > 4 * WPR) {
#pragma unroll
                for (int u = 0; u < U; u++) x[u] = x_of(s0 + min(part + u * WPR, most - 1));
            } else {
#pragma unroll
                for (int u = 0; u < 4; u++)
                    if (part + u * WPR < most) x[u] = x_of(s0 + part + u * WPR);
            }
            const float4 ml = lane < most ? ml_of(s0 + lane) : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
            const float Mn = fmaxf(M, wave_max(ml.x));
            const float c = M == Mn ? 1.0f : fast_exp2(M - Mn);
            // a state that saw nothing weighs nothing; one of NaN scores (l is NaN) makes the row NaN
            const float f = ml.y == 0.0f ? 0.0f : fast_exp2(ml.x - Mn);
            M = Mn;
            L = fmaf(L, c, wave_sum(f * ml.y));
            acc.x *= c;
            acc.y *= c;
            acc.z *= c;
            acc.w *= c;
            const float wt = f * ml.z;
            for (int k = part; k < most; k += U * WPR) {
                float4 nx[U];
#pragma unroll
                for (int u = 0; u < U; u++)
                    if (k + U * WPR < most) nx[u] = x_of(s0 + min(k + (U + u) * WPR, most - 1));
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const float fu = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wt), min(k + u * WPR, 63)));
                    if (k + u * WPR < most) {
                        acc.x = fmaf(fu, x[u].x, acc.x);
                        acc.y = fmaf(fu, x[u].y, acc.y);
                        acc.z = fmaf(fu, x[u].z, acc.z);
                        acc.w = fmaf(fu, x[u].w, acc.w);
                    }
                    x[u] = nx[u];
                }
            }
        }
    };
    // tile states hold O / l in steps of their scale, register states O
    add(nt,
        [&](int s) {
            const float4 v = a.tile_ml[(size_t)s * nrows + row];
            return make_float4(v.x, v.y, v.z * v.y, 0.0f);
        },
        [&](int s) { return unpack16x4(a.tile_o[((size_t)s * nrows + row) * (HD / 4) + lane]); });
    add(ns_shared,
        [&](int s) {
            const float2 v = a.part_ml[(size_t)s * nrows + row];
            return make_float4(v.x, v.y, 1.0f, 0.0f);
        },
        [&](int s) { return *reinterpret_cast<const float4*>(a.part_o + ((size_t)s * nrows + row) * HD + 4 * lane); });
    add(segs,
        [&](int s) {
            const float2 v = a.own_ml[seg0 + (size_t)s * a.nq * GRP];
            return make_float4(v.x, v.y, 1.0f, 0.0f);
        },
        [&](int s) { return *reinterpret_cast<const float4*>(a.own_o + (seg0 + (size_t)s * a.nq * GRP) * HD + 4 * lane); });
    if constexpr (WPR > 1) {
        s_o[wave][lane] = acc;
        __syncthreads();
        if (part != 0) return;
#pragma unroll
        for (int k = 1; k < WPR; k++) {
            const float4 x = s_o[wave + k][lane];
            acc.x += x.x;
            acc.y += x.y;
            acc.z += x.z;
            acc.w += x.w;
        }
    }
    float v[4] = {acc.x / L * sigmoid(gv.x), acc.y / L * sigmoid(gv.y), acc.z / L * sigmoid(gv.z), acc.w / L * sigmoid(gv.w)};
    if (L == 0.0f) v[0] = v[1] = v[2] = v[3] = 0.0f;  // no key was seen
    *reinterpret_cast<uint2*>(out16 + (size_t)row * HD + 4 * lane) =
        make_uint2((uint32_t)f2h_bits(v[0]) | ((uint32_t)f2h_bits(v[1]) << 16),
                   (uint32_t)f2h_bits(v[2]) | ((uint32_t)f2h_bits(v[3]) << 16));
    if (do_q) {
        // ActQ8 of 32 values in 8 lanes: d = amax / 127, q = round-half-even(v / d), s = d * sum(q)
        auto max8 = [](float x) {
            x = fmaxf(x, row_move<0xB1>(x));
            x = fmaxf(x, row_move<0x4E>(x));
            return fmaxf(x, row_move<0x141>(x));
        };
        auto sum8 = [](float x) {
            x += row_move<0xB1>(x);
            x += row_move<0x4E>(x);
            return x + row_move<0x141>(x);
        };
        const float d = max8(fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])))) / 127.0f;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int qi = d > 0.0f ? (int)__builtin_rintf(v[j] / d) : 0;
            oq.q[(size_t)row * HD + 4 * lane + j] = (int8_t)qi;
            sum += (float)qi;
        }
        sum = sum8(sum);
        if ((lane & 7) == 0) {
            oq.d[(size_t)row * (HD / 32) + lane / 8] = d;
            oq.s[(size_t)row * (HD / 32) + lane / 8] = d * sum;
        }
    }
}

template <int KVT>
static void launch_ranges(const BatchArgs& a, const qwa_kv_layer& kv, const qwa_kv_pages& p, const BatchPlan& b,
                          hipStream_t st) {
    const dim3 block(64 * BT_WAVES);
#define QWA_BT(K, RT, GRID, ...) hipLaunchKernelGGL((K<KVT, RT>), dim3(GRID), block, 0, st, a, kv, p, __VA_ARGS__)
    if (b.nt > 0)
        hipLaunchKernelGGL(k_bt_tiles<KVT>, dim3(b.blocks * b.nt * NKV), dim3(64 * BT_TWAVES), 0, st, a, kv, p, b.blocks, b.nt);
    if (b.ns_shared > 0) {
        if (b.rt_shared == 1) QWA_BT(k_bt_shared, 1, b.ns_shared * NKV, b.len_shared);
        else QWA_BT(k_bt_shared, 2, b.ns_shared * NKV, b.len_shared);
    }
    if (b.wgs > 0) {
        const int grid = (b.wgs * NKV + 7) / 8 * 8 * b.groups;
        if (b.rt_own == 1) QWA_BT(k_bt_own, 1, grid, b.groups);
        else QWA_BT(k_bt_own, 2, grid, b.groups);
    }
#undef QWA_BT
}

hipError_t launch_decode_batch(const float* q, const float* gate, const qwa_kv_layer& kv, int kvt, const qwa_kv_pages& p,
                               const int* seqs, int n, int nq, int n_shared, int max_len, uint16_t* out16,
                               const qwa_act_q8* oq, void* work, hipStream_t st) {
    const BatchPlan b = batch_plan(n, nq, n_shared, max_len);
    const BatchWork w = batch_work(b, n, nq);
    uint8_t* base = static_cast<uint8_t*>(work);
    const BatchArgs a{q, seqs, reinterpret_cast<PfPartO*>(base + w.tile_o), reinterpret_cast<PfPartMl*>(base + w.tile_ml),
                      reinterpret_cast<float*>(base + w.o), reinterpret_cast<float2*>(base + w.ml),
                      reinterpret_cast<float*>(base + w.own_o), reinterpret_cast<float2*>(base + w.own_ml),
                      reinterpret_cast<int*>(base + w.begin), n, nq, n_shared, max_len, b.wgs};
    switch (kvt) {
        case QWA_KV_F16: launch_ranges<QWA_KV_F16>(a, kv, p, b, st); break;
        case QWA_KV_Q8_0: launch_ranges<QWA_KV_Q8_0>(a, kv, p, b, st); break;
        default: launch_ranges<QWA_KV_Q4_0>(a, kv, p, b, st); break;
    }
    const qwa_act_q8 act = oq ? *oq : qwa_act_q8{nullptr, nullptr, nullptr};
    // with many states a workgroup per row, else a wave (us, wave / workgroup: 768 rows of about 72 states 22.0 / 11.6, 840 of
    // 66 12.7 / 8.8, 48 of 97 14.0 / 7.4; 576 of 10 5.2 / 5.5, those of 128 sequences of 19 11.0 / 19.2, 9600 of 2 11.6 / 29.2)
    const int rows = n * nq * NH, states = b.nt + b.ns_shared + (b.wgs > 0 ? b.wgs / n + 1 : 0);
    if (states > 24)
        hipLaunchKernelGGL(k_bt_combine<4>, dim3(rows), dim3(256), 0, st, a, gate, b.nt, b.ns_shared, out16, act,
                           oq != nullptr ? 1 : 0);
    else
        hipLaunchKernelGGL(k_bt_combine<1>, dim3((rows + 3) / 4), dim3(256), 0, st, a, gate, b.nt, b.ns_shared, out16,
                           act, oq != nullptr ? 1 : 0);
    return hipGetLastError();
}

}  // namespace qwa
