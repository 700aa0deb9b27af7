// Attention of few rows over a paged cache, the keys straight into registers: what the batched decode and the short chunks of new
// tokens have in common.  The waves of a workgroup take the tiles of a key range in turn, each with its own running maximum, sum
// and O, and merge at the end through LDS.
#pragma once

#include "paged_tiles.hpp"

namespace qwa {

__device__ __forceinline__ f4 bt_mfma16k16(h4 a, h4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
}

// lane FROM of each row of 16 lanes, in all of them
template <int FROM>
__device__ __forceinline__ float row_lane(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + FROM, 0xF, 0xF, true));
}
// Scores of 16 keys from block S's products: a lane holds keys 4 lg + i, and lane 4 i + S / 2 of its row of 16 the scales of
// blocks S, S ^ 1 of key 4 lg + i (even block in `even`).
template <int S>
__device__ __forceinline__ void add_block(f4& score, const f4& product, float even, float odd) {
    const float d = S % 2 ? odd : even;
    score[0] = fmaf(row_lane<S / 2>(d), product[0], score[0]);
    score[1] = fmaf(row_lane<4 + S / 2>(d), product[1], score[1]);
    score[2] = fmaf(row_lane<8 + S / 2>(d), product[2], score[2]);
    score[3] = fmaf(row_lane<12 + S / 2>(d), product[3], score[3]);
    // (the sums stay where they are: put off past the last block, they kept all scales and products, and spilled)
    asm volatile("" : "+v"(score));
}
__device__ __forceinline__ void add_block(int s, f4& score, const f4& product, float even, float odd) {  // s: unrolled
    switch (s) {
        case 0: add_block<0>(score, product, even, odd); break;
        case 1: add_block<1>(score, product, even, odd); break;
        case 2: add_block<2>(score, product, even, odd); break;
        case 3: add_block<3>(score, product, even, odd); break;
        case 4: add_block<4>(score, product, even, odd); break;
        case 5: add_block<5>(score, product, even, odd); break;
        case 6: add_block<6>(score, product, even, odd); break;
        default: add_block<7>(score, product, even, odd); break;
    }
}
// lane rows 0, 1 of b for lane rows 2, 3 of a
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
    const auto x = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = x[0];
    b = x[1];
}
// lane rows 0, 2 of b for lane rows 1, 3 of a
__device__ __forceinline__ void swap_rows(uint32_t& a, uint32_t& b) {
    const auto x = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = x[0];
    b = x[1];
}

template <int KVT, int RT>
struct BtCfg {
    // 16-key groups of a tile, as two waves per SIMD leave registers for (raw bytes of 32 keys: F16 128 registers, Q8_0 66)
    static constexpr int KT = KVT == QWA_KV_F16 || RT > 1 ? 1 : 2;
};

template <int KVT, int RT, int WAVES, bool SUM>
struct BtLds {
    union {
        h8 q[RT][8][2][64];     // while the keys are walked: hi and lo part of Q / 16
        f4 o[WAVES][8][64];  // while the waves' states are joined, half of the output tiles at a time
    };
    float ml[WAVES][SUM ? 3 : 2][64];
};

// One key range of a workgroup: rows [row0, rows) of the KV head (row 6 * token + head of the group), keys [k0, k1) of the
// sequence whose table row is `table`, positions below lo excluded.
struct BtRange {
    const int* table;
    int row0, rows, k0, k1, lo;
};

// The segments of a workgroup of ROWS::WAVES waves, one after the other: `next` says whether there is another one, and which.  ROWS
// knows the rows of a segment (SEGMENT, a BtRange and what it likes to add): where Q has row r, how many positions the row sees,
// and what becomes of its state: `place` of the row, sums(place, m, l, sum of the unrounded probabilities, where ROWS::SUM), o(place).
template <int KVT, int RT, class ROWS, class NEXT>
__device__ __forceinline__ void bt_walk(BtLds<KVT, RT, ROWS::WAVES, ROWS::SUM>& lds, const ROWS& rows, const qwa_kv_layer& kv,
                                        const qwa_kv_pages& p, int g, typename ROWS::SEGMENT seg, NEXT next) {
    constexpr int WAVES = ROWS::WAVES, QS = 8 / WAVES;  // steps of Q, and pairs of output tiles in a round, that a wave has
    auto& s_o = lds.o;
    auto& s_ml = lds.ml;
    constexpr int KT = BtCfg<KVT, RT>::KT, VB = value_bytes(KVT), TILE = 16 * KT;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const int i16 = lane & 15, lg = lane >> 4;
    const uint8_t* const kh = kv.k + (size_t)g * kv.capacity * VB;
    const uint8_t* const vh = kv.v + (size_t)g * kv.capacity * VB;
    const uint16_t* const ksh = KVT == QWA_KV_F16 ? nullptr : kv.ks + (size_t)g * kv.capacity * 8;
    const uint16_t* const vsh = KVT == QWA_KV_F16 ? nullptr : kv.vs + (size_t)g * kv.capacity * 8;

    // The pool positions of the wave's tiles, 64 tiles ahead: lane l has those of tile l.  (Looked up a tile at a time they
    // were a memory round trip each, and a wait for all loads on their way.)
    constexpr int STRIDE = TILE * WAVES;
    int ahead[KT], tile, kb, k1;
    auto place = [&](int kb, int* at) {
        if ((tile & 63) == 0)
#pragma unroll
            for (int kt = 0; kt < KT; kt++) ahead[kt] = bt_place(p, seg.table, kb + STRIDE * lane + 16 * kt, k1);
#pragma unroll
        for (int kt = 0; kt < KT; kt++) at[kt] = __builtin_amdgcn_readlane(ahead[kt], tile & 63);
        tile++;
    };
    // Raw bytes of a tile.  K: 16-byte piece 4 i + lg of row i16 in words 4 i .. 4 i + 3, so that one load instruction takes
    // 64 consecutive bytes of 16 rows.  V: the lane's 16 dims of row 4 lg + j, F16 as two runs of 8 dims 128 apart (whole cache
    // lines).  Block scales: the 16 rows' 256 bytes, a dword a lane, handed out by lane permutes when they are used.
    // Each 16 keys are a buffer that ends with the range: rows past it, and groups without a place, read as zeros.  So the
    // loads need no branch, and the waits for K leave V's on their way and the other way round.
    constexpr bool SC = KVT != QWA_KV_F16;
    constexpr int KW = VB / 16, VW = VB / 64;  // words per lane of a K row and of a V row
    uint32_t kr[KT][KW], vr[4 * KT][VW], ksd[KT], vsd[KT];
    auto rows_of = [&](int at, int kb) { return at < 0 ? 0 : min(max(k1 - kb, 0), 16); };
    auto load_ks = [&](const int* at, int kb) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
            const size_t pos = (size_t)__builtin_amdgcn_readfirstlane(max(at[kt], 0));
            const int n = __builtin_amdgcn_readfirstlane(rows_of(at[kt], kb + 16 * kt));
            const auto r = bt_buffer(kh + pos * VB, n * VB);
#pragma unroll
            for (int i = 0; i < KW / 4; i++) {
                const uint4 x = bt_ld16(r, i16 * VB + 16 * lg + 64 * i);
                kr[kt][4 * i] = x.x; kr[kt][4 * i + 1] = x.y; kr[kt][4 * i + 2] = x.z; kr[kt][4 * i + 3] = x.w;
            }
            if constexpr (SC) ksd[kt] = __builtin_amdgcn_raw_buffer_load_b32(bt_buffer(ksh + pos * 8, n * 16), 4 * lane, 0, 0);
        }
    };
    auto load_vs = [&](const int* at, int kb) {
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
            const size_t pos = (size_t)__builtin_amdgcn_readfirstlane(max(at[kt], 0));
            const int n = __builtin_amdgcn_readfirstlane(rows_of(at[kt], kb + 16 * kt));
            const auto r = bt_buffer(vh + pos * VB, n * VB);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                uint32_t* const w = vr[4 * kt + j];
                if constexpr (VW == 2) {
                    const uint2 x = bt_ld8(r, 4 * lg * VB + 8 * i16 + j * VB);
                    w[0] = x.x; w[1] = x.y;
                } else {
#pragma unroll
                    for (int i = 0; i < VW / 4; i++) {
                        const uint4 x = bt_ld16(r, 4 * lg * VB + 16 * i16 + j * VB + 256 * i);
                        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
                    }
                }
            }
            if constexpr (SC) vsd[kt] = __builtin_amdgcn_raw_buffer_load_b32(bt_buffer(vsh + pos * 8, n * 16), 4 * lane, 0, 0);
        }
    };
    // half h (0 / 1) of lane `from`'s dword x, in both halves
    auto scale_of = [&](uint32_t x, int from, int h) {
        const uint32_t u = __builtin_amdgcn_ds_bpermute(4 * from, (int)x);
        return bits_h2(__builtin_amdgcn_perm(u, u, h ? 0x03020302u : 0x01000100u));
    };

    // rows of this lane: keys below vis are seen; Q / 16 as the B operand in the K operand's dim order (step s: block s, of which
    // the lane holds 8 dims from qd on), of which a wave makes QS
    const int qd = KVT == QWA_KV_Q8_0 ? 16 * (lg & 1) + 8 * (lg >> 1) : 8 * lg;
    int vis[RT], vmin, at[KT];
    float4 qx[RT][QS][2];
    // A segment's first loads: what is read of Q and the lengths is on its way while the pages are looked up.
    auto begin = [&]() {
        k1 = __builtin_amdgcn_readfirstlane(seg.k1);
        kb = __builtin_amdgcn_readfirstlane(seg.k0) + TILE * wave;
        vmin = k1;
        tile = 0;
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const int r = seg.row0 + 16 * rt + i16, tok = r / GRP;
            const bool valid = r < seg.rows;
            vis[rt] = valid ? min(rows.seen(seg, tok), k1) : 0;
            if (valid) vmin = min(vmin, vis[rt]);
            const float* qrow = rows.q(seg, valid ? tok : seg.row0 / GRP) + (g * GRP + r % GRP) * HD + qd;
#pragma unroll
            for (int i = 0; i < QS; i++) {
                const float* src = qrow + 32 * (QS * wave + i);
                qx[rt][i][0] = *reinterpret_cast<const float4*>(src);
                qx[rt][i][1] = *reinterpret_cast<const float4*>(src + 4);
            }
        }
        place(kb, at);
        load_ks(at, kb);
        load_vs(at, kb);
    };
    begin();
    while (true) {
        // (converted while the first tile is on its way)
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const bool valid = seg.row0 + 16 * rt + i16 < seg.rows;
#pragma unroll
            for (int i = 0; i < QS; i++) {
                const float4 x0 = qx[rt][i][0], x1 = qx[rt][i][1];
                const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
                h8 hi, lo;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float y = valid ? x[k_perm<KVT>(j)] * 0.0625f : 0.0f;
                    hi[j] = q_hi(y);
                    lo[j] = q_lo(y);
                }
                lds.q[rt][QS * wave + i][0][lane] = hi;
                lds.q[rt][QS * wave + i][1][lane] = lo;
            }
        }
        __syncthreads();
        // (uniform: the least over the 16 lanes that hold different rows)
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) vmin = min(vmin, __shfl_xor(vmin, o, 64));
        vmin = __builtin_amdgcn_readfirstlane(vmin);

        f4 o[RT][16];
        float m[RT], l[RT], lx[RT];
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            m[rt] = -INFINITY;
            l[rt] = lx[rt] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < 16; dt++) o[rt][dt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        }

        for (; kb < k1; kb += STRIDE) {
            const int nb = kb + STRIDE;
            int nat[KT];
            place(nb, nat);
            f4 S[RT][KT];
#pragma unroll
            for (int rt = 0; rt < RT; rt++)
#pragma unroll
                for (int kt = 0; kt < KT; kt++) S[rt][kt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            // The lanes' pieces become blocks, 8 dims a lane: Q4_0, where a lane has a whole block, by exchanging words and lane
            // rows (word k of lane row r <-> word r of lane row k), Q8_0, where two lanes have one, half of that.
            float even[KT], odd[KT];
            if constexpr (SC) {
#pragma unroll
                for (int kt = 0; kt < KT; kt++) {
#pragma unroll
                    for (int i = 0; i < KW; i += 4) {
                        uint32_t* const w = kr[kt] + i;
                        swap_halves(w[0], w[2]);
                        swap_halves(w[1], w[3]);
                        if constexpr (KVT == QWA_KV_Q4_0) {
                            swap_rows(w[0], w[1]);
                            swap_rows(w[2], w[3]);
                        }
                    }
                    // (dword l of the 16 rows' scales is in lane l: rows 4 lg .. 4 lg + 3 in this lane's row of 16)
                    even[kt] = h2f_bits((uint16_t)ksd[kt]);
                    odd[kt] = h2f_bits((uint16_t)(ksd[kt] >> 16));
                }
            }
            // products of blocks s and s - LAG, where the registers allow the latter
            constexpr int LAG = RT == 1 ? 1 : 0;
            f4 T[1 + LAG][RT][KT];
#pragma unroll
            for (int s = 0; s < 8; s++) {
                h8 ka[KT];
#pragma unroll
                for (int kt = 0; kt < KT; kt++) {
                    uint32_t w[4];
                    if constexpr (KVT == QWA_KV_F16) {
#pragma unroll
                        for (int i = 0; i < 4; i++) w[i] = kr[kt][4 * s + i];
                    } else if constexpr (KVT == QWA_KV_Q8_0) {
                        q8_word_int(kr[kt][2 * s], w);
                        q8_word_int(kr[kt][2 * s + 1], w + 2);
                    } else {
                        bt_q4_codes(kr[kt][s], w);
                    }
                    ka[kt] = make_h8(w[0], w[1], w[2], w[3]);
                }
#pragma unroll
                for (int part = 1; part >= 0; part--) {
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        const h8 b = lds.q[rt][s][part][lane];
#pragma unroll
                        for (int kt = 0; kt < KT; kt++) {
                            if constexpr (SC) {
                                const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                                T[s & LAG][rt][kt] = mfma16(ka[kt], b, part ? zero : T[s & LAG][rt][kt]);
                            } else {
                                S[rt][kt] = mfma16(ka[kt], b, S[rt][kt]);
                            }
                        }
                    }
                    if (RT > 1) __builtin_amdgcn_sched_barrier(0);  // (registers)
                }
                if constexpr (SC) {
                    if (s >= LAG)
#pragma unroll
                        for (int rt = 0; rt < RT; rt++)
#pragma unroll
                            for (int kt = 0; kt < KT; kt++)
                                add_block(s - LAG, S[rt][kt], T[(s - LAG) & LAG][rt][kt], even[kt], odd[kt]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (SC && LAG > 0) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int kt = 0; kt < KT; kt++) add_block(7, S[rt][kt], T[7 & LAG][rt][kt], even[kt], odd[kt]);
            }
            load_ks(nat, nb);
            if constexpr (!SC) {
                static_assert(SC || KT == 1, "all scores");
                if constexpr (RT == 1) mfma_settle(S[0][0]);
                else mfma_settle(S[0][0], S[1][0]);
            }

            // online softmax: a lane holds keys kb + 16 kt + 4 lg + i of row i16
            bool masked = kb < seg.lo || kb + TILE > vmin;
#pragma unroll
            for (int kt = 0; kt < KT; kt++) masked |= at[kt] < 0;
            h8 p8[RT];
            float cr[RT];
            bool moved = false;
#pragma unroll
            for (int rt = 0; rt < RT; rt++) {
                if (masked) {
#pragma unroll
                    for (int kt = 0; kt < KT; kt++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int key = kb + 16 * kt + 4 * lg + i;
                            S[rt][kt][i] = at[kt] >= 0 && key >= seg.lo && key < vis[rt] ? S[rt][kt][i] : -INFINITY;
                        }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int kt = 0; kt < KT; kt++) mx = max3f(max3f(mx, S[rt][kt][0], S[rt][kt][1]), S[rt][kt][2], S[rt][kt][3]);
                mx = rows_max(mx);
                const float mx2 = mx * PF_LOG2E, mn = mx2 > m[rt] + BT_HEAD ? mx2 - BT_RAISE : m[rt];
                const float ref = mn == -INFINITY ? 0.0f : mn;  // a row that saw nothing keeps l = 0, O = 0
                cr[rt] = mn == m[rt] ? 1.0f : fast_exp2(m[rt] - mn);
                // the sum is that of the rounded probabilities, the weights that P V applies
                const h2 one2 = {(_Float16)1.0f, (_Float16)1.0f};
                float rs = 0.0f, rx = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float x = j < 4 * KT ? fast_exp2(fmaf(S[rt][(j >> 2) % KT][j & 3], PF_LOG2E, -ref)) : 0.0f;
                    p8[rt][j] = (_Float16)x;
                    if (ROWS::SUM && j < 4 * KT) rx += x;
                }
#pragma unroll
                for (int j = 0; j < 4 * KT; j += 2) rs = __builtin_amdgcn_fdot2(h2{p8[rt][j], p8[rt][j + 1]}, one2, rs, false);
                l[rt] = l[rt] * cr[rt] + rs;
                if (ROWS::SUM) lx[rt] = lx[rt] * cr[rt] + rx;
                m[rt] = mn;
                moved |= cr[rt] != 1.0f;
            }
            if (__any(moved)) {
#pragma unroll
                for (int rt = 0; rt < RT; rt++)
#pragma unroll
                    for (int dt = 0; dt < 16; dt++) o[rt][dt] *= cr[rt];
            }

            // O^T += V^T P^T: output tile dt holds the lane's dim dt
            uint32_t vd[4 * KT];
#pragma unroll
            for (int j = 0; j < 4 * KT; j++)
                vd[j] = SC ? h2_bits(scale_of(vsd[j / 4], 4 * (4 * lg + j % 4) + (i16 >> 2), (i16 >> 1) & 1)) & 0xFFFFu : 0u;
            constexpr int DPW = 16 / VW;
            if (masked) {
                us2 top = {0, 0};
#pragma unroll
                for (int j = 0; j < 4 * KT; j++) {
                    if constexpr (SC) {
                        top = max_bits(top, vd[j]);
                    } else {
#pragma unroll
                        for (int wi = 0; wi < VW; wi++) top = max_bits(top, vr[j][wi]);
                    }
                }
                if (__any(reaches(top, ODD_FROM<KVT>))) {
                    // which rows see how many such values: the product of ones in their place with ones for the seen keys
                    const f4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
                    h4 seen[RT][KT];
#pragma unroll
                    for (int rt = 0; rt < RT; rt++)
#pragma unroll
                        for (int kt = 0; kt < KT; kt++)
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const int key = kb + 16 * kt + 4 * lg + j;
                                seen[rt][kt][j] = at[kt] >= 0 && key >= seg.lo && key < vis[rt] ? (_Float16)1.0f : (_Float16)0.0f;
                            }
                    if constexpr (SC) {  // (a block as a whole; the lane's 16 dims lie in one)
                        h4 ones[KT];
#pragma unroll
                        for (int j = 0; j < 4 * KT; j++) {
                            const bool odd = (vd[j] & 0x7FFFu) >= ODD_FROM<KVT>;
                            ones[j / 4][j % 4] = odd ? (_Float16)1.0f : (_Float16)0.0f;
                            vd[j] = odd ? 0u : vd[j];
                        }
#pragma unroll
                        for (int rt = 0; rt < RT; rt++) {
                            f4 count = zero;
#pragma unroll
                            for (int kt = 0; kt < KT; kt++) count = bt_mfma16k16(ones[kt], seen[rt][kt], count);
#pragma unroll
                            for (int dt = 0; dt < 16; dt++) nan_where(o[rt][dt], count);
                        }
                    } else {
#pragma unroll
                        for (int wi = 0; wi < VW; wi++) {
                            uint32_t ones[4], lo[DPW], hi[DPW];
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const uint32_t odd = odd_halves(vr[j][wi]);
                                ones[j] = odd & 0x3C003C00u;
                                vr[j][wi] &= ~odd;
                            }
                            bt_v_pair<KVT>(ones[0], ones[1], 0, 0, lo);
                            bt_v_pair<KVT>(ones[2], ones[3], 0, 0, hi);
#pragma unroll
                            for (int d = 0; d < DPW; d++)
#pragma unroll
                                for (int rt = 0; rt < RT; rt++)
                                    nan_where(o[rt][wi * DPW + d], bt_mfma16k16(make_h4(lo[d], hi[d]), seen[rt][0], zero));
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
            }
#pragma unroll
            for (int wi = 0; wi < VW; wi++) {
                __builtin_amdgcn_sched_barrier(0);
                uint32_t w[2 * KT][DPW];
#pragma unroll
                for (int h = 0; h < 2 * KT; h++)
                    bt_v_pair<KVT>(vr[2 * h][wi], vr[2 * h + 1][wi], vd[2 * h], vd[2 * h + 1], w[h]);
#pragma unroll
                for (int d = 0; d < DPW; d++)
#pragma unroll
                    for (int rt = 0; rt < RT; rt++) {
                        f4& acc = o[rt][wi * DPW + d];
                        if constexpr (KT == 2)
                            acc = mfma16(make_h8(w[0][d], w[1][d], w[2][d], w[3][d]), p8[rt], acc);
                        else
                            acc = bt_mfma16k16(make_h4(w[0][d], w[1][d]), h4{p8[rt][0], p8[rt][1], p8[rt][2], p8[rt][3]}, acc);
                    }
            }
            load_vs(nat, nb);
#pragma unroll
            for (int kt = 0; kt < KT; kt++) at[kt] = nat[kt];
        }

        // the next segment's first loads, where the registers hold them beside this one's sums
        const typename ROWS::SEGMENT cur = seg;
        const bool more = next(seg);
        if (RT == 1 && more) begin();
        // the waves' states, joined in two rounds of 8 output tiles (twice the LDS would cost a workgroup per CU): in round h
        // wave w takes tiles 8 h + QS w on
#pragma unroll
        for (int rt = 0; rt < RT; rt++) {
            const float lt = rows_sum(l[rt]), lxt = ROWS::SUM ? rows_sum(lx[rt]) : 0.0f;
            const int r = cur.row0 + 16 * rt + i16;
            const size_t place = rows.place(cur, r);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                __syncthreads();  // the previous round's states (or the last tile's Q) are read out
#pragma unroll
                for (int dt = 0; dt < 8; dt++) s_o[wave][dt][lane] = o[rt][8 * h + dt];
                if (h == 0) {
                    s_ml[wave][0][lane] = m[rt];
                    s_ml[wave][1][lane] = lt;
                    if constexpr (ROWS::SUM) s_ml[wave][2][lane] = lxt;
                }
                __syncthreads();
                float M = -INFINITY, L = 0.0f, X = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; w++) M = fmaxf(M, s_ml[w][0][lane]);
                f4 acc[QS] = {};
#pragma unroll
                for (int w = 0; w < WAVES; w++) {
                    const float mw = s_ml[w][0][lane], lw = s_ml[w][1][lane];
                    const float f = lw == 0.0f ? 0.0f : fast_exp2(mw - M);  // (lw: NaN scores stay NaN)
                    L = fmaf(f, lw, L);
                    if constexpr (ROWS::SUM) X = fmaf(f, s_ml[w][2][lane], X);
#pragma unroll
                    for (int t = 0; t < QS; t++) {
                        const f4 x = s_o[w][QS * wave + t][lane];
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[t][i] = fmaf(f, x[i], acc[t][i]);
                    }
                }
                if (r < cur.rows) {
                    if (h == 0 && wave == 0 && lg == 0) rows.sums(cur, place, M, L, X);
                    // (output tile dt of lane row x = 4 lg + i holds dim 16 x + dt, of F16 128 (dt / 8) + 8 x + dt % 8)
                    constexpr int STEP = KVT == QWA_KV_F16 ? 8 : 16;
                    float* dst = rows.o(cur, place) + (KVT == QWA_KV_F16 ? 128 : 8) * h + QS * wave;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        if constexpr (QS == 2)
                            *reinterpret_cast<float2*>(dst + STEP * (4 * lg + i)) = make_float2(acc[0][i], acc[1][i]);
                        else
                            dst[STEP * (4 * lg + i)] = acc[0][i];
                    }
                }
            }
        }
        if (!more) break;
        if (RT > 1) begin();
        __syncthreads();  // the states are read out of LDS
    }
}

}  // namespace qwa
