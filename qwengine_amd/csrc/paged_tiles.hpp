// Tiles of 32 keys of a paged cache on their way into LDS, and the arithmetic of their scores and of V that is not finite: what
// the batched decode and the chunks of new tokens have in common.
#pragma once

#include "attn_tiles.hpp"

namespace qwa {

// The probabilities are 2^(s log2(e) - m) for a reference m that is set BT_RAISE below a row's running maximum, and set again
// when a score exceeds m by more than BT_HEAD: at most 2^15, in full fp16 precision down to 2^-14, with fewer bits down to
// 2^-24.  Those that vanish, below 2^-25, are 2^-35 to 2^-40 of the largest: 2^18 of them are less than 2^-17 of a row's sum.
// (With m at the maximum itself they were 2^-25 of the largest, and 131071 of them moved an output by 7e-3.)
// m is kept in powers of two, as it enters the exponent: a reference in units of s, multiplied when it is used, would be another
// one by the product's rounding, 0.1 at scores of a million, and the states of a row would not weigh the same.
constexpr float BT_RAISE = 10.0f, BT_HEAD = 15.0f;

// the pool position of the 16 keys from kb on (a multiple of 16), or -1: at or past the end, or in no page of the pool
__device__ __forceinline__ int bt_place(const qwa_kv_pages& p, const int* __restrict__ table, int kb, int end) {
    if (kb >= end) return -1;
    const int pg = table[kb >> __builtin_ctz(p.page)];
    return (unsigned)pg < (unsigned)p.n_pages ? pg * p.page + (kb & (p.page - 1)) : -1;
}

// MFMA results before inline assembly reads them (max3f): the compiler puts the 8 wait states that they need before
// instructions of its own, but does not look into assembly.  F16 scores are such results (they had 9 by chance); the other
// types' have passed through their block scales.
__device__ __forceinline__ void mfma_settle(f4& x) { asm volatile("s_nop 7" : "+v"(x)); }
__device__ __forceinline__ void mfma_settle(f4& x, f4& y) { asm volatile("s_nop 7" : "+v"(x), "+v"(y)); }
// Q / 16 = hi + lo, fp16 each
__device__ __forceinline__ _Float16 q_hi(float x) { return (_Float16)x; }
__device__ __forceinline__ _Float16 q_lo(float x) { return (_Float16)(x - (float)(_Float16)x); }

// `bytes` bytes from a wave-uniform address on, in 32-bit words; what is read past them is zero
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bt_buffer(const void* base, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, bytes, 0x00027000);
}
__device__ __forceinline__ uint4 bt_ld16(__amdgpu_buffer_rsrc_t b, int off) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(b, off, 0, 0));
}
__device__ __forceinline__ uint2 bt_ld8(__amdgpu_buffer_rsrc_t b, int off) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, 0));
}

// Q4_0 codes with fewer shifts than q4_word_to_h8 / v_pair_words (the same values in the same order): a nibble that sits at
// bit 4 of a half makes 64 + n there (0x5400 | n << 4), as one at bit 0 makes 1024 + n.
// (w & mask) | magic in one instruction: the mask from a scalar register, the magic from a vector register.  As two
// instructions, which the compiler makes of two constants, 24 sequences over 16384 Q4_0 positions take 78 instead of 71 us, the
// tiles of 128 over 32768 214 instead of 209.
__device__ __forceinline__ uint32_t q4_bits(uint32_t w, uint32_t mask, uint32_t magic) {
    uint32_t r;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "s"(mask), "v"(magic));
    return r;
}
__device__ __forceinline__ h2 q4_lo(uint32_t w) {
    const h2 bias = {(_Float16)1032.0f, (_Float16)1032.0f};
    return bits_h2(q4_bits(w, 0x000F000Fu, 0x64006400u)) - bias;
}
__device__ __forceinline__ h2 q4_hi(uint32_t w) {
    const h2 bias = {(_Float16)72.0f, (_Float16)72.0f};
    return bits_h2(q4_bits(w, 0x00F000F0u, 0x54005400u)) - bias;
}
// the codes c - 8 of a word
__device__ __forceinline__ void bt_q4_codes(uint32_t w, uint32_t* out) {
    out[0] = h2_bits(q4_lo(w));
    out[1] = h2_bits(q4_hi(w));
    out[2] = h2_bits(q4_lo(w >> 8));
    out[3] = h2_bits(q4_hi(w >> 8));
}
// the same, times d (one fp16 rounding)
__device__ __forceinline__ void bt_q4_values(uint32_t w, h2 d, uint32_t* out) {
    out[0] = h2_bits(q4_lo(w) * d);
    out[1] = h2_bits(q4_hi(w) * d);
    out[2] = h2_bits(q4_lo(w >> 8) * d);
    out[3] = h2_bits(q4_hi(w >> 8) * d);
}
// out[dim] = {V_a[dim], V_b[dim]} for the 8 (Q4_0), 4 or 2 dims of a word of keys a and b
template <int KVT>
__device__ __forceinline__ void bt_v_pair(uint32_t aw, uint32_t bw, uint32_t sa, uint32_t sb, uint32_t* out) {
    if constexpr (KVT == QWA_KV_Q4_0) {
        const h2 d = scale_pair((uint16_t)sa, (uint16_t)sb);
        bt_q4_values(__builtin_amdgcn_perm(bw, aw, 0x05040100u), d, out);      // bytes {a0, a1, b0, b1}
        bt_q4_values(__builtin_amdgcn_perm(bw, aw, 0x07060302u), d, out + 4);  // bytes {a2, a3, b2, b3}
    } else {
        v_pair_words<KVT, 1>(&aw, &bw, sa, sb, out);
    }
}

// ---- V that is not finite.  A key that a row does not see has probability 0, but 0 * NaN is NaN.  So in tiles of which some
// row does not see some key, such values enter P V as zeros, and a dim of O becomes NaN in the rows that see one.
typedef unsigned short us2 __attribute__((ext_vector_type(2)));
// largest magnitude (as bits) of fp16 numbers, two at a time, and whether it reaches `least`
__device__ __forceinline__ us2 max_bits(us2 m, uint32_t w) {
    return __builtin_elementwise_max(m, __builtin_bit_cast(us2, w & 0x7FFF7FFFu));
}
__device__ __forceinline__ bool reaches(us2 m, uint16_t least) { return m[0] >= least || m[1] >= least; }
// (of a quantized type a block's values are finite as long as the largest code's is: 8 * 8188, 127 * 515.5)
template <int KVT>
constexpr uint16_t ODD_FROM = KVT == QWA_KV_Q4_0 ? 0x7000 /* 8192 */ : KVT == QWA_KV_Q8_0 ? 0x6008 /* 516 */ : 0x7C00;
// all bits of the halves that are not finite
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
    return ((w & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((w & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u);
}
__device__ __forceinline__ void nan_where(f4& o, f4 count) {
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = count[i] > 0.0f ? NAN : o[i];
}

// What a thread converts of a tile, u = t & 255.  Waves 0 .. 3 (V): dims 8 c .. 8 c + 7 (c = u & 31) of the four keys 16 h +
// 4 cb .. + 3 (h = (u >> 5) & 1, cb = u >> 6), which are neighbours in the P^T operand's key order.  Waves 4 .. 7 (K): the 32
// dims of block u & 7 of key u >> 3.  The raw bytes are in registers, loaded one tile ahead.
template <int KVT>
struct BtRaw {
    static constexpr int VB = value_bytes(KVT);
    uint32_t w[VB / 32];  // V: 4 rows of VB / 128 words; K: VB / 32 words of one row
    uint32_t sc[4];       // V: the rows' block scales; K: the block's
};

// V of the 16 keys at positions at[h] of the pool (h: the lane's half of the tile), `rows` of each half valid: rows past the
// last valid one re-read that one, a half without a place (at[h] < 0, rows[h] = 16) position 0 .. 15 of the pool.  Nothing here
// looks at what was read: that would wait for it.
template <int KVT>
__device__ __forceinline__ void bt_load_v(BtRaw<KVT>& r, const uint8_t* v, const uint16_t* vs, const int* at,
                                          const int* rows, int t) {
    constexpr int VB = BtRaw<KVT>::VB;
    const int u = t & 255, c = u & 31, k0 = 4 * (u >> 6);
    const bool h = (u >> 5) & 1;
    const size_t p0 = max(at[0], 0), p1 = max(at[1], 0);
    const uint8_t* const src = (h ? v + p1 * VB : v + p0 * VB) + (VB / 32) * c;
    const uint16_t* const ssc = (h ? vs + p1 * 8 : vs + p0 * 8) + (c >> 2);
    int row[4];
#pragma unroll
    for (int j = 0; j < 4; j++) row[j] = k0 + j;
    if (rows[0] < 16 || rows[1] < 16)
#pragma unroll
        for (int j = 0; j < 4; j++) row[j] = min(row[j], (h ? rows[1] : rows[0]) - 1);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint8_t* const s = src + (uint32_t)(row[j] * VB);
        if constexpr (KVT == QWA_KV_Q4_0) {
            r.w[j] = *reinterpret_cast<const uint32_t*>(s);
        } else if constexpr (KVT == QWA_KV_Q8_0) {
            const uint2 x = ld8(s);
            r.w[2 * j] = x.x; r.w[2 * j + 1] = x.y;
        } else {
            const uint4 x = ld16(s);
            r.w[4 * j] = x.x; r.w[4 * j + 1] = x.y; r.w[4 * j + 2] = x.z; r.w[4 * j + 3] = x.w;
        }
        r.sc[j] = KVT == QWA_KV_F16 ? 0u : ssc[(uint32_t)(8 * row[j])];
    }
}

// K of the wave's 16 keys at position `at` of the pool: a buffer of its valid rows, the others read as zeros
template <int KVT>
__device__ __forceinline__ void bt_load_k(BtRaw<KVT>& r, const uint8_t* k, const uint16_t* ks, int at, int rows, int t) {
    constexpr int VB = BtRaw<KVT>::VB;
    const int u = t & 255, row = (u >> 3) & 15, blk = u & 7, n = __builtin_amdgcn_readfirstlane(at < 0 ? 0 : rows);
    const size_t pos = __builtin_amdgcn_readfirstlane(max(at, 0));
    const auto b = bt_buffer(k + pos * VB, n * VB);
#pragma unroll
    for (int i = 0; i < VB / 128; i++) {
        const uint4 x = bt_ld16(b, row * VB + (VB / 8) * blk + 16 * i);
        r.w[4 * i] = x.x; r.w[4 * i + 1] = x.y; r.w[4 * i + 2] = x.z; r.w[4 * i + 3] = x.w;
    }
    if constexpr (KVT != QWA_KV_F16)
        r.sc[0] = __builtin_amdgcn_raw_buffer_load_b16(bt_buffer(ks + pos * 8, n * 16), 16 * row + 2 * blk, 0, 0);
}

// Into the fp16 tiles, in 16-byte units so ordered that the 16 lanes that the LDS serves together (0-3, 12-15, 20-23, 24-27,
// and so on) reach distinct banks: the unit's place modulo 16 is the reading lane's i16, or that XOR a number that such lanes
// have in common.
//  K: unit (c, key) at 32 c + (key ^ 2 (c / 4)): dims 8 c .. 8 c + 7 in the operand's order;
//  V^T: unit (cb, slot) at 256 cb + slot: keys 8 cb .. 8 cb + 7 in the P^T operand's order (4 cb + 16 h + j at 4 h + j) of the
//  dim 8 (slot % 32) + slot / 32, so that the writing lanes (c = slot % 32) lie side by side, too.
// (Rows of 528 and 80 bytes instead: half of the LDS cycles were conflicts; 128 sequences over 32768 Q4_0 positions 163 us.)
// Values that are not finite become zeros; a wave that has one notes the tile, and which: of dim d and its keys 16 h + 4 cb .. + 3
// the bits of byte 8 d + 2 cb + h.
struct alignas(16) BtOdd {
    uint8_t keys[8 * HD];
    int tile[4];  // by wave (cb)
};
template <int KVT>
__device__ __forceinline__ void bt_store_v(BtRaw<KVT>& r, _Float16* Vt, BtOdd& odd, int t, uint32_t dead, int tile) {
    constexpr int VB = BtRaw<KVT>::VB, VW = VB / 128, DPW = 8 / VW;  // words of a row, dims of a word
    const int u = t & 255;
    // (a half without a place: its probabilities are zeros, and what was read need not be finite)
    if (dead != 0 && ((dead >> ((u >> 5) & 1)) & 1)) {
#pragma unroll
        for (int i = 0; i < VB / 32; i++) r.w[i] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) r.sc[j] = 0;
    }
    us2 top = {0, 0};
    if constexpr (KVT == QWA_KV_F16) {
#pragma unroll
        for (int i = 0; i < VB / 32; i++) top = max_bits(top, r.w[i]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) top = max_bits(top, r.sc[j]);
    }
    const bool any_odd = __any(reaches(top, ODD_FROM<KVT>));
    if (any_odd && (u & 63) == 0) odd.tile[u >> 6] = tile;
    _Float16* dst = Vt + 8 * (256 * (u >> 6) + (u & 31)) + 4 * ((u >> 5) & 1);
#pragma unroll
    for (int i = 0; i < VW; i++) {
        uint32_t lo[DPW], hi[DPW];
        bt_v_pair<KVT>(r.w[i], r.w[VW + i], r.sc[0], r.sc[1], lo);
        bt_v_pair<KVT>(r.w[2 * VW + i], r.w[3 * VW + i], r.sc[2], r.sc[3], hi);
        if (any_odd) {
#pragma unroll
            for (int d = 0; d < DPW; d++) {
                const uint32_t a = odd_halves(lo[d]), b = odd_halves(hi[d]);
                odd.keys[8 * (8 * (u & 31) + DPW * i + d) + 2 * (u >> 6) + ((u >> 5) & 1)] =
                    (uint8_t)((a & 1) | (a >> 31) << 1 | (b & 1) << 2 | (b >> 31) << 3);
                lo[d] &= ~a;
                hi[d] &= ~b;
            }
        }
#pragma unroll
        for (int d = 0; d < DPW; d++) *reinterpret_cast<uint2*>(dst + 8 * 32 * (DPW * i + d)) = make_uint2(lo[d], hi[d]);
    }
}
// K's codes, and their scales: unit (16 keys, pair of blocks, 4 keys) of 16 bytes, [block of the pair][key of the four]
template <int KVT>
__device__ __forceinline__ void bt_store_k(const BtRaw<KVT>& r, _Float16* Ks, uint16_t* scales, int t) {
    const int u = t & 255;
    _Float16* dst = Ks + 8 * (32 * 4 * (u & 7) + ((u >> 3) ^ (2 * (u & 7))));
    if constexpr (KVT != QWA_KV_F16) {
        const int key = u >> 3, b = u & 7;
        scales[8 * (16 * (key >> 4) + 4 * (b >> 1) + ((key >> 2) & 3)) + 4 * (b & 1) + (key & 3)] = (uint16_t)r.sc[0];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t o[4];
        if constexpr (KVT == QWA_KV_F16) {
#pragma unroll
            for (int k = 0; k < 4; k++) o[k] = r.w[4 * i + k];
        } else if constexpr (KVT == QWA_KV_Q8_0) {
            q8_word_int(r.w[2 * i], o);
            q8_word_int(r.w[2 * i + 1], o + 2);
        } else {
            bt_q4_codes(r.w[i], o);
        }
        *reinterpret_cast<uint4*>(dst + 8 * 32 * i) = make_uint4(o[0], o[1], o[2], o[3]);
    }
}

}  // namespace qwa
