// Raw KV tiles in LDS, their conversion to fp16 MFMA tiles, and the 16-bit partial states: what the prefill kernels and the
// batched decode over a shared prefix have in common (workgroups of PF_WAVES waves, tiles of PF_TILE keys).
#pragma once

#include "kv_operands.hpp"
#include "pf_plan.hpp"

namespace qwa {

constexpr int PF_THREADS = PF_WAVES * 64;
constexpr int PF_KT = PF_TILE / 16;              // 16-key MFMA tiles per tile
constexpr int KS_LD = HD + 8;                    // K tile row stride (halves)
constexpr int VT_LD = PF_TILE + 8;               // V^T tile row stride (halves)
constexpr float PF_LOG2E = 1.4426950408889634f;
constexpr float PF_RESCALE_T = 8.0f;  // lazy-rescale threshold on the running maximum (natural-log units)

// raw bytes of one tile in LDS, in the cache's own layout: K rows, V rows, K scales, V scales (8 fp16 per row)
template <int KVT> struct PfRaw {
    static constexpr int VB = value_bytes(KVT);
    static constexpr int K = 0, V = PF_TILE * VB;
    static constexpr int SC = KVT == QWA_KV_F16 ? 0 : PF_TILE * 16;
    static constexpr int KS = 2 * PF_TILE * VB, VS = KS + SC;
    static constexpr int BYTES = 2 * PF_TILE * VB + 2 * SC;
    static constexpr int NKV = PF_TILE * VB / 1024;          // 1 KB load instructions for K (and for V)
    static constexpr int NBUF = KVT == QWA_KV_F16 ? 2 : 3;   // raw tiles in flight (F16 tiles are 32 KB)
    static constexpr int AHEAD = NBUF - 1;                    // tiles loaded ahead of the one being computed
    // load instructions of wave w per tile: K instruction i on wave i % W, V instruction i on wave (i + W / 2) % W,
    // K scales (two 256-byte instructions) on waves W - 2, W - 1, V scales on waves W / 2 - 2, W / 2 - 1
    __device__ static constexpr int count(int w) {
        int n = 0;
        for (int i = 0; i < NKV; i++) n += (i % PF_WAVES == w) + ((i + PF_WAVES / 2) % PF_WAVES == w);
        if (SC) n += (w >= PF_WAVES - 2) + (w >= PF_WAVES / 2 - 2 && w < PF_WAVES / 2);
        return n;
    }
};

// waits until at most n of this wave's direct-to-LDS loads are outstanding (n is wave-uniform)
__device__ __forceinline__ void wait_vm(int n) {
    switch (n) {
        case 0: wait_vmcnt<0>(); break;
        case 1: wait_vmcnt<1>(); break;
        case 2: wait_vmcnt<2>(); break;
        case 3: wait_vmcnt<3>(); break;
        case 4: wait_vmcnt<4>(); break;
        case 5: wait_vmcnt<5>(); break;
        case 6: wait_vmcnt<6>(); break;
        case 7: wait_vmcnt<7>(); break;
        case 8: wait_vmcnt<8>(); break;
        case 9: wait_vmcnt<9>(); break;
        case 10: wait_vmcnt<10>(); break;
        case 11: wait_vmcnt<11>(); break;
        case 12: wait_vmcnt<12>(); break;
        default: wait_vmcnt<0>(); break;
    }
}

// 4 dims of one V key as two half2 {d0, d1}, {d2, d3}, scaled by the key's block scale (one fp16 rounding)
template <int KVT>
__device__ __forceinline__ void pf_v4(const uint8_t* vrow, int dc, uint32_t sc, uint32_t* out) {
    if constexpr (KVT == QWA_KV_F16) {
        const uint2 u = *reinterpret_cast<const uint2*>(vrow + 8 * dc);
        out[0] = u.x;
        out[1] = u.y;
    } else if constexpr (KVT == QWA_KV_Q8_0) {
        const h2 d = scale_pair((uint16_t)sc, (uint16_t)sc);
        q8_word_to_h4(*reinterpret_cast<const uint32_t*>(vrow + 4 * dc), d, out);
    } else {
        const h2 d = scale_pair((uint16_t)sc, (uint16_t)sc);
        const h2 bias = {(_Float16)1032.0f, (_Float16)1032.0f};
        const uint32_t x = *reinterpret_cast<const uint16_t*>(vrow + 2 * dc);
        // byte 0 -> dims 0 (low nibble), 1 (high nibble); byte 1 -> dims 2, 3
        const uint32_t p01 = ((x & 0x0Fu) | ((x & 0xF0u) << 12)) | 0x64006400u;
        const uint32_t p23 = (((x >> 8) & 0x0Fu) | (((x >> 8) & 0xF0u) << 12)) | 0x64006400u;
        out[0] = h2_bits((bits_h2(p01) - bias) * d);
        out[1] = h2_bits((bits_h2(p23) - bias) * d);
    }
}

// Dequantises one raw tile into the fp16 tiles (thread t of 512).  K: LDS position 32 s + 8 g + j of a row holds dim
// 32 s + 8 g + perm(j) (the Q operand is loaded with the same permutation).  V^T: row d, position 8 cb + j holds key
// 16 (j / 4) + 4 cb + j % 4, the key order of the P^T operand (lane group g of a 16-key MFMA tile holds keys
// 4 g .. 4 g + 3).
template <int KVT>
__device__ __forceinline__ void pf_convert_kv(const uint8_t* raw, _Float16* Ks, _Float16* Vt, int t, bool do_k,
                                              bool do_v) {
    using L = PfRaw<KVT>;
    constexpr int VB = L::VB;
    const uint16_t* kss = reinterpret_cast<const uint16_t*>(raw + L::KS);
    const uint16_t* vss = reinterpret_cast<const uint16_t*>(raw + L::VS);
    if (!do_k) {
    } else if constexpr (KVT == QWA_KV_F16) {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int idx = t + 512 * c, key = idx >> 5, pc = idx & 31;
            *reinterpret_cast<uint4*>(Ks + key * KS_LD + 8 * pc) =
                *reinterpret_cast<const uint4*>(raw + L::K + key * VB + 16 * pc);
        }
    } else if constexpr (KVT == QWA_KV_Q8_0) {
        const int key = t >> 4, pc = t & 15;
        const uint4 u = *reinterpret_cast<const uint4*>(raw + L::K + key * VB + 16 * pc);
        const uint16_t sc = kss[key * 8 + (pc >> 1)];
        const h2 d = scale_pair(sc, sc);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; i++) q8_word_to_h4(w[i], d, o + 2 * i);
        *reinterpret_cast<uint4*>(Ks + key * KS_LD + 16 * pc) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(Ks + key * KS_LD + 16 * pc + 8) = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
        if (t < PF_TILE * 8) {
            const int key = t >> 3, pc = t & 7;
            const uint4 u = *reinterpret_cast<const uint4*>(raw + L::K + key * VB + 16 * pc);
            const uint16_t sc = kss[key * 8 + pc];
            const h2 d = scale_pair(sc, sc);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t o[4];
                q4_word_to_h8(w[i], d, o);
                *reinterpret_cast<uint4*>(Ks + key * KS_LD + 32 * pc + 8 * i) = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
    }
    if (!do_v) return;
    // V^T: thread (cb, dc, h) converts keys 16 h + 4 cb + jj (jj < 4), dims 4 dc .. 4 dc + 3
    const int cb = t & 3, dc = (t >> 2) & 63, h = t >> 8;
    uint32_t hv[4][2];
#pragma unroll
    for (int jj = 0; jj < 4; jj++) {
        const int key = 16 * h + 4 * cb + jj;
        const uint32_t sc = KVT == QWA_KV_F16 ? 0u : (uint32_t)vss[key * 8 + (dc >> 3)];
        pf_v4<KVT>(raw + L::V + key * VB, dc, sc, hv[jj]);
    }
#pragma unroll
    for (int d = 0; d < 4; d++) {
        const uint32_t sel = (d & 1) ? 0x07060302u : 0x05040100u;  // high / low half of both words
        const uint32_t w0 = __builtin_amdgcn_perm(hv[1][d >> 1], hv[0][d >> 1], sel);
        const uint32_t w1 = __builtin_amdgcn_perm(hv[3][d >> 1], hv[2][d >> 1], sel);
        *reinterpret_cast<uint2*>(Vt + (4 * dc + d) * VT_LD + 8 * cb + 4 * h) = make_uint2(w0, w1);
    }
}

// The conversion is cut into 512 K units and 512 V units, spread over the workgroup's threads
template <int KVT>
__device__ __forceinline__ void pf_convert(const uint8_t* raw, _Float16* Ks, _Float16* Vt, int t) {
    if constexpr (PF_THREADS == 512) {
        pf_convert_kv<KVT>(raw, Ks, Vt, t, true, true);
    } else {
#pragma unroll
        for (int u = t; u < 1024; u += PF_THREADS) pf_convert_kv<KVT>(raw, Ks, Vt, u & 511, u < 512, u >= 512);
    }
}

__device__ __forceinline__ h8 lds_h8(const _Float16* p) { return *reinterpret_cast<const h8*>(p); }

// max of three floats in one instruction (fmaxf would first canonicalize each MFMA result; scores are never sNaN)
__device__ __forceinline__ float max3f(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// max / sum over the four 16-lane rows of the wave (lanes l, l ^ 16, l ^ 32, l ^ 48) with the gfx950 lane swaps:
// permlane16_swap(x, x) leaves row pairs {r0, r0, r2, r2} / {r1, r1, r3, r3}, permlane32_swap {lo, lo} / {hi, hi}
__device__ __forceinline__ float rows_max(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    float y;
    asm("v_max_f32 %0, %1, %2" : "=v"(y) : "v"(__uint_as_float(a[0])), "v"(__uint_as_float(a[1])));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    asm("v_max_f32 %0, %1, %2" : "=v"(y) : "v"(__uint_as_float(b[0])), "v"(__uint_as_float(b[1])));
    return y;
}
__device__ __forceinline__ float rows_sum(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// 16-bit partials: O / l of a (split, row) as signed 16-bit fixed point against the row's largest |O / l| (the scale
// s = max / 32767 goes with (m, l)): absolute error <= s / 2 = max |O / l| * 2^-16 per value.
__device__ __forceinline__ int pf_q16(float v) { return (int)fminf(fmaxf(__builtin_rintf(v), -32767.0f), 32767.0f); }
__device__ __forceinline__ uint2 pack16x4(float a, float b, float c, float d) {
    return make_uint2(((uint32_t)pf_q16(a) & 0xFFFFu) | ((uint32_t)pf_q16(b) << 16),
                      ((uint32_t)pf_q16(c) & 0xFFFFu) | ((uint32_t)pf_q16(d) << 16));
}
__device__ __forceinline__ float4 unpack16x4(uint2 w) {
    return make_float4((float)(int16_t)(w.x & 0xFFFFu), (float)(int16_t)(w.x >> 16), (float)(int16_t)(w.y & 0xFFFFu),
                       (float)(int16_t)(w.y >> 16));
}
using PfPartO = uint2;    // four 16-bit values
using PfPartMl = float4;  // (m, l, scale, unused)

}  // namespace qwa
