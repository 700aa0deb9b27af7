// What the operators on page tables have in common.
#pragma once

#include "qwattn_common.hpp"

namespace qwa {

// pages of the first m positions (m >= 0)
__device__ __forceinline__ int pages_of(long long m, int page) { return (int)((m + page - 1) / page); }
__device__ __forceinline__ bool page_ok(int pg, const qwa_kv_pages& p) { return (unsigned)pg < (unsigned)p.n_pages; }
// entries of sequence s's row in use (a length outside [0, ld * page] is cut to it)
__device__ __forceinline__ int held(const qwa_kv_pages& p, int s) {
    const int m = p.len[s];
    return m <= 0 ? 0 : min(p.ld, pages_of(m, p.page));
}

// exclusive sum over the workgroup's T threads, and the total
template <int T>
__device__ __forceinline__ long long block_scan(long long v, long long* s_wave, long long* total) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long y = __shfl_up(x, o, 64);
        if (lane >= o) x += y;
    }
    __syncthreads();  // s_wave may still be read from the last scan
    if (lane == 63) s_wave[wave] = x;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        const long long y = s_wave[w];
        if (w < wave) before += y;
        all += y;
    }
    *total = all;
    return before + x - v;
}

struct PageLayers {
    qwa_kv_layer l[QWA_PAGES_MAXL];
};

inline PageLayers page_layers(const qwa_kv_layer* layers, int n_layers) {
    PageLayers pl = {};
    for (int i = 0; i < n_layers; i++) pl.l[i] = layers[i];
    return pl;
}

}  // namespace qwa
