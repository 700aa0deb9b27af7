// Eviction from a paged cache by the attention weight that positions gathered (gfx950).
//
// A sequence of m positions is cut to `keep`: each KV head of each layer keeps its last min(recent, keep) positions and, of the
// others, those of the largest weight w_j, the lower position of equals, in their order.  With r_0 < r_1 < ... the positions
// kept, row r_i of K, V, scales and weights moves to position i; the layers and heads keep different positions, but as many, so
// one length and one table row serve them all.
//  * k_evict_select (a workgroup per request, layer and head, and one per request for its pages) finds the smallest weight kept by
//    its bits, 11 at a time (a histogram in LDS of those that agree in the bits before), and lists the kept positions' places in
//    the pool.  Nothing changes yet.
//  * k_evict_plan (one workgroup) checks all requests, takes pages for those of the first `keep` positions that other sequences
//    hold too, and changes the tables.
//  * k_evict_move (one or four workgroups per request, layer, head, and K or V) moves the rows in order, a run at a time: position
//    i <= r_i, so a run is written where no later run reads, and after all of it has been read.
#include <algorithm>

#include "launch.hpp"
#include "page_tables.hpp"

namespace qwa {

constexpr int EV_T = 1024;       // threads of the selecting and the planning workgroups
constexpr int EV_E = 32;         // most weights a thread holds
constexpr int EV_BINS = 2048;
constexpr int EV_LANE = 16;      // weights a lane holds where one wave does
static_assert(64 * EV_LANE < 1 << 15 && EV_LANE % 16 == 0, "counts of both kinds in a word, a page a 16 positions");
static_assert(EV_T >= QWA_PAGES_MAXN, "one thread per request");

// work buffer (ints): whether the plan holds, then per request its number of shared pages (-1: invalid, -2: nothing to do), the
// kept part's pages that are shared, the pages taken for them, then the kept positions' places and weights [request][layer]
// [head][max_keep]
struct EvictWork {
    size_t count, shared, fresh, rows, mass, ints;
};
__host__ __device__ inline EvictWork evict_work(const qwa_kv_pages& p, int n, int n_layers, int max_keep) {
    const size_t pages = (size_t)n * ((max_keep + p.page - 1) / p.page), rows = (size_t)n * n_layers * NKV * max_keep;
    EvictWork w;
    w.count = 4;
    w.shared = w.count + n;
    w.fresh = w.shared + pages;
    w.rows = w.fresh + pages;
    w.mass = w.rows + rows;
    w.ints = w.mass + rows;
    return w;
}
size_t evict_work_bytes(const qwa_kv_pages& p, int n, int n_layers, int max_keep) {
    return 4 * evict_work(p, n, n_layers, max_keep).ints;
}

struct EvictArgs {
    qwa_kv_pages p;
    const int* seqs;
    const int* keep;
    int n, n_layers, recent, max_keep;
    float* mass;  // [layer][sequence][KV head][ld * page]
    int* work;
};

// a number's place in the order of numbers, NaN first
__device__ __forceinline__ uint32_t ev_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 is 0)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A workgroup reads up to EV_T * EV_E weights once, into registers (more of them once for each histogram and once for what stays), and
// is then bound by its own instructions and barriers: of 36 us for 32768 positions (64 workgroups) the weights and the first
// histogram take 7, a histogram's search and the next one 4 to 5 each, counting what stays 7, writing it 7.  Measured and as fast:
// neighbouring positions over a wave's lanes instead of in a thread's registers (and places by ballots); slower (42): the first 11
// bits by counting bit by bit.
__global__ void __launch_bounds__(EV_T) k_evict_select(EvictArgs a) {
    __shared__ __attribute__((aligned(16))) int s_hist[EV_BINS];
    __shared__ long long s_wave[EV_T / 64];
    __shared__ int s_bin, s_above;
    const int t = threadIdx.x, i = blockIdx.y, lh = blockIdx.x;
    const EvictWork w = evict_work(a.p, a.n, a.n_layers, a.max_keep);
    const int seq = a.seqs[i], keep = a.keep[i];
    int m = -1;
    if (seq >= 0 && seq < a.p.n_seq && keep >= 0 && keep <= a.max_keep) m = a.p.len[seq];
    const bool valid = m >= 0 && m <= (long long)a.p.ld * a.p.page;
    const int* __restrict__ table = a.p.table + (size_t)max(seq, 0) * a.p.ld;
    if (lh == a.n_layers * NKV) {  // the request's pages, by a workgroup of its own
        int bad = !valid, shared = 0;
        if (valid && m > keep) {
            const int kept = pages_of(keep, a.p.page), per = pages_of(a.max_keep, a.p.page);
            for (int e = t; e < pages_of(m, a.p.page); e += EV_T) {
                const int pg = table[e];
                if (!page_ok(pg, a.p)) bad = 1;
                else if (e < kept) {
                    const int x = a.p.ref[pg] > 1;
                    a.work[w.shared + (size_t)i * per + e] = x;
                    shared += x;
                }
            }
        }
        long long all;
        block_scan<EV_T>(((long long)bad << 32) + shared, s_wave, &all);
        if (t == 0) a.work[w.count + i] = (all >> 32) ? -1 : m > keep ? (int)(all & 0xffffffffLL) : -2;
        return;
    }
    if (!valid || m <= keep || keep == 0) return;

    const int near = min(a.recent, keep), c = m - near;  // candidates [0, c), of which `want` stay
    int want = keep - near;
    const size_t ld = (size_t)a.p.ld * a.p.page;
    const int l = lh / NKV, h = lh % NKV;
    const float* __restrict__ mass = a.mass + (((size_t)l * a.p.n_seq + seq) * NKV + h) * ld;
    // Runs of EV_T * per positions, `per` neighbouring ones a thread (a multiple of 4: the loads).  One run is read once.
    const int per = min(EV_E, (m + 4 * EV_T - 1) / (4 * EV_T) * 4), run = EV_T * per, runs = (m + run - 1) / run;
    float x[EV_E];
    auto load = [&](int r) {
        const int j0 = r * run + t * per;
#pragma unroll
        for (int e = 0; e < EV_E; e += 4)
            if (e < per) {
                if (j0 + e + 3 < m) {
                    const float4 v = *reinterpret_cast<const float4*>(mass + j0 + e);
                    x[e] = v.x; x[e + 1] = v.y; x[e + 2] = v.z; x[e + 3] = v.w;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) x[e + k] = j0 + e + k < m ? mass[j0 + e + k] : 0.0f;
                }
            }
    };
    if (runs == 1) load(0);
    const size_t at = ((size_t)i * a.n_layers * NKV + lh) * a.max_keep;
    int* const rows = a.work + w.rows + at;
    float* const out = reinterpret_cast<float*>(a.work + w.mass) + at;
    const int sh = __builtin_ctz(a.p.page);
    if (m <= 64 * EV_LANE) {
        // Few positions: one wave, EV_LANE neighbouring ones a lane, without LDS or barriers.  The key, the largest that at least
        // `want` candidates reach, bit by bit.  (By the histograms below 600 positions take 19 us, this way 13.)
        if (t >= 64) return;
        float x[EV_LANE];
        uint32_t k[EV_LANE];
        const int j0 = EV_LANE * t;
        int pg[EV_LANE / 16];
#pragma unroll
        for (int e = 0; e < EV_LANE; e++) x[e] = j0 + e < m ? mass[j0 + e] : 0.0f;
#pragma unroll
        for (int e = 0; e < EV_LANE / 16; e++)
            pg[e] = table[min(j0 + 16 * e, m - 1) >> sh];  // (a foreign page's request changes nothing)
#pragma unroll
        for (int e = 0; e < EV_LANE; e++) k[e] = j0 + e < c ? ev_key(x[e]) : 0u;
        uint32_t key = 0;
        if (want > 0) {
            for (int bit = 31; bit >= 0; bit--) {
                const uint32_t up = key | 1u << bit;
                int reach = 0;
#pragma unroll
                for (int e = 0; e < EV_LANE; e++) reach += __popcll(__ballot(k[e] >= up));
                if (reach >= want) key = up;
            }
            int above = 0;
#pragma unroll
            for (int e = 0; e < EV_LANE; e++) above += __popcll(__ballot(k[e] > key));
            want -= above;  // of those that equal it
        }
        int more = 0, same = 0;
#pragma unroll
        for (int e = 0; e < EV_LANE; e++) {
            const bool last = j0 + e >= c && j0 + e < m, cand = j0 + e < c && keep > near;
            more += last || (cand && k[e] > key);
            same += cand && k[e] == key;
        }
        int sum = more | same << 16;  // (at most 64 * EV_LANE of both)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int y = __shfl_up(sum, o, 64);
            if (t >= o) sum += y;
        }
        sum -= more | same << 16;
        int before = sum >> 16, place = (sum & 0xffff) + min(before, want);
#pragma unroll
        for (int e = 0; e < EV_LANE; e++) {
            const bool cand = j0 + e < c && keep > near;
            bool stays = (j0 + e >= c && j0 + e < m) || (cand && k[e] > key);
            if (cand && k[e] == key) stays = before++ < want;
            if (stays && place < keep) {
                rows[place] = (pg[e / 16] << sh) + ((j0 + e) & (a.p.page - 1));
                out[place++] = x[e];
            }
        }
        return;
    }
    // the smallest key that stays, by its highest 11 bits, the next 11 and the last 10
    uint32_t key = 0;
    if (want > 0) {
#pragma unroll
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : EV_BINS;
            for (int k = t; k < EV_BINS; k += EV_T) s_hist[k] = 0;
            __syncthreads();
            for (int r = 0; r < runs; r++) {
                if (runs > 1) load(r);
                const int j0 = r * run + t * per;
#pragma unroll
                for (int e = 0; e < EV_E; e++)
                    if (e < per && j0 + e < c) {
                        const uint32_t k = ev_key(x[e]);
                        if (pass == 0 || (k >> (pass == 1 ? 21 : 10)) == (key >> (pass == 1 ? 21 : 10)))
                            atomicAdd(&s_hist[(k >> shift) & (bins - 1)], 1);
                    }
            }
            __syncthreads();
            // from the highest bin down: the first at which `want` are reached
            const int b1 = bins - 1 - 2 * t, b0 = b1 - 1;
            const int n1 = b1 >= 0 ? s_hist[b1] : 0, n0 = b0 >= 0 ? s_hist[b0] : 0;
            long long all;
            const int above = (int)block_scan<EV_T>(n1 + n0, s_wave, &all);
            if (above < want && want <= above + n1) {
                s_bin = b1;
                s_above = above;
            } else if (above + n1 < want && want <= above + n1 + n0) {
                s_bin = b0;
                s_above = above + n1;
            }
            __syncthreads();
            key |= (uint32_t)s_bin << shift;
            want -= s_above;  // of those that agree up to here
            __syncthreads();
        }
    }
    // kept: the last ones, those above the key, and the first `want` that equal it
    const int all_want = keep - near;
    long long done = 0;  // kept so far, and (upper half) equals so far
    for (int r = 0; r < runs; r++) {
        if (runs > 1) load(r);
        const int j0 = r * run + t * per;
        // the pages of the thread's positions (of 16 positions at least: three for 32), on their way meanwhile
        int pg[3];
#pragma unroll
        for (int k = 0; k < 3; k++) pg[k] = table[min((j0 >> sh) + k, (m - 1) >> sh)];
        int more = 0, same = 0;
#pragma unroll
        for (int e = 0; e < EV_E; e++)
            if (e < per && j0 + e < m) {
                const uint32_t k = ev_key(x[e]);
                const bool last = j0 + e >= c;
                more += last || (all_want > 0 && k > key);
                same += !last && all_want > 0 && k == key;
            }
        long long total;
        const long long mine = done + block_scan<EV_T>(((long long)same << 32) + more, s_wave, &total);
        done += total;
        int before = (int)(mine >> 32);                                  // equals before the thread's
        int place = (int)(mine & 0xffffffffLL) + min(before, want);
        if (more + same > 0) {
#pragma unroll
            for (int e = 0; e < EV_E; e++)
                if (e < per && j0 + e < m) {
                    const uint32_t k = ev_key(x[e]);
                    const bool last = j0 + e >= c;
                    bool stays = last || (all_want > 0 && k > key);
                    if (!last && all_want > 0 && k == key) stays = before++ < want;
                    if (stays && place < keep) {
                        const int k = ((j0 + e) >> sh) - (j0 >> sh);
                        const int base = k == 0 ? pg[0] : k == 1 ? pg[1] : pg[2];
                        rows[place] = (base << sh) + ((j0 + e) & (a.p.page - 1));  // (a foreign page's request changes nothing)
                        out[place++] = x[e];
                    }
                }
        }
    }
}

// The requests together: all of them, or none.  One workgroup's latency: 4 to 9 us.
__global__ void __launch_bounds__(EV_T) k_evict_plan(EvictArgs a, int* __restrict__ dropped, int* __restrict__ status) {
    __shared__ long long s_wave[EV_T / 64];
    __shared__ int s_seq[EV_T], s_count[EV_T], s_base[EV_T], s_bad;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const EvictWork w = evict_work(a.p, a.n, a.n_layers, a.max_keep);
    const int seq = t < a.n ? a.seqs[t] : -1, count = t < a.n ? a.work[w.count + t] : -2;
    s_seq[t] = seq;
    s_count[t] = count;
    if (t == 0) s_bad = EV_T;
    __syncthreads();
    bool ok = count != -1;
    for (int j = 0; j < min(a.n, t); j++) ok &= s_seq[j] != seq;
    if (t < a.n && !ok) atomicMin(&s_bad, t);
    long long total;
    s_base[t] = (int)block_scan<EV_T>(max(count, 0), s_wave, &total);
    if (t < a.n) dropped[t] = 0;
    if (s_bad < EV_T) {  // (every thread passed block_scan's barriers after the atomicMin)
        if (t == 0) {
            *status = -(s_bad + 1);
            a.work[0] = 0;
        }
        return;
    }
    // the lowest free pages
    int* const fresh = a.work + w.fresh;
    long long found = 0;
    for (long long i0 = 0; i0 < a.p.n_pages && found < total; i0 += 4 * EV_T) {
        const int i = (int)i0 + 4 * t;
        int f[4], c = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) f[k] = i + k < a.p.n_pages ? a.p.ref[i + k] : 1;
#pragma unroll
        for (int k = 0; k < 4; k++) c += f[k] <= 0;
        long long got;
        long long at = found + block_scan<EV_T>(c, s_wave, &got);
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (f[k] <= 0) {
                if (at < total) fresh[at] = i + k;
                at++;
            }
        found += got;
    }
    if (found < total) {
        if (t == 0) {
            *status = (int)min(total - found, 0x7fffffffLL);
            a.work[0] = 0;
        }
        return;
    }
    __syncthreads();
    // the tables, a wave a request
    const int per = pages_of(a.max_keep, a.p.page);
    for (int i = wave; i < a.n; i += EV_T / 64) {
        if (s_count[i] < 0) continue;
        const int s = s_seq[i], keep = a.keep[i], m = a.p.len[s], kept = pages_of(keep, a.p.page);
        int* const row = a.p.table + (size_t)s * a.p.ld;
        int base = s_base[i];
        for (int e0 = 0; e0 < pages_of(m, a.p.page); e0 += 64) {
            const int e = e0 + lane;
            const bool used = e < pages_of(m, a.p.page);
            const bool copied = used && e < kept && a.work[w.shared + (size_t)i * per + e] != 0;
            const unsigned long long mask = __ballot(copied);
            if (used && (copied || e >= kept)) {
                const int pg = row[e];
                atomicSub(a.p.ref + pg, 1);
                int to = -1;
                if (copied) {
                    to = fresh[base + __popcll(mask & ((1ull << lane) - 1))];
                    a.p.ref[to] = 1;
                }
                row[e] = to;
            }
            base += __popcll(mask);
        }
        if (lane == 0) {
            a.p.len[s] = keep;
            dropped[i] = m - keep;
        }
    }
    if (t == 0) {
        *status = 0;
        a.work[0] = 1;
    }
}

// The rows of a request, layer and head, of K or V.  While a run is written, the next one is on its way, and the places of that after
// it.  The order of the rows binds a workgroup, but their columns do not depend on each other: of F16 each of four workgroups has
// 128 bytes of a row (6 sequences of up to 8000 cut to 2000 or less in 16 layers, 1.41 GB: 310 us, 4.5 TB/s; whole rows 349).
// Rows of the quantized types, of 256 and 128 bytes, stay whole (one Q4_0 document of 32768 cut to 4096 in 16 layers: 51 us, in four
// parts 52; 151 MB, but a row's 16 bytes of scales are read as a line of 128, 0.21 GB; two Q8_0 of 600 to 256 10, in parts 12).
constexpr int EV_MT = 512;  // threads
template <int KVT>
constexpr int EV_PARTS = KVT == QWA_KV_F16 ? 4 : 1;
template <int KVT>
__global__ void __launch_bounds__(EV_MT) k_evict_move(EvictArgs a, PageLayers layers) {
    constexpr int PARTS = EV_PARTS<KVT>;
    constexpr int VB = value_bytes(KVT), UNITS = VB / 16 / PARTS;  // 16-byte units of a row's part
    constexpr int U = PARTS == 1 ? 8 : 4;                          // units a thread moves of a run
    constexpr int ROWS = EV_MT * U / UNITS;                        // rows of it
    constexpr int SU = KVT == QWA_KV_F16 ? 0 : (ROWS + EV_MT - 1) / EV_MT;  // rows whose scales it moves
    const int t = threadIdx.x;
    const EvictWork w = evict_work(a.p, a.n, a.n_layers, a.max_keep);
    // (parts of the same rows 8 workgroups apart: one XCD, whose L2 then holds their lines)
    const int part = blockIdx.x / 8 % PARTS, unit = blockIdx.x / (8 * PARTS) * 8 + blockIdx.x % 8;
    const int which = unit & 1, lh = unit >> 1, i = blockIdx.y;
    const int l = lh / NKV, h = lh % NKV;
    if (a.work[0] == 0 || a.work[w.count + i] < 0) return;
    const int seq = a.seqs[i], keep = a.keep[i], sh = __builtin_ctz(a.p.page);
    const int* __restrict__ table = a.p.table + (size_t)seq * a.p.ld;
    const size_t at = ((size_t)i * a.n_layers * NKV + lh) * a.max_keep;
    const int* __restrict__ rows = a.work + w.rows + at;
    const qwa_kv_layer& kv = layers.l[l];
    const size_t head = (size_t)h * kv.capacity;
    uint8_t* const vals = (which ? kv.v : kv.k) + head * VB + (VB / PARTS) * part;
    uint16_t* const scales = KVT == QWA_KV_F16 ? nullptr : (which ? kv.vs : kv.ks) + head * 8;
    const bool do_scales = SU > 0 && part == 0;
    if (which == 0 && part == PARTS - 1) {
        float* const mass = a.mass + (((size_t)l * a.p.n_seq + seq) * NKV + h) * ((size_t)a.p.ld * a.p.page);
        const float* const src = reinterpret_cast<const float*>(a.work + w.mass) + at;
        for (int r = t; r < keep; r += EV_MT) mass[r] = src[r];
    }
    struct Places {
        int from[U], to[U], sfrom[SU > 0 ? SU : 1], sto[SU > 0 ? SU : 1];
    };
    struct Values {
        uint4 x[U], sc[SU > 0 ? SU : 1];
    };
    auto look = [&](Places& b, int r0) {  // (equal ones: nothing to move)
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = min(r0 + (t + EV_MT * u) / UNITS, keep - 1);
            b.from[u] = rows[r];
            b.to[u] = (table[r >> sh] << sh) + (r & (a.p.page - 1));
        }
        if (do_scales)
#pragma unroll
            for (int u = 0; u < SU; u++) {
                const int r = min(r0 + t + EV_MT * u, keep - 1);
                b.sfrom[u] = rows[r];
                b.sto[u] = (table[r >> sh] << sh) + (r & (a.p.page - 1));
            }
    };
    // which of the places are the run's
    auto live = [&](int r0, int u) { return r0 + (t + EV_MT * u) / UNITS < keep; };
    auto slive = [&](int r0, int u) { return do_scales && t + EV_MT * u < ROWS && r0 + t + EV_MT * u < keep; };
    auto load = [&](Values& v, const Places& b, int r0) {
#pragma unroll
        for (int u = 0; u < U; u++)
            if (live(r0, u) && b.from[u] != b.to[u])
                v.x[u] = *reinterpret_cast<const uint4*>(vals + (size_t)b.from[u] * VB + 16 * ((t + EV_MT * u) % UNITS));
        if constexpr (SU > 0)
#pragma unroll
            for (int u = 0; u < SU; u++)
                if (slive(r0, u) && b.sfrom[u] != b.sto[u])
                    v.sc[u] = *reinterpret_cast<const uint4*>(scales + (size_t)b.sfrom[u] * 8);
    };
    auto store = [&](Values& v, const Places& b, int r0) {
        // everything of the run is in registers before any of it is written
#pragma unroll
        for (int u = 0; u < U; u++) asm volatile("" : "+v"(v.x[u].x), "+v"(v.x[u].y), "+v"(v.x[u].z), "+v"(v.x[u].w));
        if constexpr (SU > 0)
#pragma unroll
            for (int u = 0; u < SU; u++) asm volatile("" : "+v"(v.sc[u].x), "+v"(v.sc[u].y), "+v"(v.sc[u].z), "+v"(v.sc[u].w));
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++)
            if (live(r0, u) && b.from[u] != b.to[u])
                *reinterpret_cast<uint4*>(vals + (size_t)b.to[u] * VB + 16 * ((t + EV_MT * u) % UNITS)) = v.x[u];
        if constexpr (SU > 0)
#pragma unroll
            for (int u = 0; u < SU; u++)
                if (slive(r0, u) && b.sfrom[u] != b.sto[u]) *reinterpret_cast<uint4*>(scales + (size_t)b.sto[u] * 8) = v.sc[u];
    };
    if (keep == 0) return;
    // a run is read behind all places of those before it that are still to be written
    Places p0, p1, p2;
    Values v0 = {}, v1 = {};
    look(p0, 0);
    look(p1, ROWS);
    load(v0, p0, 0);
    for (int r0 = 0; r0 < keep; r0 += 2 * ROWS) {
        look(p2, r0 + 2 * ROWS);
        load(v1, p1, r0 + ROWS);
        store(v0, p0, r0);
        p0 = p2;
        look(p2, r0 + 3 * ROWS);
        load(v0, p0, r0 + 2 * ROWS);
        store(v1, p1, r0 + ROWS);
        p1 = p2;
    }
}

hipError_t launch_pages_evict(const qwa_kv_pages& p, const int* seqs, const int* keep, int n, int recent, int max_keep,
                              const qwa_kv_layer* layers, int n_layers, int kvt, float* mass, int* dropped, int* status,
                              void* work, hipStream_t st) {
    const EvictArgs a{p, seqs, keep, n, n_layers, recent, max_keep, mass, static_cast<int*>(work)};
    if (n > 0) hipLaunchKernelGGL(k_evict_select, dim3(n_layers * NKV + 1, n), dim3(EV_T), 0, st, a);
    hipLaunchKernelGGL(k_evict_plan, dim3(1), dim3(EV_T), 0, st, a, dropped, status);
    if (n == 0) return hipGetLastError();
    const PageLayers pl = page_layers(layers, n_layers);
#define QWA_EV(T) \
    hipLaunchKernelGGL(k_evict_move<T>, dim3(2 * n_layers * NKV * EV_PARTS<T>, n), dim3(EV_MT), 0, st, a, pl)
    switch (kvt) {
        case QWA_KV_F16: QWA_EV(QWA_KV_F16); break;
        case QWA_KV_Q8_0: QWA_EV(QWA_KV_Q8_0); break;
        default: QWA_EV(QWA_KV_Q4_0); break;
    }
#undef QWA_EV
    return hipGetLastError();
}

}  // namespace qwa
