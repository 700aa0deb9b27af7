// Page tables of a batch of sequences (gfx950): room with copy-on-write, forks, trims, compaction.
//
// A page is a run of positions of a KV layer (the pool), so a page is 4 runs (KV heads) in each of K, V and their scale
// rows, and the same tables serve every layer.  The tables, lengths and reference counts live on the device and change in
// stream order: a decode step (room, prep, attention) is captured once and replayed while the sequences grow, and beams
// are permuted from indices that only the device knows.
//
// Every operator gives the same result whatever the order in which workgroups run: counts change by integer atomics whose
// sum does not depend on the order, and which page goes where is decided by one workgroup (k_extend, k_compact) from
// prefix sums.  One workgroup suffices: it reads the counts once (4 B a page).
#include <algorithm>

#include "launch.hpp"
#include "page_tables.hpp"

namespace qwa {

constexpr int PG_T = 1024;  // threads of the planning workgroups; also the most requests of a call (one a thread)
static_assert(PG_T >= QWA_PAGES_MAXN, "one thread per request");

struct PageMove {
    int from, to, rows;  // pages, and how many of their first positions
};

// work buffer: the number of moves, then the moves, then what each operator needs besides
//  extend: PG_T moves, free pages [n_pages];  compact: n_pages / 2 + 1 moves, new number of each page [n_pages];
//  fork: per request its page count (-1: ignored) and length, then the staged rows [n][ld]
constexpr int PG_HDR = 4;  // ints
__host__ __device__ inline size_t pg_moves_ints(int moves) { return PG_HDR + 3 * (size_t)moves; }

size_t pages_work_bytes(const qwa_kv_pages& p) {
    const size_t ext = pg_moves_ints(PG_T) + p.n_pages;
    const size_t cmp = pg_moves_ints(p.n_pages / 2 + 1) + p.n_pages;
    const size_t n = p.n_seq < QWA_PAGES_MAXN ? p.n_seq : QWA_PAGES_MAXN;
    const size_t frk = n * (2 + (size_t)p.ld);
    return 4 * std::max(ext, std::max(cmp, frk));
}

constexpr int PG_PT = 4;  // counts per thread and round of the searches through ref

// Room, by a workgroup of T >= n threads: thread i plans request i.  Requests are served in order (an exclusive sum of the
// pages that they need), and of the requests whose last, partly filled page is the same, the first ref - 1 move away to
// copies and the last may keep it.  Latency: the tables, the counts and three barriers' round trips, 4.5 us for 3 requests, 8.8
// for 100 of which each looks at all before it.
template <int T>
__global__ void __launch_bounds__(T) k_extend(qwa_kv_pages p, const int* __restrict__ seqs,
                                                 const int* __restrict__ add, int n, int* __restrict__ status,
                                                 int* __restrict__ work) {
    __shared__ long long s_wave[T / 64];
    __shared__ int2 s_req[T];  // (sequence, last page)
    __shared__ int s_base[T], s_have[T];
    __shared__ int s_bad;
    const int t = threadIdx.x;
    PageMove* moves = reinterpret_cast<PageMove*>(work + PG_HDR);
    int* free_list = work + pg_moves_ints(PG_T);
    if (t == 0) s_bad = PG_T;
    int s = -1, m = 0, a = 0, tail = -1, r = 0;
    bool ok = true;
    if (t < n) {
        s = seqs[t];
        a = add[t];
        ok = s >= 0 && s < p.n_seq;
        if (ok) {
            m = p.len[s];
            ok = a >= 0 && m >= 0 && (long long)m + a <= (long long)p.ld * p.page && (long long)m + a <= 0x7fffffffLL;
        }
        if (ok && a > 0 && m % p.page != 0) {
            tail = p.table[(size_t)s * p.ld + m / p.page];
            ok = page_ok(tail, p);
            if (ok) r = p.ref[tail];
            else tail = -1;
        }
    }
    s_req[t] = make_int2(s, tail);
    __syncthreads();
    int rank = 0, same = 0;
#pragma unroll 8
    for (int j = 0; j < min(n, t); j++) {
        const int2 q = s_req[j];
        same += q.x == s;
        rank += q.y == tail;
    }
    ok = ok && same == 0;
    if (t < n && !ok) atomicMin(&s_bad, t);
    const bool cow = tail >= 0 && rank < r - 1;
    const int have = ok ? pages_of(m, p.page) : 0;
    const int need = t < n && ok ? pages_of((long long)m + a, p.page) - have + cow : 0;
    // pages and copies in one sum (at most PG_T copies)
    constexpr int CB = 12;
    static_assert(PG_T < 1 << CB, "the copies' field");
    long long total;
    long long base = block_scan<T>(((long long)need << CB) + (cow && ok), s_wave, &total);
    const int cbase = (int)(base & ((1 << CB) - 1)), copies = (int)(total & ((1 << CB) - 1));
    base >>= CB;
    total >>= CB;
    if (t == 0) work[0] = 0;
    if (s_bad < PG_T) {  // (every thread passed block_scan's barriers after the atomicMin)
        if (t == 0) *status = -(s_bad + 1);
        return;
    }
    // the lowest free pages
    long long found = 0;
    for (long long i0 = 0; i0 < p.n_pages && found < total; i0 += T * PG_PT) {
        const int i = (int)i0 + PG_PT * t;
        int f[PG_PT], c = 0;
#pragma unroll
        for (int k = 0; k < PG_PT; k++) f[k] = i + k < p.n_pages ? p.ref[i + k] : 1;
#pragma unroll
        for (int k = 0; k < PG_PT; k++) c += f[k] <= 0;
        long long got;
        long long at = found + block_scan<T>(c, s_wave, &got);
#pragma unroll
        for (int k = 0; k < PG_PT; k++)
            if (f[k] <= 0) {
                if (at < total) free_list[at] = i + k;
                at++;
            }
        found += got;
    }
    if (found < total) {
        if (t == 0) *status = (int)(total - found > 0x7fffffffLL ? 0x7fffffffLL : total - found);
        return;
    }
    // (total <= n_pages from here on)
    s_base[t] = (int)base;
    // request t's plan, for the threads that carry it out
    s_have[t] = cow ? -have : have;  // (a copied page: have >= 1)
    __syncthreads();
    for (int k = t; k < (int)total; k += T) {
        // the last request whose base is at most k needs page k
        int lo = 0, hi = n;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_base[mid] <= k) lo = mid;
            else hi = mid;
        }
        const int h = s_have[lo], first = h < 0 ? -h - 1 : h;  // first entry that gets a page
        const int pg = free_list[k];
        p.table[(size_t)s_req[lo].x * p.ld + first + (k - s_base[lo])] = pg;
        p.ref[pg] = 1;
    }
    if (t < n) {
        if (cow) {
            moves[cbase] = {tail, free_list[base], m % p.page};
            atomicSub(p.ref + tail, 1);
        }
        p.len[s] = m + a;
    }
    if (t == 0) {
        work[0] = copies;
        *status = 0;
    }
}

// Compaction: pages in use at or past their number n_live move to the free ones below it, in order.
__global__ void __launch_bounds__(PG_T) k_compact(qwa_kv_pages p, int* __restrict__ n_live, int* __restrict__ work) {
    __shared__ long long s_wave[PG_T / 64];
    const int t = threadIdx.x;
    PageMove* moves = reinterpret_cast<PageMove*>(work + PG_HDR);
    int* map = work + pg_moves_ints(p.n_pages / 2 + 1);
    int c = 0;
    for (long long i = t; i < p.n_pages; i += PG_T) c += p.ref[i] > 0;
    long long live;
    block_scan<PG_T>(c, s_wave, &live);
    long long holes = 0, movers = 0;
    for (long long i0 = 0; i0 < p.n_pages; i0 += PG_T * PG_PT) {
        const int i = (int)i0 + PG_PT * t;
        int f[PG_PT];
        long long h = 0;  // holes, and movers in the upper half
#pragma unroll
        for (int k = 0; k < PG_PT; k++) f[k] = i + k < p.n_pages ? p.ref[i + k] > 0 : -1;
#pragma unroll
        for (int k = 0; k < PG_PT; k++) h += f[k] < 0 ? 0 : i + k < live ? !f[k] : (long long)f[k] << 32;
        long long got;
        const long long at = block_scan<PG_T>(h, s_wave, &got);
        long long hole = holes + (at & 0xffffffffLL), mover = movers + (at >> 32);
#pragma unroll
        for (int k = 0; k < PG_PT; k++) {
            if (f[k] < 0) continue;
            if (i + k < live) {
                if (!f[k]) moves[hole++].to = i + k;
            } else {
                map[i + k] = i + k;
                if (f[k]) moves[mover++].from = i + k;
            }
        }
        holes += got & 0xffffffffLL;
        movers += got >> 32;
    }
    __syncthreads();  // holes == movers <= n_pages / 2: both counts are pages in use above n_live
    for (long long k = t; k < movers; k += PG_T) {
        const int from = moves[k].from, to = moves[k].to;
        moves[k].rows = p.page;
        map[from] = to;
        p.ref[to] = p.ref[from];
        p.ref[from] = 0;
    }
    if (t == 0) {
        work[0] = (int)movers;
        *n_live = (int)live;
    }
}

// Carries out the moves in every layer: a unit is a move of one layer and KV head (a run of K and one of V rows, and
// their scale rows), units are strided over the workgroups.  A move's source and target are different pages, and no page
// is both, so the order does not matter.  Bytes: compacting 1500 Q4_0 pages of 16 layers moves 876 MB in 181 us (4.8 TB/s; a
// large copy reaches 5.15), 100 copies of 43 F16 positions in 16 layers take 59 us (282 MB written, the one source is read
// from the caches).  REMAP: the tables follow the moves (map of the pages from n_live on).
template <bool REMAP>
__global__ void __launch_bounds__(256) k_move(qwa_kv_pages p, const int* __restrict__ work, PageLayers layers,
                                              int n_layers, int vb, int sb, const int* __restrict__ map,
                                              const int* __restrict__ n_live) {
    const int t = threadIdx.x;
    if (REMAP) {
        const int live = *n_live;
        for (int s = blockIdx.x; s < p.n_seq; s += gridDim.x) {
            const int k = held(p, s);
            for (int e = t; e < k; e += 256) {
                const int pg = p.table[(size_t)s * p.ld + e];
                if (page_ok(pg, p) && pg >= live) p.table[(size_t)s * p.ld + e] = map[pg];
            }
        }
    }
    const PageMove* moves = reinterpret_cast<const PageMove*>(work + PG_HDR);
    const long long units = (long long)work[0] * n_layers * NKV;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int h = (int)(u % NKV), li = (int)(u / NKV % n_layers);
        const PageMove mv = moves[u / NKV / n_layers];
        const qwa_kv_layer& kv = layers.l[li];
        const size_t from = (size_t)h * kv.capacity + (size_t)mv.from * p.page;
        const size_t to = (size_t)h * kv.capacity + (size_t)mv.to * p.page;
        const int nv = mv.rows * (vb / 16);
        const uint4* ks = reinterpret_cast<const uint4*>(kv.k + from * vb);
        const uint4* vs = reinterpret_cast<const uint4*>(kv.v + from * vb);
        uint4* kd = reinterpret_cast<uint4*>(kv.k + to * vb);
        uint4* vd = reinterpret_cast<uint4*>(kv.v + to * vb);
        for (int e = t; e < nv; e += 256) {
            const uint4 a = ks[e], b = vs[e];
            kd[e] = a;
            vd[e] = b;
        }
        if (sb) {
            for (int e = t; e < 2 * mv.rows; e += 256) {
                const uint16_t* src = e < mv.rows ? kv.ks : kv.vs;
                uint16_t* dst = e < mv.rows ? kv.ks : kv.vs;
                const int row = e < mv.rows ? e : e - mv.rows;
                reinterpret_cast<uint4*>(dst + to * 8)[row] = reinterpret_cast<const uint4*>(src + from * 8)[row];
            }
        }
    }
}

// Forks and trims: a workgroup has PG_CH requests, a thread an entry of their rows.  Neighbouring requests often hold the
// same page there (forks of one prompt), so a thread adds up the changes of equal pages in a row and sends one atomic for
// them.  (One request per workgroup, one atomic per request and page: 100 forks of 313 pages 11 instead of 5 us a kernel.)
constexpr int PG_CH = 16;
constexpr int PG_RT = 512;  // threads

struct PageSum {
    int page = -1, count = 0;
    __device__ __forceinline__ void add(const qwa_kv_pages& p, int pg, int by) {
        if (pg != page) {
            flush(p);
            page = pg;
        }
        count += by;
    }
    __device__ __forceinline__ void flush(const qwa_kv_pages& p) {
        if (count != 0 && page_ok(page, p)) atomicAdd(p.ref + page, count);
        count = 0;
    }
};

// which of the workgroup's requests [i0, i0 + PG_CH) are repeated by a later one that counts (bit k: request i0 + k gives way)
template <class COUNTS>
__device__ __forceinline__ uint32_t repeated(const int* __restrict__ seqs, int n, int i0, uint32_t* s_mask, COUNTS counts) {
    if (threadIdx.x == 0) *s_mask = 0;
    __syncthreads();
    constexpr int L = PG_RT / PG_CH;  // threads per request
    const int k = threadIdx.x / L, i = i0 + k;
    bool later = false;
    if (i < n) {
        const int s = seqs[i];
        for (int j = i + 1 + (int)(threadIdx.x % L); j < n; j += L) later |= seqs[j] == s && counts(j);
    }
    if (later) atomicOr(s_mask, 1u << k);
    __syncthreads();
    return *s_mask;
}

// Fork, first half: the requests' new rows are staged, and their pages counted once more, before any row changes.
// work: page counts [n] (-1: ignored), lengths [n], rows [n][ld].
__global__ void __launch_bounds__(PG_RT) k_fork_stage(qwa_kv_pages p, const int* __restrict__ src,
                                                      const int* __restrict__ dst, int n, int* __restrict__ work) {
    __shared__ uint32_t s_mask;
    __shared__ int s_src[PG_CH], s_k[PG_CH];
    const int i0 = blockIdx.x * PG_CH, t = threadIdx.x;
    const uint32_t gone = repeated(dst, n, i0, &s_mask, [&](int j) { return src[j] < p.n_seq; });
    if (t < PG_CH) {
        const int i = i0 + t;
        int s = -1, k = -1, m = 0;
        if (i < n) {
            s = src[i];
            const int d = dst[i];
            if (!((gone >> t) & 1) && d >= 0 && d < p.n_seq && s < p.n_seq) {
                k = s < 0 ? 0 : held(p, s);
                m = s < 0 ? 0 : p.len[s];
            }
            work[i] = k;
            work[n + i] = m;
        }
        s_src[t] = s;
        s_k[t] = k;
    }
    __syncthreads();
    int most = 0;
#pragma unroll
    for (int k = 0; k < PG_CH; k++) most = max(most, s_k[k]);
    for (int e = t; e < most; e += PG_RT) {
        PageSum sum;
        int pg[PG_CH];
#pragma unroll
        for (int k = 0; k < PG_CH; k++) pg[k] = e < s_k[k] ? p.table[(size_t)s_src[k] * p.ld + e] : -1;
#pragma unroll
        for (int k = 0; k < PG_CH; k++)
            if (e < s_k[k]) {
                work[2 * (size_t)n + (size_t)(i0 + k) * p.ld + e] = pg[k];
                sum.add(p, pg[k], 1);
            }
        sum.flush(p);
    }
}

// Second half: the old pages are given back and the staged rows put in their place.
__global__ void __launch_bounds__(PG_RT) k_fork_commit(qwa_kv_pages p, const int* __restrict__ dst, int n,
                                                       const int* __restrict__ work) {
    __shared__ int s_dst[PG_CH], s_k[PG_CH], s_old[PG_CH];
    const int i0 = blockIdx.x * PG_CH, t = threadIdx.x;
    if (t < PG_CH) {
        const int i = i0 + t, k = i < n ? work[i] : -1, d = k < 0 ? 0 : dst[i];
        s_dst[t] = d;
        s_k[t] = k;
        s_old[t] = k < 0 ? -1 : held(p, d);
        if (k >= 0) p.len[d] = work[n + i];  // (no other workgroup has this sequence)
    }
    __syncthreads();
    int most = 0;
#pragma unroll
    for (int k = 0; k < PG_CH; k++) most = max(most, max(s_k[k], s_old[k]));
    for (int e = t; e < most; e += PG_RT) {
        PageSum sum;
        int pg[PG_CH], to[PG_CH];
#pragma unroll
        for (int k = 0; k < PG_CH; k++) {
            pg[k] = e < s_old[k] ? p.table[(size_t)s_dst[k] * p.ld + e] : -1;
            to[k] = e < s_k[k] ? work[2 * (size_t)n + (size_t)(i0 + k) * p.ld + e] : -1;
        }
#pragma unroll
        for (int k = 0; k < PG_CH; k++) {
            if (e < s_old[k]) sum.add(p, pg[k], -1);
            if (e < max(s_k[k], s_old[k])) p.table[(size_t)s_dst[k] * p.ld + e] = to[k];
        }
        sum.flush(p);
    }
}

__global__ void __launch_bounds__(PG_RT) k_trim(qwa_kv_pages p, const int* __restrict__ seqs, const int* __restrict__ lens,
                                                int n) {
    __shared__ uint32_t s_mask;
    __shared__ int s_seq[PG_CH], s_keep[PG_CH], s_old[PG_CH];
    const int i0 = blockIdx.x * PG_CH, t = threadIdx.x;
    // (Another workgroup may be cutting len[s] meanwhile, to the length of the last request that counts.  That one counts
    // before and after; those behind it, longer than the sequence or negative, do not; those before it give way to it.)
    const uint32_t gone = repeated(seqs, n, i0, &s_mask, [&](int j) {
        const int s = seqs[j], to = lens ? lens[j] : 0;
        return s >= 0 && s < p.n_seq && to >= 0 && to <= p.len[s];
    });
    if (t < PG_CH) {
        const int i = i0 + t;
        int s = 0, keep = 0, old = 0;
        if (i < n && !((gone >> t) & 1)) {
            s = seqs[i];
            if (s >= 0 && s < p.n_seq) {
                const int to = lens ? lens[i] : 0;
                if (to >= 0 && to <= p.len[s]) {
                    keep = pages_of(to, p.page);
                    old = held(p, s);
                    p.len[s] = to;  // (no other workgroup has this sequence)
                }
            } else {
                s = 0;
            }
        }
        s_seq[t] = s;
        s_keep[t] = keep;
        s_old[t] = old;
    }
    __syncthreads();
    int most = 0;
#pragma unroll
    for (int k = 0; k < PG_CH; k++) most = max(most, s_old[k]);
    int least = most;  // (nothing to give back: no entries)
#pragma unroll
    for (int k = 0; k < PG_CH; k++)
        if (s_keep[k] < s_old[k]) least = min(least, s_keep[k]);
    for (int e = least + t; e < most; e += PG_RT) {
        PageSum sum;
        int pg[PG_CH];
#pragma unroll
        for (int k = 0; k < PG_CH; k++)
            pg[k] = e >= s_keep[k] && e < s_old[k] ? p.table[(size_t)s_seq[k] * p.ld + e] : -1;
#pragma unroll
        for (int k = 0; k < PG_CH; k++)
            if (e >= s_keep[k] && e < s_old[k]) {
                sum.add(p, pg[k], -1);
                p.table[(size_t)s_seq[k] * p.ld + e] = -1;
            }
        sum.flush(p);
    }
}

constexpr long long PG_MOVE_WG = 4096;  // workgroups of k_move at most

hipError_t launch_pages_extend(const qwa_kv_pages& p, const int* seqs, const int* add, int n, const qwa_kv_layer* layers,
                               int n_layers, int kvt, int* status, void* work, hipStream_t st) {
    int* w = static_cast<int*>(work);
    // (few requests: the barriers of a small workgroup cost less; 3 requests 9.9 instead of 12.5 us)
    if (n <= 256) hipLaunchKernelGGL(k_extend<256>, dim3(1), dim3(256), 0, st, p, seqs, add, n, status, w);
    else hipLaunchKernelGGL(k_extend<PG_T>, dim3(1), dim3(PG_T), 0, st, p, seqs, add, n, status, w);
    const long long units = std::max(1LL, (long long)n * n_layers * NKV);
    hipLaunchKernelGGL(k_move<false>, dim3((unsigned)std::min(units, PG_MOVE_WG)), dim3(256), 0, st, p, w,
                       page_layers(layers, n_layers), n_layers, value_bytes(kvt), kvt == QWA_KV_F16 ? 0 : 16,
                       (const int*)nullptr, (const int*)nullptr);
    return hipGetLastError();
}

hipError_t launch_pages_compact(const qwa_kv_pages& p, const qwa_kv_layer* layers, int n_layers, int kvt, int* n_live,
                                void* work, hipStream_t st) {
    int* w = static_cast<int*>(work);
    hipLaunchKernelGGL(k_compact, dim3(1), dim3(PG_T), 0, st, p, n_live, w);
    const long long units = std::max((long long)(p.n_pages / 2) * n_layers * NKV, (long long)p.n_seq);
    hipLaunchKernelGGL(k_move<true>, dim3((unsigned)std::min(units, PG_MOVE_WG)), dim3(256), 0, st, p, w,
                       page_layers(layers, n_layers), n_layers, value_bytes(kvt), kvt == QWA_KV_F16 ? 0 : 16,
                       w + pg_moves_ints(p.n_pages / 2 + 1), n_live);
    return hipGetLastError();
}

hipError_t launch_pages_fork(const qwa_kv_pages& p, const int* src, const int* dst, int n, void* work, hipStream_t st) {
    int* w = static_cast<int*>(work);
    const dim3 grid((n + PG_CH - 1) / PG_CH), block(PG_RT);
    hipLaunchKernelGGL(k_fork_stage, grid, block, 0, st, p, src, dst, n, w);
    hipLaunchKernelGGL(k_fork_commit, grid, block, 0, st, p, dst, n, w);
    return hipGetLastError();
}

hipError_t launch_pages_trim(const qwa_kv_pages& p, const int* seqs, const int* lens, int n, hipStream_t st) {
    hipLaunchKernelGGL(k_trim, dim3((n + PG_CH - 1) / PG_CH), dim3(PG_RT), 0, st, p, seqs, lens, n);
    return hipGetLastError();
}

}  // namespace qwa
