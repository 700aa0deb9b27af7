"""Eviction by accumulated attention weight against a literal account on the CPU: tables, lengths, counts, weights and every byte
of the pools are equal (rows and weights are moved, never computed: no tolerance)."""
import numpy as np
import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from pageref import PageRef
from test_gpu_attn_batch import EPS, THETA, i32

pytestmark = pytest.mark.gpu


def evicted(pages, layers, mass, seqs, keep, recent, max_keep):
    """(PageRef after the call, weights after it, dropped, status) from the definition."""
    ref, w = PageRef.of(pages, layers), mass.cpu().numpy().copy()
    page, dropped = ref.page, [0] * len(seqs)
    n_seq, ld = len(ref.len), len(ref.table[0]) * page
    shared, need = {}, 0
    for i, (s, k) in enumerate(zip(seqs, keep)):
        ok = 0 <= s < n_seq and s not in seqs[:i] and 0 <= k <= max_keep and 0 <= ref.len[s] <= ld
        if ok and ref.len[s] > k:
            ok = all(0 <= ref.table[s][e] < len(ref.ref) for e in range(ref.pages_of(ref.len[s])))
        if not ok:
            return ref, w, dropped, -(i + 1)
        if ref.len[s] > k:
            shared[i] = [e for e in range(ref.pages_of(k)) if ref.ref[ref.table[s][e]] > 1]
            need += len(shared[i])
    free = [p for p, r in enumerate(ref.ref) if r <= 0]
    if need > len(free):
        return ref, w, dropped, need - len(free)
    pools, per = [p.copy() for p in ref.pools], len(ref.pools) // len(layers)
    for i, (s, k) in enumerate(zip(seqs, keep)):
        if i not in shared:
            continue
        m, old = ref.len[s], list(ref.table[s])
        for e in range(ref.pages_of(m)):
            if e >= ref.pages_of(k):
                ref.ref[old[e]] -= 1
                ref.table[s][e] = -1
            elif e in shared[i]:
                ref.ref[old[e]] -= 1
                ref.table[s][e] = free.pop(0)
                ref.ref[ref.table[s][e]] = 1
        near = min(recent, k)
        for l in range(len(layers)):
            for h in range(4):
                x = w[l, s, h, :m - near].astype(np.float64)
                x[np.isnan(x)] = -np.inf
                nan = np.isnan(w[l, s, h, :m - near])
                order = sorted(range(m - near), key=lambda j: (nan[j], -x[j] if not nan[j] else 0.0, j))
                rows = sorted(order[:k - near]) + list(range(m - near, m))
                frm = [old[j // page] * page + j % page for j in rows]
                to = [ref.table[s][j // page] * page + j % page for j in range(k)]
                for a in range(per * l, per * (l + 1)):
                    ref.pools[a][h, to] = pools[a][h, frm]
                w[l, s, h, :k] = w[l, s, h, rows].copy()
        ref.len[s] = k
        dropped[i] = m - k
    return ref, w, dropped, 0


def make(kvt, lens, page, layers, shared=0, spare=0, seed=1, ld=None):
    """Sequences over a scattered pool, the first `shared` pages of all the same; pools of random bytes."""
    up = lambda m: -(-m // page)
    n_pages = shared + sum(max(0, up(m) - shared) for m in lens) + spare
    pages = ops.KVPages.allocate(len(lens), ld or max(1, max(lens)), n_pages, page)
    perm, at = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist(), shared
    for i, m in enumerate(lens):
        row = perm[:min(shared, up(m))] + perm[at:at + max(0, up(m) - shared)]
        at += max(0, up(m) - shared)
        if row:
            pages.table[i, :len(row)] = i32(row)
            pages.ref.index_add_(0, i32(row), torch.ones(len(row), dtype=torch.int32, device="cuda"))
    pages.len.copy_(i32(lens))
    kvs = [ops.KVLayer.allocate(kvt, n_pages * page + 3) for _ in range(layers)]
    g = torch.Generator(device="cuda").manual_seed(seed)
    for kv in kvs:
        for t in (kv.k, kv.v, kv.ks, kv.vs):
            if t is not None:
                t.view(torch.uint8).random_(0, 256, generator=g)
    mass = torch.exp(2.0 * torch.randn((layers, len(lens), 4, pages.table.shape[1] * page), generator=g, device="cuda"))
    return pages, kvs, mass


def run(pages, kvs, kvt, mass, seqs, keep, recent, max_keep=None):
    max_keep = max(keep + [0]) if max_keep is None else max_keep
    want = evicted(pages, kvs, mass, seqs, keep, recent, max_keep)
    n = len(seqs)
    dropped, status = i32([77] * max(n, 1)), i32([77])
    work = torch.full((ops.kv_pages_evict_work_bytes(pages, n, len(kvs), max_keep),), 0xFF, dtype=torch.uint8, device="cuda")
    ops.kv_pages_evict(pages, i32(seqs), i32(keep), recent, max_keep, kvs, kvt, mass, dropped, status, work)
    torch.cuda.synchronize()
    ref, w, drop, st = want
    assert int(status) == st
    assert dropped.tolist()[:n] == drop
    ref.same(pages, kvs)
    assert np.array_equal(mass.cpu().numpy().view(np.uint32), w.view(np.uint32))
    return ref


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
@pytest.mark.parametrize("lens, keep, recent, page, layers", [
    ([50], [20], 5, 16, 1), ([64], [63], 0, 64, 2), ([64], [1], 1, 16, 1), ([33], [0], 4, 32, 1), ([300, 40], [100, 40], 100, 16, 3),
    ([1000, 37, 513, 0], [256, 36, 1, 0], 7, 64, 2), ([700, 600], [300, 299], 1000, 128, 2)], ids=str)
def test_evict(gpu, kvt, lens, keep, recent, page, layers):
    pages, kvs, mass = make(kvt, lens, page, layers)
    run(pages, kvs, kvt, mass, list(range(len(lens))), keep, recent).check()


def test_long_sequences(gpu):
    """More weights than a workgroup holds at once; the runs that move are longer than one."""
    pages, kvs, mass = make(ops.Q4_0, [70000, 33000], 256, 1)
    run(pages, kvs, ops.Q4_0, mass, [1, 0], [5000, 40001], 300).check()


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_equal_and_odd_weights(gpu, kvt):
    """Ties go to the lower position; zeros of both signs, negative ones, infinities, denormals; NaN goes first."""
    pages, kvs, mass = make(kvt, [400, 400, 400, 400], 32, 2)
    mass[:, 0] = 1.0
    values = torch.tensor([0.0, -0.0, 1e-45, -1e-45, 3.0, -3.0, torch.inf, -torch.inf, torch.nan, 1e-30], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    mass[:, 1] = values[torch.randint(0, 10, mass[:, 1].shape, generator=g, device="cuda")]
    mass[:, 2] = torch.randint(0, 4, mass[:, 2].shape, generator=g, device="cuda").float()
    mass[:, 3] = torch.nan
    run(pages, kvs, kvt, mass, [3, 2, 1, 0], [100, 150, 200, 250], 10).check()


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_shared_pages(gpu, kvt):
    """Pages of the kept part that others hold stay as they are; sequences that are cut together leave none of each other's
    rows; pages that nobody holds any more are free."""
    pages, kvs, mass = make(kvt, [300, 310, 290, 100], 32, 2, shared=3, spare=9)
    run(pages, kvs, kvt, mass, [2, 0], [150, 70], 20).check()
    run(pages, kvs, kvt, mass, [3, 1], [40, 200], 0).check()


def test_all_or_nothing(gpu):
    """Missing pages, invalid requests, broken tables: nothing changes."""
    kvt = ops.Q8_0
    pages, kvs, mass = make(kvt, [300, 310, 290], 32, 1, shared=4, spare=3)
    run(pages, kvs, kvt, mass, [0, 1], [100, 100], 0)      # 8 shared pages, 3 free ones
    assert pages.len.tolist() == [300, 310, 290]
    for seqs, keep, max_keep in (([0, 5], [10, 10], 10), ([0, -1], [10, 10], 10), ([1, 1], [10, 10], 10), ([0, 1], [10, -1], 10),
                                 ([0, 1], [10, 11], 10)):
        run(pages, kvs, kvt, mass, seqs, keep, 0, max_keep)
        assert pages.len.tolist() == [300, 310, 290]
    run(pages, kvs, kvt, mass, [], [], 0, 10)
    pages.table[0, 7] = 1 << 20
    run(pages, kvs, kvt, mass, [1, 0], [20, 20], 0)
    run(pages, kvs, kvt, mass, [1, 0], [20, 300], 0)       # (a sequence that is not cut is not looked at)
    pages.len[2] = 10 * 32 + 1
    run(pages, kvs, kvt, mass, [2], [20], 0)
    pages.len[2] = -1
    run(pages, kvs, kvt, mass, [2], [20], 0)


def test_many_requests(gpu):
    n = 1024
    pages, kvs, mass = make(ops.Q4_0, [20 + i % 60 for i in range(n)], 16, 1)
    run(pages, kvs, ops.Q4_0, mass, list(range(n - 1, -1, -1)), [(7 * i) % 50 for i in range(n)], 3, 50).check()


def test_pools_past_32_bits(gpu):
    """Rows past 4 GiB of a head."""
    kvt, page, n_pages = ops.F16, 1024, 8400
    pages = ops.KVPages.allocate(1, 3 * page, n_pages, page)
    pages.table[0, :3] = i32([n_pages - 1, n_pages - 3, n_pages - 2])
    pages.len.fill_(3000)
    pages.ref[n_pages - 3:] = 1
    kv = ops.KVLayer.allocate(kvt, n_pages * page)
    j = torch.arange(3000, device="cuda")
    slot = pages.table[0].long()[j // page] * page + j % page
    rows = seeded_normal((2, 4, 3000, 256), 5).half().view(torch.uint8)
    kv.k[:, slot], kv.v[:, slot] = rows[0], rows[1]
    mass = torch.rand((1, 1, 4, 3 * page), generator=torch.Generator(device="cuda").manual_seed(4), device="cuda")
    before = mass.clone()
    dropped, status = i32([0]), i32([9])
    work = torch.empty(ops.kv_pages_evict_work_bytes(pages, 1, 1, 1500), dtype=torch.uint8, device="cuda")
    ops.kv_pages_evict(pages, i32([0]), i32([1500]), 100, 1500, [kv], kvt, mass, dropped, status, work)
    torch.cuda.synchronize()
    assert int(status) == 0 and int(dropped) == 1500 and int(pages.len) == 1500 and pages.table[0].tolist()[2] == -1
    for h in range(4):
        top = before[0, 0, h, :2900].sort(descending=True, stable=True).indices[:1400].sort().values
        keep = torch.cat([top, torch.arange(2900, 3000, device="cuda")])
        assert torch.equal(kv.k[h, slot[:1500]], rows[0, h, keep]) and torch.equal(kv.v[h, slot[:1500]], rows[1, h, keep])
        assert torch.equal(mass[0, 0, h, :1500], before[0, 0, h, keep])


def test_graph_and_stream(gpu):
    """Captured once: sequences that have outgrown their budget are cut at each replay, the others left alone."""
    kvt = ops.Q8_0
    pages, kvs, mass = make(kvt, [200, 90], 16, 2, ld=512, spare=8)
    seqs, keep, dropped, status = i32([0, 1]), i32([120, 100]), i32([0, 0]), i32([9])
    work = torch.empty(ops.kv_pages_evict_work_bytes(pages, 2, 2, 120), dtype=torch.uint8, device="cuda")
    room = torch.empty(ops.kv_pages_work_bytes(pages), dtype=torch.uint8, device="cuda")
    call = lambda st=None: ops.kv_pages_evict(pages, seqs, keep, 10, 120, kvs, kvt, mass, dropped, status, work, stream=st)
    torch.cuda.synchronize()
    state = [t.clone() for t in (pages.table, pages.len, pages.ref, mass, *[x for kv in kvs for x in (kv.k, kv.v, kv.ks, kv.vs)])]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for t, x in zip((pages.table, pages.len, pages.ref, mass, *[x for kv in kvs for x in (kv.k, kv.v, kv.ks, kv.vs)]), state):
        t.copy_(x)
    for add in (0, 30, 0, 60):
        if add:
            ops.kv_pages_extend(pages, i32([1]), i32([add]), kvs, kvt, status, room)
        want = evicted(pages, kvs, mass, [0, 1], [120, 100], 10, 120)
        graph.replay()
        torch.cuda.synchronize()
        assert int(status) == want[3] == 0 and dropped.tolist() == want[2]
        want[0].same(pages, kvs)
        assert np.array_equal(mass.cpu().numpy(), want[1])
    # on a stream of its own
    side = torch.cuda.Stream()
    keep.fill_(50)
    want = evicted(pages, kvs, mass, [0, 1], [50, 50], 10, 120)
    torch.cuda.synchronize()
    call(side)
    side.synchronize()
    want[0].same(pages, kvs)
    want[0].check()


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_served_with_a_budget(gpu, kvt):
    """As an engine serves with a budget: a prompt in chunks with its weights, eviction, then tokens whose rotary positions go
    on from before it.  After the eviction attention is that over the kept rows alone."""
    page, n_pages, ld, L = 16, 60, 512, 2
    pages = ops.KVPages.allocate(2, ld, n_pages, page)
    kvs = [ops.KVLayer.allocate(kvt, n_pages * page) for _ in range(L)]
    room, status = torch.empty(ops.kv_pages_work_bytes(pages), dtype=torch.uint8, device="cuda"), i32([9])
    mass, turn = torch.zeros((L, 2, 4, ld), device="cuda"), i32([0, 0])
    w = 1 + 0.1 * seeded_normal((256,), 7)
    seed = 50
    kept = {}

    def step(counts, layer_check=None):
        nonlocal seed
        n, off = 2, [0, counts[0], sum(counts)]
        rows = off[-1]
        ops.kv_pages_extend(pages, i32([0, 1]), i32(counts), kvs, kvt, status, room)
        scratch = torch.empty(ops.attn_prefill_batch_work_bytes(n, rows, ld), dtype=torch.uint8, device="cuda")
        extra = torch.empty(ops.attn_weights_batch_work_bytes(n, rows, ld), dtype=torch.uint8, device="cuda")
        outs = []
        for l in range(L):
            seed += 5
            qg, k, v = seeded_normal((rows, 24, 512), seed), seeded_normal((rows, 4, 256), seed + 1), seeded_normal((rows, 4, 256), seed + 2)
            q, gate = torch.empty((rows, 24, 256), device="cuda"), torch.empty((rows, 24, 256), device="cuda")
            out, lse = torch.empty((rows, 24, 256), dtype=torch.float16, device="cuda"), torch.empty((rows, 24), device="cuda")
            ops.attn_prep_rows_batch(qg, k, v, w, w, pages, None, i32(off), n, rows, THETA, EPS, kvt, kvs[l], q, gate, rope_off=turn)
            ops.attn_prefill_batch(q, gate, kvs[l], kvt, pages, None, i32(off), n, rows, ld, out, scratch, lse=lse)
            ops.attn_weights_batch(q, lse, kvs[l], kvt, pages, None, i32(off), n, rows, ld, mass[l], extra)
            outs.append((q, gate, out, qg, k, v))
        torch.cuda.synchronize()
        assert int(status) == 0
        return outs

    step([200, 31])
    step([100, 1])
    dropped = i32([0, 0])
    work = torch.empty(ops.kv_pages_evict_work_bytes(pages, 2, L, 128), dtype=torch.uint8, device="cuda")
    want = evicted(pages, kvs, mass, [0, 1], [128, 128], 32, 128)
    ops.kv_pages_evict(pages, i32([0, 1]), i32([128, 128]), 32, 128, kvs, kvt, mass, dropped, status, work)
    turn += dropped
    torch.cuda.synchronize()
    assert dropped.tolist() == [172, 0] and pages.len.tolist() == [128, 32]
    want[0].same(pages, kvs)
    outs = step([1, 3])
    # the new rows were rotated as positions 300 and 32 .. 34, and stored at 128 and 32 .. 34
    for l, (q, gate, out, qg, k, v) in enumerate(outs):
        for r, s, at, pos in ((0, 0, 128, 300), (1, 1, 32, 32), (3, 1, 34, 34)):
            flat = ops.KVLayer.allocate(kvt, 64)
            src = [ops.RowSrc.device(t[r].contiguous(), x) for t, x in ((qg, 24 * 512), (k, 1024), (v, 1024))]
            q1, g1 = torch.empty((1, 24, 256), device="cuda"), torch.empty((1, 24, 256), device="cuda")
            ops.attn_prep_multi(*src, w, w, 0, pos, 1, THETA, EPS, kvt, flat, q1, g1)
            slot = int(pages.table[s, at // page]) * page + at % page
            torch.cuda.synchronize()
            assert torch.equal(q1[0], q[r]) and torch.equal(kvs[l].k[:, slot], flat.k[:, 0])
    assert (mass[:, 0, :, 128] > 0).all() and (mass[:, 1, :, 34] > 0).all()
