"""Batched prep and decode attention over a paged cache against their definitions in 64 bits, and against the
one-sequence operators on a contiguous cache.

Tolerance of the attention.  Q / 16, the dequantized K and V, the probabilities and the output are rounded to fp16, half a
step of 2^-11 relative each.  A score is a sum of 256 products of two rounded factors: for K, Q ~N(0,1) its error has a
standard deviation of about sqrt(256) / 16 * sqrt(2) * 0.29 * 2^-10 = 4e-4, which enters the output in proportion to the
probabilities, as their own rounding does, and averages over the keys: below 1e-3 of the output's norm, 2e-3 for any element,
the bar of the one-sequence operators (kvutil).  With few keys nothing averages, and V, P and the output's own rounding add
up to 3 half steps of the element: 3 * 2^-11 |out|."""
import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, MAX_ABS, REL_L2, seeded_normal
from pageref import batch_attention

pytestmark = pytest.mark.gpu
THETA, EPS = 1e7, 1e-6


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def close(got, want, what=""):
    got, want = got.double().cpu(), want.double().cpu()
    d = (got - want).abs()
    assert torch.isfinite(got).all(), what
    over = (d - 3 * 2.0**-11 * want.abs()).max().item()
    rel = (d.norm() / want.norm().clamp_min(1e-30)).item()
    print(f"{what}: max-abs {d.max().item():.2e}, rel-L2 {rel:.2e}", flush=True)
    assert over <= MAX_ABS and rel <= REL_L2, f"{what}: {d.max().item():.3e}, rel-L2 {rel:.3e}"


class Batch:
    """Sequences of given lengths over a scattered pool whose first `shared` positions are the same pages; the contiguous
    caches that hold the same rows.  Pool bytes that no sequence holds are NaN patterns."""

    def __init__(self, kvt, lens, shared=0, page=64, seed=5, ld=None):
        self.kvt, self.lens, self.page = kvt, lens, page
        whole = shared // page
        up = lambda m: -(-m // page)
        n_pages = whole + sum(max(0, up(m) - whole) for m in lens) + 3
        g = torch.Generator().manual_seed(seed)
        perm = torch.randperm(n_pages, generator=g).tolist()
        self.pages = ops.KVPages.allocate(len(lens), (ld or max(1, max(up(m) for m in lens))) * page, n_pages, page)
        self.kv = ops.KVLayer.allocate(kvt, n_pages * page + 5)
        for t in (self.kv.k, self.kv.v, self.kv.ks, self.kv.vs):
            if t is not None:
                t.view(torch.uint8).fill_(0xFF)
        K0, V0 = seeded_normal((max(shared, 1), 4, 256), seed), seeded_normal((max(shared, 1), 4, 256), seed + 1)
        self.caches, used, rows = [], whole, []
        for i, m in enumerate(lens):
            K = torch.cat([K0[:min(shared, m)], seeded_normal((max(0, m - shared), 4, 256), seed + 10 + i)])
            V = torch.cat([V0[:min(shared, m)], seeded_normal((max(0, m - shared), 4, 256), seed + 500 + i)])
            cache = ops.KVLayer.allocate(kvt, max(m, 1))
            if m:
                ops.kv_append(K, V, 0, m, kvt, cache)
            self.caches.append(cache)
            own = max(0, up(m) - whole)
            row = perm[:min(whole, up(m))] + perm[used:used + own]
            used += own
            rows.append(row)
            if row:
                self.pages.table[i, :len(row)] = i32(row)
            at = torch.arange(m, device="cuda")
            slot = i32(row or [0]).long()[at // page] * page + at % page
            for dst, src in ((self.kv.k, cache.k), (self.kv.v, cache.v), (self.kv.ks, cache.ks), (self.kv.vs, cache.vs)):
                if dst is not None:
                    dst[:, slot] = src[:, :m]
        self.pages.len.copy_(i32(lens))
        self._rows = {}

    def values(self, b):
        """K, V of sequence b as stored, [4][len][256] in 64 bits."""
        if b not in self._rows:
            c, out = self.caches[b], []
            for v, d in ((c.k, c.ks), (c.v, c.vs)):
                if self.kvt == ops.F16:
                    x = v.view(torch.float16).double()
                else:
                    x = v.view(torch.int8).double() if self.kvt == ops.Q8_0 else \
                        torch.stack([v & 15, v >> 4], -1).flatten(-2).double() - 8
                    x = x * d.view(torch.float16).double().repeat_interleave(32, -1)
                out.append(x.cpu())
            self._rows[b] = out
        return self._rows[b]

    def run(self, nq, shared, max_len, seqs=None, seed=77, oq=None, work=None):
        n = len(self.lens if seqs is None else seqs)
        q, gate = seeded_normal((n * nq, 24, 256), seed), seeded_normal((n * nq, 24, 256), seed + 1)
        out = torch.full((n * nq, 24, 256), float("nan"), dtype=torch.float16, device="cuda")
        if work is None:
            work = torch.full((ops.attn_batch_work_bytes(n, nq, shared, max_len),), 0xFF, dtype=torch.uint8, device="cuda")
        ops.attn_decode_batch(q, gate, self.kv, self.kvt, self.pages, None if seqs is None else i32(seqs), n, nq, shared,
                              max_len, out, work, oq)
        torch.cuda.synchronize()
        return q, gate, out

    def check(self, nq, shared, max_len=None, seqs=None, what="", **kw):
        max_len = max_len or max(self.lens)
        q, gate, out = self.run(nq, shared, max_len, seqs, **kw)
        order = list(range(len(self.lens))) if seqs is None else seqs
        n_seq = len(self.lens)
        length = lambda s: min(self.lens[s], max_len) if 0 <= s < n_seq else 0
        want = batch_attention(q, gate, lambda t: self.values(order[t // nq]),
                               [length(order[t // nq]) - nq + t % nq + 1 for t in range(len(order) * nq)])
        close(out, want, what or f"{KV_NAMES[self.kvt]} {self.lens} shared {shared} nq {nq}")
        return out


@pytest.mark.parametrize("nq", [1, 3, 8])
@pytest.mark.parametrize("page", [16, 32, 64, 1024])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_unshared_ragged(gpu, kvt, page, nq):
    Batch(kvt, [8, 17, 130, 63, 64, 65, 31, 257], page=page).check(nq, 0)


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
@pytest.mark.parametrize("shared", [1, 15, 16, 64, 200, 513])
def test_shared_prefix(gpu, kvt, shared):
    """Prefixes that end at, before and inside a page; own parts from one position on."""
    lens = [shared + m for m in (1, 2, 70, 129, 16, 300)]
    b = Batch(kvt, lens, shared=shared, page=64)
    b.check(1, shared)
    b.check(1, shared // 2)     # less than what is shared
    b.check(2, shared, what=f"two queries, shared {shared}")


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_everything_shared(gpu, kvt):
    """No position is a sequence's own: the call's last key is a shared one."""
    b = Batch(kvt, [128, 128, 128], shared=128)
    b.check(1, 128)
    b.check(4, 128)


@pytest.mark.parametrize("n", [1, 2, 5, 6, 11, 40, 130])
def test_batch_sizes(gpu, n):
    lens = [600 + (37 * i) % 90 for i in range(n)]
    Batch(ops.Q8_0, lens, shared=576, page=32, seed=n).check(1, 576, what=f"{n} sequences")


def test_one_token(gpu):
    for kvt in KVTS:
        Batch(kvt, [1]).check(1, 0)
        Batch(kvt, [1, 1, 2], shared=1).check(1, 1)


def test_long_contexts(gpu):
    b = Batch(ops.Q4_0, [40001, 777, 39000], page=128)
    b.check(1, 0, what="long")
    b = Batch(ops.Q8_0, [20011, 20100], shared=20000, page=16)
    b.check(7, 20000, what="long shared verify")


@pytest.mark.parametrize("n, nq, shared", [(5, 1, 0), (3, 8, 0), (40, 1, 262144), (40, 1, 200000)])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_longest_sequences(gpu, kvt, n, nq, shared):
    """The largest context: every table entry names one of 64 pages at random, so that a key counts as often as its page is
    named.  (V is about the same all over a page and differs between pages, or everything would average out.)"""
    page, pages, ld = 64, 64, 4096
    K, V = seeded_normal((pages * page, 4, 256), 31), 0.1 * seeded_normal((pages * page, 4, 256), 32)
    V += seeded_normal((pages, 4, 256), 33).repeat_interleave(page, 0)
    kv, pg = ops.KVLayer.allocate(kvt, pages * page), ops.KVPages.allocate(n, ld * page, pages, page)
    ops.kv_append(K, V, 0, pages * page, kvt, kv)
    g = torch.Generator().manual_seed(34)
    table = torch.randint(0, pages, (n, ld), generator=g, dtype=torch.int32)
    table[:, :shared // page] = table[:1, :shared // page]
    lens = [ld * page - 64 * (i % 3) * (shared < ld * page) for i in range(n)]
    pg.table.copy_(table)
    pg.len.copy_(i32(lens))
    q, gate = seeded_normal((n * nq, 24, 256), 35), seeded_normal((n * nq, 24, 256), 36)
    out = torch.empty((n * nq, 24, 256), dtype=torch.float16, device="cuda")
    work = torch.empty(ops.attn_batch_work_bytes(n, nq, shared, ld * page), dtype=torch.uint8, device="cuda")
    ops.attn_decode_batch(q, gate, kv, kvt, pg, None, n, nq, shared, ld * page, out, work)
    torch.cuda.synchronize()
    b = Batch.__new__(Batch)
    b.kvt, b.caches, b._rows = kvt, [kv], {}
    k64, v64 = b.values(0)
    want = torch.zeros((n * nq, 24, 256), dtype=torch.float64)
    for t in range(n * nq):
        m = lens[t // nq] - nq + t % nq + 1
        row = table[t // nq].long()
        count = torch.bincount(row[:m // page], minlength=pages).double().repeat_interleave(page)
        if m % page:
            count[row[m // page] * page:][:m % page] += 1
        for h in range(4):
            s = q[t, 6 * h:6 * h + 6].double().cpu() @ k64[h].T / 16.0
            p = torch.exp(s - s.amax(-1, keepdim=True)) * count
            want[t, 6 * h:6 * h + 6] = (p / p.sum(-1, keepdim=True)) @ v64[h]
    close(out, want * torch.sigmoid(gate.double().cpu()), f"{KV_NAMES[kvt]} {n} x {nq}, {shared} shared")


def test_empty_rows(gpu):
    """Empty and unknown sequences, and queries before the first position, give zeros; the rest is as without them."""
    b = Batch(ops.Q8_0, [0, 200, 3, 0, 70])
    out = b.check(5, 0)
    assert not out[0:5].any() and not out[15:20].any()       # empty sequences
    assert not out[10:12].any() and out[12].any()            # length 3: the first two of five queries see nothing
    out = b.check(1, 0, seqs=[4, -1, 1, 99, 0, 1])
    assert not out[1].any() and not out[3].any() and not out[4].any()
    empty = Batch(ops.F16, [0, 0], ld=1)
    assert not empty.run(2, 0, 64)[2].any()
    assert not empty.run(2, 40, 64)[2].any()


def test_rows_shorter_than_the_shared_part(gpu):
    """A row that has only some of the shared positions sees those; the prefix is read through the longest row."""
    for lens in ([50, 300, 128, 129, 0], [100, 90, 3]):
        Batch(ops.Q4_0, lens, shared=128, page=32, ld=13).check(1, 128, max_len=400)


def test_max_len_bounds_what_is_seen(gpu):
    b = Batch(ops.Q8_0, [300, 40, 129])
    b.check(1, 0, max_len=130)
    b.check(3, 0, max_len=1)


def test_pages_outside_the_pool_are_not_seen(gpu):
    """Positions whose page number is none of the pool's count as masked."""
    b = Batch(ops.Q8_0, [200, 64, 130], page=64)
    b.pages.table[0, 1] = 10**6
    b.pages.table[1, 0] = -1
    q, gate, out = b.run(1, 0, 200)
    K, V = b.values(0)
    keep = torch.cat([torch.arange(64), torch.arange(128, 200)])
    want = batch_attention(q[:1], gate[:1], lambda t: (K[:, keep], V[:, keep]), [136])
    close(out[:1], want, "one page missing")
    assert not out[1].any()
    close(out[2:], batch_attention(q[2:], gate[2:], lambda t: b.values(2), [130]), "the others")


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_act_q8(gpu, kvt):
    """ActQ8 rows: within a step of what the values say, and the sums of their own codes."""
    b = Batch(kvt, [90, 0, 33])
    oq = ops.ActQ8.allocate(3 * 2 * 6144)
    out = b.check(2, 0, oq=oq)
    x = out.double().view(-1, 32)
    d, q = oq.d.double(), oq.q.double().view(-1, 32)
    # the fp16 output is off its fp32 value by up to 2^-11 of it, d by as much of amax / 127
    assert ((x.abs().amax(1) / 127 - d).abs() <= 2.0**-11 * x.abs().amax(1) / 127 + 2.0**-25).all()
    assert ((q * d[:, None] - x).abs() <= d[:, None] * 0.5001 + 2.0**-11 * x.abs() + 2.0**-25).all()
    assert torch.allclose(oq.s.double(), d * q.sum(1), rtol=1e-6, atol=0)


def test_same_bits_again_and_for_forks(gpu):
    """The same call gives the same bits, whatever the work buffer held, and equal sequences give equal rows."""
    b = Batch(ops.Q4_0, [333] * 5, shared=320)
    q = seeded_normal((1, 24, 256), 3).repeat(5, 1, 1).contiguous()
    gate = torch.zeros_like(q)
    outs = []
    for fill in (0, 0xFF):
        out = torch.empty((5, 24, 256), dtype=torch.float16, device="cuda")
        work = torch.full((ops.attn_batch_work_bytes(5, 1, 320, 333),), fill, dtype=torch.uint8, device="cuda")
        ops.attn_decode_batch(q, gate, b.kv, b.kvt, b.pages, i32([2] * 5), 5, 1, 320, 333, out, work)
        torch.cuda.synchronize()
        outs.append(out)
    assert torch.equal(outs[0], outs[1])
    assert all(torch.equal(outs[0][0], outs[0][i]) for i in range(5))


def test_special_values(gpu):
    """A NaN in a seen key makes its rows NaN and no others; values of masked positions never matter."""
    b = Batch(ops.F16, [80, 90], page=16)
    slot = int(b.pages.table[1, 5]) * 16 + 1
    b.kv.k.view(torch.float16)[2, slot, 7] = float("nan")  # position 81 of sequence 1, KV head 2
    _, _, out = b.run(1, 0, 90)
    bad = torch.isnan(out).flatten(2).any(-1)
    assert bad[1, 12:18].all() and not bad[1, :12].any() and not bad[1, 18:].any() and not bad[0].any()
    b.pages.len[1] = 81                                     # the position is masked now
    _, _, out = b.run(1, 0, 90)
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("n", [2, 9])
@pytest.mark.parametrize("x", [float("nan"), float("inf")])
def test_nonfinite_values_of_shared_positions(gpu, n, x):
    """A value that is not finite shows in every row that sees it, and in no other KV head's rows (9 sequences: the partial
    states are fixed-point numbers, which have none)."""
    b = Batch(ops.F16, [200] * n, shared=130)
    b.kv.v.view(torch.float16)[1, int(b.pages.table[0, 1]) * 64 + 3, 9] = x  # position 67, KV head 1, dim 9
    _, _, out = b.run(1, 130, 200)
    bad = ~torch.isfinite(out)
    assert bad[:, 6:12, 9].all() and not bad[:, :6].any() and not bad[:, 12:].any()


def test_captured_calls_share_a_work_buffer(gpu):
    """Two captured batches with one work buffer, replayed in turn with eager calls in between, while the sequences shrink
    and grow: every replay has the bits of the eager call."""
    b = Batch(ops.Q4_0, [700 + 3 * i for i in range(9)], shared=512)
    few, lens = i32([3, 8]), torch.tensor(b.lens, dtype=torch.int32)
    new = lambda n, nq: (seeded_normal((n * nq, 24, 256), n), seeded_normal((n * nq, 24, 256), n + 1),
                         torch.empty((n * nq, 24, 256), dtype=torch.float16, device="cuda"))
    calls = [(*new(9, 1), None, 9, 1, 512), (*new(2, 5), few, 2, 5, 100)]
    work = torch.empty(max(ops.attn_batch_work_bytes(n, nq, sh, 768) for *_, n, nq, sh in calls), dtype=torch.uint8,
                       device="cuda")
    attend = lambda q, gate, out, seqs, n, nq, sh: ops.attn_decode_batch(q, gate, b.kv, b.kvt, b.pages, seqs, n, nq, sh, 768,
                                                                         out, work)
    graphs = []
    for c in calls:
        attend(*c)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            attend(*c)
    for cut in (0, 150, 699, 0, 40):
        b.pages.len.copy_((lens - cut).clamp_min(0))
        for c, graph in zip(calls, graphs):
            attend(*c)
            want = c[2].clone()
            c[2].fill_(7.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(c[2], want)
            c[0].mul_(-1)


def test_empty_sequences_inside_a_slice(gpu):
    """The last slice of the own positions has the end of the first sequence and, 1000 empty ones on, the only other one."""
    out = Batch(ops.Q8_0, [16384] + [0] * 999 + [50] + [0] * 23).check(1, 0, what="two of 1024")
    assert not out[1:1000].any() and not out[1001:].any()


def test_largest_batch(gpu):
    b = Batch(ops.Q8_0, [24 + i % 40 for i in range(1024)], shared=16, page=16)
    b.check(8, 16, what="1024 sequences, 8 queries")


@pytest.mark.parametrize("kvt", [ops.F16, ops.Q4_0], ids=lambda k: KV_NAMES[k])
def test_pools_past_32_bits(gpu, kvt):
    """Pages whose bytes lie more than 2^32 past the pool's and the KV head's beginning, in every operator."""
    page, slots = 64, (1 << 33) // (512 if kvt == ops.F16 else 128) // 2 + 4096
    b = Batch(kvt, [300, 280, 290, 100, 285, 270, 301], shared=256)
    small, table, n_pages = b.kv, b.pages.table.clone(), slots // page
    shift = n_pages - b.pages.ref.numel()
    b.kv = ops.KVLayer.allocate(kvt, slots, zero=False)
    for dst, src in ((b.kv.k, small.k), (b.kv.v, small.v), (b.kv.ks, small.ks), (b.kv.vs, small.vs)):
        if dst is not None:
            dst[:, shift * page:(shift + b.pages.ref.numel()) * page] = src[:, :b.pages.ref.numel() * page]
    b.pages = ops.KVPages.allocate(7, 320, n_pages, page)
    b.pages.table.copy_(torch.where(table >= 0, table + shift, table)[:, :1].expand(7, 5))
    b.pages.table[:, :table.shape[1]] = torch.where(table >= 0, table + shift, table)
    b.pages.len.copy_(i32(b.lens))
    held = torch.cat([b.pages.table[i, :-(-m // page)] for i, m in enumerate(b.lens)])
    b.pages.ref.index_add_(0, held.long(), torch.ones_like(held))
    b.check(1, 256, what="7 sequences at the end of a large pool")
    b.check(1, 0, seqs=[3, 0], what="two of them, nothing shared")
    # the same pages at the pool's beginning, then again with room for one position each
    work = torch.empty(ops.kv_pages_work_bytes(b.pages), dtype=torch.uint8, device="cuda")
    n_live, status = i32([0]), i32([9])
    ops.kv_pages_compact(b.pages, [b.kv], kvt, n_live, work)
    torch.cuda.synchronize()
    assert int(n_live) == int((b.pages.ref > 0).sum()) and int(b.pages.table.max()) == int(n_live) - 1
    b.check(1, 256, what="moved to its beginning")
    # a fork whose copied last page is the last of the pool
    b.pages.ref[int(n_live):n_pages - 1] = 1
    ops.kv_pages_trim(b.pages, i32([6]))
    free = (b.pages.ref == 0).nonzero().flatten().tolist()
    b.pages.ref[i32(free[:-1]).long()] = 1
    ops.kv_pages_fork(b.pages, i32([3]), i32([6]), work)
    ops.kv_pages_extend(b.pages, i32([6]), i32([1]), [b.kv], kvt, status, work)
    torch.cuda.synchronize()
    assert int(status) == 0 and int(b.pages.table[6, 1]) == n_pages - 1
    ops.kv_pages_trim(b.pages, i32([6]), i32([100]))
    b.lens[6], b.caches[6] = 100, b.caches[3]
    b._rows.clear()
    b.check(1, 0, seqs=[6, 3], what="a fork in its last page")
    # prep stores there
    x = lambda *s: seeded_normal(s, 91)
    ones, q = torch.ones(256, device="cuda"), torch.empty((1, 24, 256), device="cuda")
    k, v = x(1, 4, 256), x(1, 4, 256)
    ops.attn_prep_batch(x(1, 24, 512), k, v, ones, ones, b.pages, i32([6]), 1, 1, THETA, EPS, kvt, b.kv, q, q.clone())
    probe = ops.KVLayer.allocate(kvt, 1)
    ops.kv_append(k, v, 0, 1, kvt, probe)
    torch.cuda.synchronize()
    assert torch.equal(b.kv.v[:, (n_pages - 1) * page + 99 - 64], probe.v[:, 0])


# ---- prep -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nq", [1, 4, 8])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_prep_is_the_one_sequence_prep(gpu, kvt, nq):
    """Rows, queries and gates have the bits of attn_prep_multi on a contiguous cache, rotary offsets included; every
    other pool byte stays."""
    lens = [8, 100, 64, 65, 130]
    b = Batch(kvt, lens, page=32)
    n, seqs, off = 5, [3, 0, 4, 1, 2], [0, 5, -3, 100000, 7]
    qg, k, v = (seeded_normal(s, 40 + i) for i, s in enumerate([(n * nq, 24, 512), (n * nq, 4, 256), (n * nq, 4, 256)]))
    qn, kn = 1 + 0.1 * seeded_normal((256,), 50), 1 + 0.1 * seeded_normal((256,), 51)
    q, gate = torch.empty((n * nq, 24, 256), device="cuda"), torch.empty((n * nq, 24, 256), device="cuda")
    pool = [t for t in (b.kv.k, b.kv.v, b.kv.ks, b.kv.vs) if t is not None]
    want_pool = [t.clone() for t in pool]
    ops.attn_prep_batch(qg, k, v, qn, kn, b.pages, i32(seqs), n, nq, THETA, EPS, kvt, b.kv, q, gate, i32(off))
    q1, g1 = torch.empty((nq, 24, 256), device="cuda"), torch.empty((nq, 24, 256), device="cuda")
    for i, s in enumerate(seqs):
        r = slice(i * nq, (i + 1) * nq)
        src = [ops.RowSrc.device(t[r].contiguous(), w) for t, w in ((qg, 24 * 512), (k, 1024), (v, 1024))]
        p0, cache = lens[s] - nq, b.caches[s]
        ops.attn_prep_multi(*src, qn, kn, p0, p0 + off[i], nq, THETA, EPS, kvt, cache, q1, g1)
        torch.cuda.synchronize()
        assert torch.equal(q[r], q1) and torch.equal(gate[r], g1)
        at = torch.arange(p0, lens[s], device="cuda")
        slot = b.pages.table[s].long()[at // 32] * 32 + at % 32
        for w, c in zip(want_pool, [t for t in (cache.k, cache.v, cache.ks, cache.vs) if t is not None]):
            w[:, slot] = c[:, p0:lens[s]]
    for got, want in zip(pool, want_pool):
        assert torch.equal(got, want)


def test_prep_rows_without_a_place(gpu):
    """Unknown sequences, positions before the first and pages outside the pool: nothing is stored, q and gate are there; a
    sequence named twice gets the rows of the last."""
    nq, kvt = 3, ops.Q8_0
    b = Batch(kvt, [2, 64, 40, 0], page=16)
    b.pages.table[1, 3] = 1 << 30
    seqs = [1, -7, 0, 2, 9, 3, 2]
    n = len(seqs)
    qg, k, v = (seeded_normal(s, 60 + i) for i, s in enumerate([(n * nq, 24, 512), (n * nq, 4, 256), (n * nq, 4, 256)]))
    w = torch.ones(256, device="cuda")
    q, gate = (torch.full((n * nq, 24, 256), float("nan"), device="cuda") for _ in range(2))
    before = b.kv.v.clone()
    ops.attn_prep_batch(qg, k, v, w, w, b.pages, i32(seqs), n, nq, THETA, EPS, kvt, b.kv, q, gate)
    torch.cuda.synchronize()
    assert torch.isfinite(q).all() and torch.equal(gate, qg[..., 256:])
    probe = ops.KVLayer.allocate(kvt, n * nq)
    ops.kv_append(k, v, 0, n * nq, kvt, probe)
    want = before.clone()
    t0 = b.pages.table[0].tolist()
    want[:, t0[0] * 16:t0[0] * 16 + 2] = probe.v[:, 2 * nq + 1:2 * nq + 3]        # length 2: the last two of three
    t2 = b.pages.table[2].tolist()
    want[:, t2[2] * 16 + 5:t2[2] * 16 + 8] = probe.v[:, 6 * nq:7 * nq]            # named twice: the last
    torch.cuda.synchronize()
    assert torch.equal(b.kv.v, want)


# ---- a decode loop --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_decode_loop_of_forked_samples(gpu, kvt):
    """As a serving engine runs them: a prompt is stored, forked into samples, and every step makes room, appends and
    attends, captured once and replayed; after some steps the pool is compacted and the loop goes on.  Every step's output
    is that of the one-sequence decode on a contiguous cache per sample."""
    page, prompt, n, steps = 16, 41, 4, 9
    pages = ops.KVPages.allocate(n + 1, 96, 40, page)
    layers = [ops.KVLayer.allocate(kvt, 40 * page) for _ in range(2)]
    work = torch.empty(ops.kv_pages_work_bytes(pages), dtype=torch.uint8, device="cuda")
    status, n_live = i32([5]), i32([0])
    w = torch.ones(256, device="cuda")
    new = lambda *s: torch.empty(s, device="cuda")
    # the prompt, 7 positions at a time, as sequence n; an unrelated sequence in between scatters the pages
    qg, k, v = seeded_normal((prompt, 24, 512), 1), seeded_normal((prompt, 4, 256), 2), seeded_normal((prompt, 4, 256), 3)
    flat = [[ops.KVLayer.allocate(kvt, 96) for _ in layers] for _ in range(n)]
    for p0 in range(0, prompt, 7):
        m = min(7, prompt - p0)
        ops.kv_pages_extend(pages, i32([n, 0]), i32([m, 2]), layers, kvt, status, work)
        for li, kv in enumerate(layers):
            r = slice(p0, p0 + m)
            ops.attn_prep_batch(qg[r], k[r] + li, v[r], w, w, pages, i32([n]), 1, m, THETA, EPS, kvt, kv, new(m, 24, 256),
                                new(m, 24, 256))
            src = [ops.RowSrc.device(t, x) for t, x in ((qg[r], 24 * 512), (k[r] + li, 1024), (v[r], 1024))]
            for f in flat:
                ops.attn_prep_multi(*src, w, w, p0, p0, m, THETA, EPS, kvt, f[li], new(m, 24, 256), new(m, 24, 256))
                torch.cuda.synchronize()
    ops.kv_pages_trim(pages, i32([0]))
    samples = i32(list(range(n)))
    ops.kv_pages_fork(pages, i32([n] * n), samples, work)
    ops.kv_pages_trim(pages, i32([n]))                       # the samples hold the prompt now

    ones = i32([1] * n)
    QG, K, V = new(n, 24, 512), new(2, n, 4, 256), new(2, n, 4, 256)
    q, gate = new(2, n, 24, 256), new(2, n, 24, 256)
    out = torch.empty((2, n, 24, 256), dtype=torch.float16, device="cuda")
    scratch = torch.empty(ops.attn_batch_work_bytes(n, 1, 32, 96), dtype=torch.uint8, device="cuda")

    def step():
        ops.kv_pages_extend(pages, samples, ones, layers, kvt, status, work)
        for li, kv in enumerate(layers):
            ops.attn_prep_batch(QG, K[li], V[li], w, w, pages, samples, n, 1, THETA, EPS, kvt, kv, q[li], gate[li])
            ops.attn_decode_batch(q[li], gate[li], kv, kvt, pages, samples, n, 1, 32, 96, out[li], scratch)

    graph = None
    dec_work = torch.empty(ops.attn_work_bytes(96) // 4 + 1, device="cuda")
    want, wq, wg = new(1, 24, 256), new(1, 24, 256), new(1, 24, 256)
    for i in range(steps):
        QG.copy_(seeded_normal((n, 24, 512), 100 + i))
        K.copy_(seeded_normal((2, n, 4, 256), 200 + i))
        V.copy_(seeded_normal((2, n, 4, 256), 300 + i))
        if i == 0:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        else:
            graph.replay()
        torch.cuda.synchronize()
        assert int(status) == 0
        for b in range(n):
            for li in range(2):
                src = [ops.RowSrc.device(t[b], x) for t, x in ((QG, 24 * 512), (K[li], 1024), (V[li], 1024))]
                ops.attn_prep_multi(*src, w, w, prompt + i, prompt + i, 1, THETA, EPS, kvt, flat[b][li], wq, wg)
                ops.attn_decode(wq, wg, flat[b][li], kvt, prompt + i + 1, dec_work, want)
                torch.cuda.synchronize()
                assert torch.equal(wq[0], q[li, b])
                close(out[li, b], want[0], f"step {i} sample {b} layer {li}")
        if i == 4:
            ops.kv_pages_compact(pages, layers, kvt, n_live, work)
            torch.cuda.synchronize()
            assert int(n_live) == int((pages.ref > 0).sum())
    assert pages.len.tolist() == [prompt + steps] * n + [0]


@pytest.mark.parametrize("n, nq, shared", [(1, 1, 0), (3, 1, 128), (5, 1, 128), (9, 2, 128), (7, 8, 100), (33, 1, 130)])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_nothing_past_the_ends(gpu, kvt, n, nq, shared):
    """Output rows behind the batch, bytes behind the workspace's size and the pool stay as they were."""
    b = Batch(kvt, [shared + 10 + 31 * (i % 7) for i in range(n)], shared=shared)
    most = max(b.lens)
    need = ops.attn_batch_work_bytes(n, nq, shared, most)
    work = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
    out = torch.full((n * nq + 5, 24, 256), 7.0, dtype=torch.float16, device="cuda")
    oq = ops.ActQ8(torch.full(((n * nq + 5) * 6144,), 99, dtype=torch.int8, device="cuda"),
                   *(torch.full(((n * nq + 5) * 192,), 55.0, device="cuda") for _ in range(2)))
    pool = [t for t in (b.kv.k, b.kv.v, b.kv.ks, b.kv.vs) if t is not None]
    before = [t.clone() for t in pool]
    q, gate = seeded_normal((n * nq, 24, 256), 3), seeded_normal((n * nq, 24, 256), 4)
    ops.attn_decode_batch(q, gate, b.kv, kvt, b.pages, None, n, nq, shared, most, out, work, oq)
    torch.cuda.synchronize()
    assert (work[need:] == 0xAB).all() and (out[n * nq:] == 7.0).all()
    assert (oq.q[n * nq * 6144:] == 99).all() and (oq.d[n * nq * 192:] == 55).all() and (oq.s[n * nq * 192:] == 55).all()
    assert all(torch.equal(x, y) for x, y in zip(pool, before))
    want = batch_attention(q, gate, lambda t: b.values(t // nq), [b.lens[t // nq] - nq + t % nq + 1 for t in range(n * nq)])
    close(out[:n * nq], want, "the rows themselves")


def test_other_streams_and_work_on_them(gpu):
    """A call on a stream of its own, ordered by events, while another runs on the default stream with another work
    buffer."""
    b = Batch(ops.Q8_0, [500, 400, 300], shared=256)
    _, _, want = b.run(1, 256, 500)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _, _, a = b.run(1, 256, 500)
    _, _, c = b.run(1, 256, 500)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert torch.equal(a, want) and torch.equal(c, want)


def test_refusals_on_the_gpu(gpu):
    b = Batch(ops.Q8_0, [40])
    q = torch.zeros((1, 24, 256), device="cuda")
    out = torch.zeros((1, 24, 256), dtype=torch.float16, device="cuda")
    need = ops.attn_batch_work_bytes(1, 1, 0, 40)
    call = lambda work, out=out, q=q: ops.attn_decode_batch(q, q, b.kv, b.kvt, b.pages, None, 1, 1, 0, 40, out, work)
    with pytest.raises(ops.QwaError, match="workspace"):
        call(torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    with pytest.raises(ops.QwaError, match="out16"):
        call(work, out=q)
    with pytest.raises(ops.QwaError, match="contiguous"):
        call(work, q=torch.zeros((1, 24, 512), device="cuda")[..., :256])
    with pytest.raises(ops.QwaError, match="workspace"):
        ops.kv_pages_fork(b.pages, i32([0]), i32([0]), torch.empty(8, dtype=torch.uint8, device="cuda"))
    call(work)
    torch.cuda.synchronize()
