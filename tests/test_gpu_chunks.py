"""Prep and attention of chunks (any number of new tokens a sequence) over a paged cache against their definitions in 64 bits,
and against the one-sequence operators on a contiguous cache.

Tolerances.  The output, V as stored (d * code) and the probabilities are rounded to fp16: at most half a step of 2^-11 relative
each, with a standard deviation of at most 2^-11 / sqrt(3).  The sum over the keys of p_j V_j e_j, with independent e_j, has
the norm sqrt(sum p^2 V^2) times that, and so has the output for independent V_j: a relative L2 of at most
sqrt(3) * 2^-11 / sqrt(3) = 4.9e-4.  An element whose terms cancel is off by more than half steps of itself: 2e-3, the bar of the
one-sequence operators (kvutil), and 3 * 2^-11 |out| where there are few keys.
The log sum's error is that of the scores: 256 products of fp32 accumulation, each sum rounded by at most 2^-24 of
sum |q_i k_i| / 16, about 256 * 0.64 / 16 = 10 for N(0,1): 256 * 2^-24 * 10 = 1.6e-4 at worst, and 2^-22 * 10 for the parts of Q."""
import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, MAX_ABS, seeded_normal
from test_gpu_attn_batch import EPS, THETA, Batch, i32

pytestmark = pytest.mark.gpu
REL, LSE = 5e-4, 2e-4


def offsets(counts):
    off = [0]
    for c in counts:
        off.append(off[-1] + c)
    return off


def close(got, want, what="", max_abs=MAX_ABS, rel_l2=REL):
    got, want = got.double().cpu(), want.double().cpu()
    assert torch.isfinite(got).all(), what
    d = (got - want).abs()
    rel = (d.norm() / want.norm().clamp_min(1e-30)).item()
    over = (d - 3 * 2.0**-11 * want.abs()).max().item() if d.numel() else 0.0
    print(f"{what}: max-abs {d.max().item() if d.numel() else 0:.2e}, rel-L2 {rel:.2e}", flush=True)
    assert over <= max_abs and rel <= rel_l2, f"{what}: {d.max().item():.3e}, rel-L2 {rel:.3e}"


def attention(q, gate, rows, seen):
    """q, gate [T][24][256] and, per token, K / V (rows(t): [4][m][256], 64 bits) of which it sees the first seen[t]: the outputs
    and log sums, 64 bits, on the CPU.  Neighbouring tokens of the same K are taken together."""
    q, gate = q.double().cpu(), gate.double().cpu()
    out, lse = torch.zeros(q.shape, dtype=torch.float64), torch.full(q.shape[:2], -torch.inf, dtype=torch.float64)
    t = 0
    while t < len(seen):
        K, V = rows(t)
        e = t + 1
        while e < len(seen) and rows(e)[0] is K:
            e += 1
        m = max([0] + [min(x, K.shape[1]) for x in seen[t:e]])
        if m > 0:
            hidden = torch.arange(m) >= torch.tensor(seen[t:e])[:, None, None]
            for g in range(4):
                s = (q[t:e, 6 * g:6 * g + 6] @ K[g, :m].T / 16.0).masked_fill(hidden, -torch.inf)
                x = torch.logsumexp(s, -1)
                lse[t:e, 6 * g:6 * g + 6] = x
                out[t:e, 6 * g:6 * g + 6] = torch.where(torch.isfinite(x)[..., None], torch.softmax(s, -1), 0.0) @ V[g, :m]
        t = e
    return out * torch.sigmoid(gate), lse


def prefill(b, off, n, rows, max_len, seqs=None, seed=77, lse=True, q=None, gate=None, work=None):
    q = seeded_normal((rows, 24, 256), seed) if q is None else q
    gate = seeded_normal((rows, 24, 256), seed + 1) if gate is None else gate
    out = torch.full((rows, 24, 256), 7.0, dtype=torch.float16, device="cuda")
    lse = torch.full((rows, 24), 7.0, device="cuda") if lse else None
    if work is None:
        work = torch.full((ops.attn_prefill_batch_work_bytes(n, rows, max_len),), 0xFF, dtype=torch.uint8, device="cuda")
    ops.attn_prefill_batch(q, gate, b.kv, b.kvt, b.pages, None if seqs is None else i32(seqs), i32(off), n, rows, max_len, out,
                           work, lse=lse)
    torch.cuda.synchronize()
    return q, gate, out, lse


def check(b, counts, seqs=None, pad=0, max_len=None, what="", **kw):
    """The chunks of the last counts[i] tokens of sequence seqs[i] against the definition."""
    off, n, n_seq = offsets(counts), len(counts), len(b.lens)
    max_len, order = max_len or max(b.lens), list(range(n_seq)) if seqs is None else seqs
    rows = off[-1] + pad
    q, gate, out, lse = prefill(b, off, n, rows, max_len, seqs, **kw)
    empty = (torch.zeros((4, 0, 256), dtype=torch.float64),) * 2
    src, seen = [], []
    for i, c in enumerate(counts):
        known = 0 <= order[i] < n_seq
        m = min(b.lens[order[i]], max_len) if known else 0
        src += [b.values(order[i]) if known else empty] * c
        seen += [m - c + t + 1 for t in range(c)]
    T = off[-1]
    want, want_lse = attention(q[:T], gate[:T], lambda t: src[t], seen)
    what = what or f"{KV_NAMES[b.kvt]} {b.lens} chunks {counts}"
    close(out[:T], want, what)
    assert (out[T:] == 7.0).all()
    if lse is not None:
        none = torch.isinf(want_lse)
        got = lse[:T].double().cpu()
        assert torch.equal(torch.isinf(got), none) and (got[none] < 0).all()
        err = (got[~none] - want_lse[~none]).abs()
        assert err.numel() == 0 or err.max().item() <= LSE, f"{what}: log sums off by {err.max().item():.2e}"
        assert (lse[T:] == 7.0).all()
    return out, lse


SIZES = [
    # a chunk alone: one token, row blocks of 128 rows that end inside a token (21, 22, 43), lengths around a tile
    ([1], [1], 16), ([31], [31], 16), ([32], [32], 32), ([33], [33], 64), ([65], [1], 64), ([300], [21], 16), ([300], [22], 64),
    ([64], [43], 128), ([700], [333], 256), ([2100], [5], 1024),
    # together: ragged lengths and chunks, an empty chunk, a sequence of fewer positions than its chunk has tokens
    ([40, 1, 513, 96], [40, 1, 300, 7], 16), ([100, 90, 80], [100, 0, 1], 32), ([5, 129, 0], [9, 30, 2], 64),
    ([1000, 1001, 64, 63, 62], [1, 1, 64, 1, 1], 64),
]


@pytest.mark.parametrize("lens, counts, page", SIZES, ids=lambda v: str(v).replace(" ", "") if isinstance(v, list) else v)
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_attention(gpu, kvt, lens, counts, page):
    b = Batch(kvt, lens, page=page)
    out, lse = check(b, counts, pad=5)
    # without the log sums: the same bits
    assert torch.equal(check(b, counts, pad=5, lse=False)[0], out)


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_sequences_named(gpu, kvt):
    """Any order, a sequence twice (each chunk by itself), unknown ones (zeros), a bound below a length."""
    b = Batch(kvt, [200, 77, 410, 0, 33])
    check(b, [3, 50, 1, 20, 4, 0, 2], seqs=[2, 0, -1, 2, 9, 1, 3], pad=1)
    check(b, [30, 3, 40], seqs=[2, 4, 0], max_len=128)


def test_shared_pages_and_many_chunks(gpu):
    """Forks of a prompt whose pages several sequences hold; as many chunks as a call takes."""
    b = Batch(ops.Q8_0, [300, 280, 260, 300], shared=192)
    check(b, [90, 1, 3, 41])
    b = Batch(ops.Q4_0, [17 + i % 40 for i in range(1024)], page=16)
    check(b, [(i * 7) % 3 for i in range(1024)])


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_rows_of_no_chunk(gpu, kvt):
    """Rows before the first chunk and between chunks stay; a chunk that overlaps an earlier one, runs backwards or leaves the
    buffers counts as empty."""
    b = Batch(kvt, [100, 200, 300])
    for off, real in (([2, 10, 10, 30], [(0, 2, 10), (2, 10, 30)]), ([0, 20, 10, 15], [(0, 0, 20)]),
                      ([-3, 4, 9, 1 << 30], [(1, 4, 9)]), ([0, 41, 1, 2], [(2, 1, 2)])):
        rows = 40
        q, gate, out, lse = prefill(b, off, 3, rows, 300)
        src, seen, at = [], [], []
        for s, a, e in real:
            src += [b.values(s)] * (e - a)
            seen += [b.lens[s] - (e - a) + t + 1 for t in range(e - a)]
            at += list(range(a, e))
        want, want_lse = attention(q[at], gate[at], lambda t: src[t], seen)
        close(out[at], want, f"{off}")
        rest = [r for r in range(rows) if r not in at]
        assert (out[rest] == 7.0).all() and (lse[rest] == 7.0).all(), off


def test_long_context(gpu):
    """A decoded token and a chunk of 100 at 40000 positions beside short ones: blocks of several slices."""
    b = Batch(ops.Q4_0, [40000, 300, 39000, 2], page=256)
    check(b, [1, 40, 100, 1])


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_outlier_keys(gpu, kvt):
    """1% of the keys eight times as large: scores are exact, so the error stays that of the roundings."""
    b = Batch(kvt, [900, 400])
    for s in range(2):
        c = b.caches[s]
        at = torch.arange(0, b.lens[s], 97, device="cuda")
        K = 8.0 * seeded_normal((len(at), 4, 256), 900 + s)
        for r, j in enumerate(at.tolist()):
            ops.kv_append(K[r:r + 1].contiguous(), None, j, 1, kvt, c)
        torch.cuda.synchronize()
        slot = b.pages.table[s].long()[at // b.page] * b.page + at % b.page
        b.kv.k[:, slot] = c.k[:, at]
        if c.ks is not None:
            b.kv.ks[:, slot] = c.ks[:, at]
    check(b, [200, 5], lse=False)


def test_scores_of_a_million(gpu):
    """Scores far apart and huge: a row's states of several slices weigh the same to the last bit; one key takes all."""
    b = Batch(ops.F16, [5000])
    q = 3000.0 * seeded_normal((8, 24, 256), 3)
    check(b, [8], q=q, lse=False)


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_not_finite(gpu, kvt):
    """A V value that is not finite, and K likewise, shows in the rows that see it and in no other; one of a hidden position
    nowhere."""
    b = Batch(kvt, [150, 150])
    counts, off = [60, 60], offsets([60, 60])
    q, gate, clean, clean_lse = prefill(b, off, 2, 120, 150)
    bad = 120  # a position inside the chunk: tokens from 30 on see it
    slot = int(b.pages.table[0, bad // b.page]) * b.page + bad % b.page
    nan = 0x7E00
    keep = b.kv.v[1, slot].clone(), None if b.kv.vs is None else b.kv.vs[1, slot].clone()
    if kvt == ops.F16:
        b.kv.v[1, slot].view(torch.int16)[5] = nan
        dims = [5]
    else:
        b.kv.vs[1, slot, 2] = nan
        dims = list(range(64, 96))
    _, _, out, _ = prefill(b, off, 2, 120, 150, q=q, gate=gate)
    mark = torch.zeros((120, 24, 256), dtype=torch.bool, device="cuda")
    for d in dims:
        mark[30:60, 6:12, d] = True
    assert not torch.isfinite(out[mark]).any()
    assert torch.equal(out[~mark], clean[~mark])
    b.kv.v[1, slot] = keep[0]
    if keep[1] is not None:
        b.kv.vs[1, slot] = keep[1]
    # K
    if kvt == ops.F16:
        b.kv.k[2, slot].view(torch.int16)[200] = nan
    else:
        b.kv.ks[2, slot, 6] = nan
    _, _, out, lse = prefill(b, off, 2, 120, 150, q=q, gate=gate)
    mark[:] = False
    mark[30:60, 12:18] = True
    assert torch.isnan(out[mark]).all() and torch.isnan(lse[30:60, 12:18]).all()
    assert torch.equal(out[~mark], clean[~mark])


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_pages_outside_the_pool(gpu, kvt):
    """Positions of a page that is none of the pool's are not seen."""
    b = Batch(kvt, [400, 64], page=32)
    for e, bad in ((2, -1), (7, 1 << 30)):
        b.pages.table[0, e] = bad
    q, gate, out, lse = prefill(b, [0, 50, 53], 2, 53, 400)
    gone = torch.zeros(400, dtype=torch.bool)
    gone[64:96] = True
    gone[224:256] = True
    K, V = b.values(0)
    K, V, kept = K[:, ~gone], V[:, ~gone], (~gone).cumsum(0)
    want, want_lse = attention(q[:50], gate[:50], lambda t: (K, V), [int(kept[350 + t]) for t in range(50)])
    close(out[:50], want, "holes")
    assert (lse[:50].double().cpu() - want_lse).abs().max() <= LSE


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_images_of_odd_keys(gpu, kvt):
    """Both of the above for a chunk of many blocks, whose keys are brought into LDS's form once."""
    b, n = Batch(kvt, [700], page=32), 300
    q, gate, clean, _ = prefill(b, [0, n], 1, n, 700)
    bad = 600  # tokens from 200 on see it
    slot = int(b.pages.table[0, bad // b.page]) * b.page + bad % b.page
    keep = [None if x is None else x[1, slot].clone() for x in (b.kv.v, b.kv.vs, b.kv.k, b.kv.ks)]
    mark = torch.zeros((n, 24, 256), dtype=torch.bool, device="cuda")
    for values, scales, what in ((b.kv.v, b.kv.vs, "v"), (b.kv.k, b.kv.ks, "k")):
        if kvt == ops.F16:
            values[1, slot].view(torch.int16)[5] = 0x7E00
            dims = [5]
        else:
            scales[1, slot, 2] = 0x7E00
            dims = list(range(64, 96))
        _, _, out, lse = prefill(b, [0, n], 1, n, 700, q=q, gate=gate)
        mark[:] = False
        mark[200:, 6:12, dims if what == "v" else slice(None)] = True
        assert torch.isnan(out[mark]).all() and torch.equal(out[~mark], clean[~mark])
        assert torch.isnan(lse[200:, 6:12]).all() == (what == "k") and torch.isfinite(lse[:200]).all()
        for x, y in zip((b.kv.v, b.kv.vs, b.kv.k, b.kv.ks), keep):
            if x is not None:
                x[1, slot] = y
    for e, none in ((2, -1), (7, 1 << 30), (21, b.pages.ref.numel())):
        b.pages.table[0, e] = none
    _, _, out, lse = prefill(b, [0, n], 1, n, 700, q=q, gate=gate)
    gone = torch.zeros(700, dtype=torch.bool)
    gone[64:96] = gone[224:256] = gone[672:] = True
    K, V = b.values(0)
    K, V, kept = K[:, ~gone], V[:, ~gone], (~gone).cumsum(0)
    want, want_lse = attention(q, gate, lambda t: (K, V), [int(kept[400 + t]) for t in range(n)])
    close(out, want, "holes")
    assert (lse.double().cpu() - want_lse).abs().max() <= LSE


def test_repeated_calls_streams_and_graphs(gpu):
    """The same bits again, on another stream beside it, and from a captured graph that follows the device's numbers."""
    kvt, n, rows = ops.Q8_0, 3, 200
    b = Batch(kvt, [900, 350, 64], ld=1024)
    counts = [100, 1, 64]
    q, gate = seeded_normal((rows, 24, 256), 1), seeded_normal((rows, 24, 256), 2)
    off, size = i32(offsets(counts)), ops.attn_prefill_batch_work_bytes(n, rows, 1000)
    new = lambda: (torch.zeros((rows, 24, 256), dtype=torch.float16, device="cuda"), torch.zeros((rows, 24), device="cuda"),
                   torch.empty(size, dtype=torch.uint8, device="cuda"))

    def call(o, stream=None):
        ops.attn_prefill_batch(q, gate, b.kv, kvt, b.pages, None, off, n, rows, 1000, o[0], o[2], lse=o[1], stream=stream)

    first, second, third = new(), new(), new()
    call(first)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        call(second, streams[0])
        call(third, streams[1])
    torch.cuda.synchronize()
    for o in (second, third):
        assert torch.equal(o[0], first[0]) and torch.equal(o[1], first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(second)
    for lens, cs in (([900, 350, 64], counts), ([200, 350, 10], [7, 100, 10]), ([0, 1, 64], [0, 1, 40])):
        off.copy_(i32(offsets(cs)))
        b.pages.len.copy_(i32(lens))
        for o in (second, third):
            o[0].zero_()
            o[1].zero_()
        graph.replay()
        torch.cuda.synchronize()
        call(third)
        torch.cuda.synchronize()
        assert torch.equal(second[0], third[0]) and torch.equal(second[1], third[1])
        assert bool(third[0].abs().sum() > 0)


def test_offsets_past_32_bits(gpu):
    """A pool whose rows lie past 4 GiB of their head's, and heads past 8 GiB: the last pages of it."""
    kvt, page = ops.F16, 1024
    small = Batch(kvt, [3000], page=page)
    n_pages = 8400  # 8.6 million positions: 4.4 GB a head, 17.6 GB for K and V each
    kv = ops.KVLayer.allocate(kvt, n_pages * page)
    pages = ops.KVPages.allocate(1, 3 * page, n_pages, page)
    last = [n_pages - 1, n_pages - 3, n_pages - 2]
    pages.table[0, :3] = i32(last)
    pages.len.fill_(3000)
    for e, pg in enumerate(last):
        old = int(small.pages.table[0, e])
        for dst, src in ((kv.k, small.kv.k), (kv.v, small.kv.v)):
            dst[:, pg * page:(pg + 1) * page] = src[:, old * page:(old + 1) * page]
    _, _, want, want_lse = prefill(small, [0, 70], 1, 70, 3000)
    small.kv, small.pages = kv, pages
    _, _, out, lse = prefill(small, [0, 70], 1, 70, 3000)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)


# ---- prep
def prep_inputs(rows, seed=31):
    return (seeded_normal((rows, 24, 512), seed), seeded_normal((rows, 4, 256), seed + 1), seeded_normal((rows, 4, 256), seed + 2),
            1 + 0.1 * seeded_normal((256,), seed + 3), 1 + 0.1 * seeded_normal((256,), seed + 4))


def tables(lens, page, n_pages, seed=9):
    pages = ops.KVPages.allocate(len(lens), max(max(lens), 1), n_pages, page)
    perm, at = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist(), 0
    for i, m in enumerate(lens):
        k = -(-m // page)
        if k:
            pages.table[i, :k] = i32(perm[at:at + k])
        at += k
    pages.len.copy_(i32(lens))
    return pages


@pytest.mark.parametrize("counts, lens, page", [([1], [1], 16), ([20, 17], [320, 17], 64), ([3, 0, 130, 1], [3, 9, 400, 33], 128)])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_prep(gpu, kvt, counts, lens, page):
    """Bits of attn_prep_multi on contiguous caches; no other byte of the pool, q and gate changes."""
    off, n, pad = offsets(counts), len(counts), 3
    T, rows = off[-1], off[-1] + pad
    qg, k, v, qn, kn = prep_inputs(rows)
    pages = tables(lens, page, sum(-(-m // page) for m in lens) + 2)
    kv = ops.KVLayer.allocate(kvt, pages.ref.numel() * page + 7)
    bufs = [t for t in (kv.k, kv.v, kv.ks, kv.vs) if t is not None]
    for t in bufs:
        t.view(torch.uint8).fill_(0x5A)
    want = [t.clone() for t in bufs]
    q, gate = torch.full((rows, 24, 256), 7.0, device="cuda"), torch.full((rows, 24, 256), 7.0, device="cuda")
    turn = i32([5 * i for i in range(n)])
    ops.attn_prep_rows_batch(qg, k, v, qn, kn, pages, None, i32(off), n, rows, THETA, EPS, kvt, kv, q, gate, rope_off=turn)
    torch.cuda.synchronize()
    for b, c in enumerate(counts):
        if c == 0:
            continue
        flat = ops.KVLayer.allocate(kvt, lens[b])
        r = slice(off[b], off[b + 1])
        src = [ops.RowSrc.device(t[r].contiguous(), x) for t, x in ((qg, 24 * 512), (k, 1024), (v, 1024))]
        q1, g1 = torch.empty((c, 24, 256), device="cuda"), torch.empty((c, 24, 256), device="cuda")
        p0 = lens[b] - c
        ops.attn_prep_multi(*src, qn, kn, p0, p0 + 5 * b, c, THETA, EPS, kvt, flat, q1, g1)
        torch.cuda.synchronize()
        assert torch.equal(q[r], q1) and torch.equal(gate[r], g1)
        at = torch.arange(p0, lens[b], device="cuda")
        slot = pages.table[b].long()[at // page] * page + at % page
        for w, f in zip(want, [t for t in (flat.k, flat.v, flat.ks, flat.vs) if t is not None]):
            w[:, slot] = f[:, at]
    assert (q[T:] == 7.0).all() and (gate[T:] == 7.0).all()
    for t, w in zip(bufs, want):
        assert torch.equal(t, w)


def test_prep_of_odd_requests(gpu):
    """Rows before the first position, of unknown sequences and in foreign pages are not stored; of two chunks of a sequence the
    later one is; chunks that overlap, run backwards or leave the buffers are nobody's."""
    kvt, page = ops.Q8_0, 32
    pages = tables([70, 4, 50], page, 9)
    pages.table[2, 0] = 1 << 20
    kv = ops.KVLayer.allocate(kvt, 9 * page)

    def run(off, seqs, rows=30):
        for t in (kv.k, kv.v, kv.ks, kv.vs):
            t.view(torch.uint8).fill_(0x5A)
        qg, k, v, qn, kn = prep_inputs(rows)
        q, gate = torch.full((rows, 24, 256), 7.0, device="cuda"), torch.full((rows, 24, 256), 7.0, device="cuda")
        ops.attn_prep_rows_batch(qg, k, v, qn, kn, pages, i32(seqs), i32(off), len(seqs), rows, THETA, EPS, kvt, kv, q, gate)
        torch.cuda.synchronize()
        changed = (kv.v.view(torch.uint8) != 0x5A).any(-1).any(0).nonzero()[:, 0].tolist()
        return (q != 7.0).any(-1).any(-1).nonzero()[:, 0].tolist(), set(changed)

    slot = lambda s, j: int(pages.table[s, j // page]) * page + j % page
    # 6 tokens for 4 positions; an unknown sequence; positions 30, 31 of a foreign page, 32 .. 49 of the pool's
    rows, stored = run([0, 6, 8, 28], [1, 7, 2])
    assert rows == list(range(28)) and stored == {slot(1, j) for j in range(4)} | {slot(2, j) for j in range(32, 50)}
    # the later chunk of sequence 0 counts, an empty one behind it does not
    rows, stored = run([0, 10, 13, 13], [0, 0, 0])
    assert rows == list(range(13)) and stored == {slot(0, j) for j in range(67, 70)}
    for off, real in (([0, 20, 10, 15], range(20)), ([-3, 4, 9, 1 << 30], range(4, 9)), ([2, 31, 1, 3], range(1, 3))):
        assert run(off, [0, 0, 0])[0] == list(real)


# ---- together
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_prompts_through_pages(gpu, kvt):
    """As an engine serves: room, prep and attention of ragged chunks beside decoded tokens, a fork that goes on with chunks of
    its own; cache rows have the bits of contiguous caches, attention is that of the one-sequence prefill."""
    page, n_pages, ld = 16, 90, 512
    pages = ops.KVPages.allocate(4, ld, n_pages, page)
    kv = ops.KVLayer.allocate(kvt, n_pages * page)
    work = torch.empty(ops.kv_pages_work_bytes(pages), dtype=torch.uint8, device="cuda")
    status = i32([9])
    flats = [ops.KVLayer.allocate(kvt, ld) for _ in range(4)]
    lens = [0] * 4
    w = 1 + 0.1 * seeded_normal((256,), 7)
    ops.attn_prefill_reserve(256, ld)
    seed = 100
    steps = [([0, 1], [150, 33]), ([0, 2, 1], [1, 70, 5]), ("fork", 0, 3), ([3, 0, 2], [64, 1, 40]), ([1, 3], [1, 1])]
    for step in steps:
        if step[0] == "fork":
            ops.kv_pages_fork(pages, i32([step[1]]), i32([step[2]]), work)
            lens[step[2]] = lens[step[1]]
            for dst, src in zip((flats[step[2]].k, flats[step[2]].v, flats[step[2]].ks, flats[step[2]].vs),
                                (flats[step[1]].k, flats[step[1]].v, flats[step[1]].ks, flats[step[1]].vs)):
                if dst is not None:
                    dst.copy_(src)
            continue
        seqs, counts = step
        seed += 10
        n, off = len(seqs), offsets(counts)
        rows = off[-1] + 2
        ops.kv_pages_extend(pages, i32(seqs), i32(counts), [kv], kvt, status, work)
        qg, k, v = seeded_normal((rows, 24, 512), seed), seeded_normal((rows, 4, 256), seed + 1), seeded_normal((rows, 4, 256), seed + 2)
        q, gate = torch.zeros((rows, 24, 256), device="cuda"), torch.zeros((rows, 24, 256), device="cuda")
        out = torch.zeros((rows, 24, 256), dtype=torch.float16, device="cuda")
        scratch = torch.empty(ops.attn_prefill_batch_work_bytes(n, rows, ld), dtype=torch.uint8, device="cuda")
        ops.attn_prep_rows_batch(qg, k, v, w, w, pages, i32(seqs), i32(off), n, rows, THETA, EPS, kvt, kv, q, gate)
        ops.attn_prefill_batch(q, gate, kv, kvt, pages, i32(seqs), i32(off), n, rows, ld, out, scratch)
        torch.cuda.synchronize()
        assert int(status) == 0
        for i, (s, c) in enumerate(zip(seqs, counts)):
            r, p0 = slice(off[i], off[i + 1]), lens[s]
            rope, q1, g1 = torch.empty((c, 64), device="cuda"), torch.empty((c, 24, 256), device="cuda"), torch.empty((c, 24, 256), device="cuda")
            want = torch.empty((c, 24, 256), dtype=torch.float16, device="cuda")
            ops.rope_table(p0, c, THETA, rope)
            ops.attn_prep_rows(qg[r].contiguous(), k[r].contiguous(), v[r].contiguous(), w, w, c, p0, rope, EPS, kvt, flats[s], q1, g1)
            ops.attn_prefill(q1, g1, flats[s], kvt, c, p0, want)
            torch.cuda.synchronize()
            assert torch.equal(q1, q[r]) and torch.equal(g1, gate[r])
            # (the one-sequence prefill rounds Q / 16 and d * code to fp16: 1e-3 of its own)
            close(out[r], want, f"sequence {s}", rel_l2=1.5e-3)
            lens[s] += c
            at = torch.arange(lens[s], device="cuda")
            slot = pages.table[s].long()[at // page] * page + at % page
            for a, f in ((kv.k, flats[s].k), (kv.v, flats[s].v), (kv.ks, flats[s].ks), (kv.vs, flats[s].vs)):
                if a is not None:
                    assert torch.equal(a[:, slot], f[:, :lens[s]])
