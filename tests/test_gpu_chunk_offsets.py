"""Offsets that run backwards, leave the buffers or name a sequence twice: every operator on chunks takes the same ones for chunks,
however many there are.  What counts is counted here one after the other: a chunk is not empty, lies inside the rows and does not
begin before the furthest end of the earlier ones that do."""
import random

import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from test_gpu_attn_batch import EPS, THETA, Batch, i32
from test_gpu_chunks import LSE, attention, close, prefill, prep_inputs, tables
from test_gpu_weights import log_sums, near, weights

pytestmark = pytest.mark.gpu


def live(off, rows):
    """(batch row, first row, end) of the chunks that count."""
    out, far = [], 0
    for b, (first, end) in enumerate(zip(off, off[1:])):
        if 0 <= first < end <= rows:
            if first >= far:
                out.append((b, first, end))
            far = max(far, end)
    return out


def last_of(chunks, seqs):
    """The chunks that are the last of their sequence."""
    return [c for i, c in enumerate(chunks) if seqs[c[0]] not in [seqs[x[0]] for x in chunks[i + 1:]]]


def some_offsets(n, rows, seed, most=6):
    """n + 1 offsets: mostly chunks of up to `most` tokens, between them ones that run back a little, empty ones far ahead behind
    an offset that is outside, and ends outside."""
    rng, off, at = random.Random(seed), [0], 0
    while len(off) < n + 1:
        x = rng.random()
        if x < 0.12 and at > 4:
            back = at - rng.randint(1, 4)
            off += [back, back + rng.randint(1, 2)]
        elif x < 0.2:
            ahead = min(rows, at + rng.randint(5, 40))
            off += [-1, ahead, ahead, at]
        elif x < 0.25:
            off += [rows + 1, at]
        at = min(rows, at + rng.randint(0, most))
        off.append(at)
    return off[:n + 1]


def prep(pages, kv, kvt, off, seqs, rows, data):
    for t in (kv.k, kv.v, kv.ks, kv.vs):
        if t is not None:
            t.view(torch.uint8).fill_(0x5A)
    qg, k, v, qn, kn = data
    q, gate = torch.full((rows, 24, 256), 7.0, device="cuda"), torch.full((rows, 24, 256), 7.0, device="cuda")
    for o, s in zip(off, seqs):
        ops.attn_prep_rows_batch(qg, k, v, qn, kn, pages, i32(s), i32(o), len(s), rows, THETA, EPS, kvt, kv, q, gate)
    torch.cuda.synchronize()
    return [t.clone() for t in (kv.k, kv.v, kv.ks, kv.vs) if t is not None], q, gate


def check_prep(kvt, off, seqs, rows, lens, page=16):
    """The call leaves what calls of one chunk each do: rows of every chunk that counts, K and V of the last of each sequence."""
    pages = tables(lens, page, sum(-(-m // page) for m in lens) + 2)
    kv, data = ops.KVLayer.allocate(kvt, pages.ref.numel() * page), prep_inputs(rows)
    chunks = live(off, rows)
    assert chunks
    _, q1, g1 = prep(pages, kv, kvt, [[a, e] for _, a, e in chunks], [[seqs[b]] for b, _, _ in chunks], rows, data)
    kept = last_of(chunks, seqs)
    want, _, _ = prep(pages, kv, kvt, [[a, e] for _, a, e in kept], [[seqs[b]] for b, _, _ in kept], rows, data)
    got, q, gate = prep(pages, kv, kvt, [off], [seqs], rows, data)
    assert torch.equal(q, q1) and torch.equal(gate, g1)
    for x, y in zip(got, want):
        assert torch.equal(x, y), f"stored rows differ: {off[:12]} {seqs[:12]}"


# a later chunk of the same sequence that overlaps; an empty one far ahead; one that is void because a void one reaches further
ODD = [([0, 20, 10, 15], [0, 0, 0]), ([30, 30, 5, 12], [1, 1, 1]), ([0, 10, 5, 25, 20, 30, 26, 31], [0, 1, 0, 2, 1, 2, 0]),
       ([0, 6, 9, 3, 8, 9, 14], [2, 0, 2, 0, 0, 2]), ([0, 8, -1, 25, 25, 8, 20], [0, 1, 1, 1, 1, 0])]


@pytest.mark.parametrize("off, seqs", ODD, ids=str)
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_prep_of_odd_offsets(gpu, kvt, off, seqs):
    check_prep(kvt, off, seqs, 32, [40, 33, 70])


@pytest.mark.parametrize("n", [40, 64, 65, 130, 513, 700, 1024])
def test_prep_of_many(gpu, n):
    """Sequences named several times: chunks on either side of a wave's 64, and of a workgroup's 512 threads."""
    rng = random.Random(n)
    for seed in range(3):
        seqs = [rng.randint(0, n // 3) for _ in range(n)]
        check_prep(ops.Q8_0, some_offsets(n, 3 * n, seed), seqs, 3 * n, [3 + (i * 5) % 40 for i in range(n // 3 + 1)])


def check_attention(b, off, seqs, rows, max_len):
    n, chunks = len(seqs), live(off, rows)
    q, gate, out, lse = prefill(b, off, n, rows, max_len, seqs)
    src, seen, at = [], [], []
    for i, a, e in chunks:
        m = min(b.lens[seqs[i]], max_len)
        src += [b.values(seqs[i])] * (e - a)
        seen += [m - (e - a) + t + 1 for t in range(e - a)]
        at += list(range(a, e))
    want, want_lse = attention(q[at], gate[at], lambda t: src[t], seen)
    close(out[at], want, f"{KV_NAMES[b.kvt]} {n} chunks, {len(chunks)} count")
    none = torch.isinf(want_lse)
    got = lse[at].double().cpu()
    assert torch.equal(torch.isinf(got), none) and (got[~none] - want_lse[~none]).abs().max().item() <= LSE
    rest = [r for r in range(rows) if r not in set(at)]
    assert (out[rest] == 7.0).all() and (lse[rest] == 7.0).all(), off


def check_weights(b, off, seqs, rows, max_len):
    n, chunks = len(seqs), live(off, rows)
    q = seeded_normal((rows, 24, 256), 5)
    lse = torch.full((rows, 24), float("nan"), device="cuda")
    before = seeded_normal((len(b.lens), 4, b.pages.table.shape[1] * b.page), 9).abs()
    want = before.double().cpu()
    for i, a, e in chunks:
        x, sums = log_sums(b, q[a:e], [seqs[i]], [e - a], max_len)
        lse[a:e] = x.float().cuda()
        if (i, a, e) in last_of(chunks, seqs):
            m = min(b.lens[seqs[i]], max_len)
            want[seqs[i], :, max(0, m - (e - a)):m] = 0.0
            want[seqs[i], :, :m] += sums[0]
    mass = before.clone()
    weights(b, q, lse, off, n, rows, max_len, mass, seqs)
    near(mass, want, f"{KV_NAMES[b.kvt]} {n} chunks, {len(chunks)} count")


@pytest.mark.parametrize("n", [0, 64, 65, 130, 1024])
@pytest.mark.parametrize("off, seqs", ODD, ids=str)
def test_odd_offsets(gpu, off, seqs, n):
    """Attention and weights, with as many empty chunks behind as make the wave's plan one of a workgroup; the prep's chunks
    (test_prep_of_odd_offsets) are the same."""
    b = Batch(ops.Q8_0, [40, 33, 70])
    more = max(0, n - len(seqs))
    off, seqs = off + [off[-1]] * more, seqs + [i % 3 for i in range(more)]
    check_attention(b, off, seqs, 32, 70)
    check_weights(b, off, seqs, 32, 70)


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_odd_offsets_of_many(gpu, kvt):
    """The same of up to 64 chunks, and more, of which those of one or two tokens are walked by themselves."""
    for n in (40, 64, 65, 130, 513):
        rng, rows = random.Random(n), 3 * n
        b = Batch(kvt, [3 + (i * 5) % 40 for i in range(n // 3 + 1)], page=16, ld=64)
        seqs = [rng.randint(0, n // 3) for _ in range(n)]
        off = some_offsets(n, rows, n)
        check_attention(b, off, seqs, rows, (1024, 40)[n % 2])
        check_weights(b, off, seqs, rows, 1024)
        off[:4] = [rows, rows, 0, 3]  # an empty chunk at the end of the buffers first
        check_attention(b, off, seqs, rows, 1024)
        check_weights(b, off, seqs, rows, 1024)
