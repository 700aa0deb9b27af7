"""Offsets that run backwards, leave the buffers or name a sequence twice: every operator on chunks takes the same ones for chunks,
however many there are.  What counts is counted here one after the other: a chunk is not empty, lies inside the rows and does not
begin before the furthest end of the earlier ones that do."""
import random

import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES
from test_gpu_attn_batch import EPS, THETA, i32
from test_gpu_chunks import prep_inputs, tables

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
