"""The weights where their plan is made by a workgroup, and what they leave as it is.  Definition and tolerances as in
test_gpu_weights."""
import random

import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from test_gpu_attn_batch import EPS, THETA, Batch, i32
from test_gpu_chunks import offsets
from test_gpu_weights import check, near, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [2, 70])
@pytest.mark.parametrize("tokens", [3, 40, 50, 130])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_own_positions_without_a_place(gpu, kvt, tokens, n):
    """A chunk's own positions in a foreign page are seen by no token: their weights stay, as those of older ones do.  Chunks of one
    wave's rows, of one block and of several, by both plans."""
    b = Batch(kvt, [400, 64], page=32)
    rows, lse0 = tokens + 3, 8.0
    off = offsets([tokens, 3]) + [rows] * (n - 2)
    q, lse = seeded_normal((rows, 24, 256), 3), torch.full((rows, 24), lse0, device="cuda")
    gone = [torch.zeros(400, dtype=torch.bool), torch.zeros(64, dtype=torch.bool)]
    for s, e in ((0, 2), (0, 11), (0, 12), (1, 1)):  # positions 64 .. 95, 352 .. 399 of sequence 0, 32 .. 63 of 1
        b.pages.table[s, e] = -1 if e != 11 else b.pages.ref.numel()
        gone[s][32 * e:32 * (e + 1)] = True
    before = seeded_normal((2, 4, b.pages.table.shape[1] * 32), 9)
    before[:, :, ::7] = -0.0
    mass, want = before.clone(), before.double().cpu()
    weights(b, q, lse, off, n, rows, 400, mass, [0, 1] + [0] * (n - 2))
    for s, (m, c) in enumerate(((400, tokens), (64, 3))):
        x = q[off[s]:off[s + 1]].double().cpu().view(c, 4, 6, 256)
        p = torch.exp(torch.einsum("tghd,gjd->tghj", x, b.values(s)[0]) / 16.0 - lse0)
        p = p.masked_fill((torch.arange(m) > (m - c + torch.arange(c))[:, None])[:, None, None], 0.0).sum((0, 2))
        old = want[s, :, :m].clone()
        old[:, m - c:] = 0.0
        want[s, :, :m] = torch.where(gone[s], want[s, :, :m], old + p)
    left = torch.ones(mass.shape, dtype=torch.bool)
    for s, m in ((0, 400), (1, 64)):
        left[s, :, :m] = gone[s]
    assert torch.equal(mass.cpu()[left].view(torch.int32), before.cpu()[left].view(torch.int32))
    near(mass, want, f"{KV_NAMES[kvt]} {tokens} tokens")


@pytest.mark.parametrize("n", [63, 64, 65, 128, 129, 700])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_numbers_of_chunks(gpu, kvt, n):
    """Up to 64 chunks by a wave, 128 by two, more by a workgroup of 1024: chunks of none to 30 tokens, and between them some of
    several blocks (43 tokens and up), whose sums are joined; sequences named twice, of which the last chunk with tokens counts."""
    rng = random.Random(n)
    counts = [rng.choice((0, 1, 2, rng.randint(3, 30))) for _ in range(n)]
    for i, c in zip(rng.sample(range(n), 6), (42, 43, 85, 86, 130, 200)):
        counts[i] = c
    lens = [max(1, (i * 53) % 640) for i in range(n - n // 8)]
    seqs = list(range(len(lens))) + rng.sample(range(len(lens)), n // 8)
    rng.shuffle(seqs)
    last = {s: i for i, s in enumerate(seqs) if counts[i] > 0}
    check(Batch(kvt, lens, page=32), counts, seqs=seqs, pad=2, counted=set(last.values()))


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_few_chunks_of_many_blocks(gpu, kvt):
    """More than 64 blocks of a few chunks, one of which is longer than its sequence, and one of one block."""
    check(Batch(kvt, [1200, 700, 900, 333]), [1000, 800, 900, 40], pad=1)
    check(Batch(kvt, [1200, 700, 900, 333]), [1000, 800, 900, 40], seqs=[0, 1, 0, 3], counted=[1, 2, 3])


def test_window_of_a_step_behind_an_eviction(gpu):
    """The weights of a step's last tokens alone, on entries that an eviction has left: those at and past the lengths are cleared
    before the step, as the header asks for; then the new positions gather from the window's tokens and nothing else."""
    kvt, L, ld, page = ops.Q8_0, 2, 1024, 64
    pages = ops.KVPages.allocate(2, ld, 40, page)
    kvs = [ops.KVLayer.allocate(kvt, 40 * page) for _ in range(L)]
    room, status = torch.empty(ops.kv_pages_work_bytes(pages), dtype=torch.uint8, device="cuda"), i32([9])
    mass, turn = torch.zeros((L, 2, 4, ld), device="cuda"), i32([0, 0])
    w, j = 1 + 0.1 * seeded_normal((256,), 7), torch.arange(ld, device="cuda")

    def step(counts, window, seed):
        off, rows = offsets(counts), sum(counts)
        late = [max(a, e - window) for a, e in zip(off, off[1:])]
        ops.kv_pages_extend(pages, i32([0, 1]), i32(counts), kvs, kvt, status, room)
        scratch = torch.empty(ops.attn_prefill_batch_work_bytes(2, rows, ld), dtype=torch.uint8, device="cuda")
        before, alone = mass.clone(), torch.zeros_like(mass)
        for l in range(L):
            qg, k, v = (seeded_normal((rows, *x), seed + 10 * l + i) for i, x in enumerate(((24, 512), (4, 256), (4, 256))))
            q, gate = torch.empty((rows, 24, 256), device="cuda"), torch.empty((rows, 24, 256), device="cuda")
            out, lse = torch.empty((rows, 24, 256), dtype=torch.float16, device="cuda"), torch.empty((rows, 24), device="cuda")
            ops.attn_prep_rows_batch(qg, k, v, w, w, pages, None, i32(off), 2, rows, THETA, EPS, kvt, kvs[l], q, gate, rope_off=turn)
            ops.attn_prefill_batch(q, gate, kvs[l], kvt, pages, None, i32(off), 2, rows, ld, out, scratch, lse=lse)
            for m in (mass, alone):
                # (the rows between the windows: a chunk of no sequence)
                extra = torch.empty(ops.attn_weights_batch_work_bytes(3, rows, ld), dtype=torch.uint8, device="cuda")
                ops.attn_weights_batch(q, lse, kvs[l], kvt, pages, i32([0, -1, 1]), i32([late[0], off[1], late[1], off[2]]), 3, rows, ld,
                                       m[l], extra)
        torch.cuda.synchronize()
        assert int(status) == 0
        return before, alone, [min(window, c) for c in counts]

    step([700, 400], 1000, 100)
    dropped = i32([0, 0])
    work = torch.empty(ops.kv_pages_evict_work_bytes(pages, 2, L, 200), dtype=torch.uint8, device="cuda")
    ops.kv_pages_evict(pages, i32([0, 1]), i32([200, 150]), 20, 200, kvs, kvt, mass, dropped, status, work)
    turn += dropped
    assert int(status) == 0 and (mass[:, 0, :, 200:700] > 0).all()  # what was there is left
    mass.masked_fill_(j >= pages.len[:, None, None], 0.0)
    before, alone, windows = step([90, 33], 16, 200)
    lens = pages.len.tolist()
    assert lens == [290, 183]
    near(mass, before.double() + alone.double(), "windows")
    for s, (m, x, old) in enumerate(zip(lens, windows, (200, 150))):
        assert (mass[:, s, :, old:m] <= 6.0 * x + 0.01).all() and (mass[:, s, :, m:] == 0).all()
        total = (mass.double() - before.double())[:, s].sum(-1)
        assert ((total - 6.0 * x).abs() <= 4e-4 * 6 * x + 2.0**-20 * before[:, s].double().sum(-1)).all()
