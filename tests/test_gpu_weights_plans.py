"""The weights where their plan is made by a workgroup, and what they leave as it is.  Definition and tolerances as in
test_gpu_weights."""
import random

import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from test_gpu_attn_batch import Batch
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
