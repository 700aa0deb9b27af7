"""Chunks, weights and evictions at the ends of their ranges: the longest sequences, as many rows as a call takes, no token at all.
Definitions and tolerances as in test_gpu_chunks, test_gpu_weights and test_gpu_evict."""
import pytest
import torch

import qwengine_amd.ops as ops
import test_gpu_evict
from kvutil import KVTS, KV_NAMES, seeded_normal
from test_gpu_attn_batch import EPS, THETA, Batch, i32
from test_gpu_chunks import LSE, attention, close, offsets, prefill, prep_inputs
from test_gpu_weights import log_sums, near, weights

pytestmark = pytest.mark.gpu
LONGEST = 262144


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_longest_sequences(gpu, kvt):
    """A decoded token, a few, and a chunk that is read through images, over 262144 positions.  Every table entry names one of 64
    pages, so that a key counts as often as its page is named.  (V is about the same all over a page and differs between pages,
    or everything would average out.)"""
    page, pages, ld, counts = 64, 64, LONGEST // 64, [1, 7, 240]
    n, T, off = 3, sum(counts), offsets(counts)
    K, V = seeded_normal((pages * page, 4, 256), 31), 0.1 * seeded_normal((pages * page, 4, 256), 32)
    V += seeded_normal((pages, 4, 256), 33).repeat_interleave(page, 0)
    b = Batch.__new__(Batch)
    b.kvt, b.page, b._rows = kvt, page, {}
    b.kv, b.pages = ops.KVLayer.allocate(kvt, pages * page), ops.KVPages.allocate(n, LONGEST, pages, page)
    b.caches = [b.kv]
    ops.kv_append(K, V, 0, pages * page, kvt, b.kv)
    table = torch.randint(0, pages, (n, ld), generator=torch.Generator().manual_seed(34), dtype=torch.int32)
    lens = [LONGEST, LONGEST - 37, LONGEST]
    b.pages.table.copy_(table)
    b.pages.len.copy_(i32(lens))
    q, gate, out, lse = prefill(b, off, n, T, LONGEST)
    k64, v64 = (x.cuda() for x in b.values(0))
    want, want_lse = torch.zeros((T, 24, 256), dtype=torch.float64), torch.zeros((T, 24), dtype=torch.float64)
    before = torch.ones((n, 4, LONGEST), device="cuda")
    mass, want_mass = before.clone(), before.double()
    for s, (m, c) in enumerate(zip(lens, counts)):
        slot = (table[s].long()[:, None] * page + torch.arange(page)).flatten()[:m].cuda()
        want_mass[s, :, m - c:m] = 0.0
        for t in range(c):
            r, seen = off[s] + t, m - c + t + 1
            times = torch.bincount(slot[:seen], minlength=pages * page).double()
            for h in range(4):
                x = q[r, 6 * h:6 * h + 6].double() @ k64[h].T / 16.0
                top = x.amax(-1, keepdim=True)
                e = torch.exp(x - top) * times
                want[r, 6 * h:6 * h + 6] = ((e / e.sum(-1, keepdim=True)) @ v64[h]).cpu()
                l = top[:, 0] + e.sum(-1).log()
                want_lse[r, 6 * h:6 * h + 6] = l.cpu()
                want_mass[s, h, :seen] += torch.exp(x - l.float().double()[:, None]).sum(0)[slot[:seen]]
    close(out, want * torch.sigmoid(gate.double().cpu()), f"{KV_NAMES[kvt]} longest")
    assert (lse.double().cpu() - want_lse).abs().max().item() <= LSE
    weights(b, q, want_lse.float().cuda(), off, n, T, LONGEST, mass)
    near(mass, want_mass, f"{KV_NAMES[kvt]} longest")


def test_longest_evicted(gpu):
    pages, kvs, mass = test_gpu_evict.make(ops.Q4_0, [LONGEST, 1000], 64, 1)
    test_gpu_evict.run(pages, kvs, ops.Q4_0, mass, [0, 1], [131073, 999], 4000).check()


def test_as_many_rows_as_a_call_takes(gpu):
    """65536 rows: 1024 chunks of 64 tokens, of which some are compared; the offsets' last row is the buffers' last."""
    n, c = 1024, 64
    rows = n * c
    b = Batch(ops.Q4_0, [c + (i * 29) % 64 for i in range(n)], page=16)
    off = offsets([c] * n)
    q, gate, out, lse = prefill(b, off, n, rows, 127)
    mass = torch.zeros((n, 4, b.pages.table.shape[1] * 16), device="cuda")
    weights(b, q, lse, off, n, rows, 127, mass)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    total = mass.double().sum(-1)
    assert ((total - 6.0 * c).abs() <= 4e-4 * 6 * c).all()
    for s in (0, 1, 2, 63, 64, 500, 511, 512, 777, 1022, 1023):
        at = slice(off[s], off[s + 1])
        want, want_lse = attention(q[at], gate[at], lambda t: b.values(s), [b.lens[s] - c + t + 1 for t in range(c)])
        close(out[at], want, f"chunk {s}")
        assert (lse[at].double().cpu() - want_lse).abs().max().item() <= LSE
        _, sums = log_sums(b, q[at], [s], [c], 127)
        # (lse of the call: off by up to LSE, and every weight by that much of itself)
        d = (mass[s, :, :b.lens[s]].double().cpu() - sums[0]).abs()
        assert (d <= 4e-4 * sums[0]).all()


def test_a_chunk_of_65536_tokens(gpu):
    """A prompt in one call; rows and positions from all over it are compared."""
    c, m = 65536, 65600
    b = Batch(ops.Q8_0, [m], page=1024)
    q, gate, out, lse = prefill(b, [0, c], 1, c, m)
    mass = torch.ones((1, 4, b.pages.table.shape[1] * 1024), device="cuda")
    weights(b, q, lse, [0, c], 1, c, m, mass)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all() and (mass[0, :, m:] == 1.0).all()
    k64, v64 = (x.cuda() for x in b.values(0))
    for t in (0, 1, 21, 4095, 30000, 54613, 65535):
        seen = m - c + t + 1
        for h in range(4):
            x = q[t, 6 * h:6 * h + 6].double() @ k64[h, :seen].T / 16.0
            l = torch.logsumexp(x, -1)
            want = torch.exp(x - l[:, None]) @ v64[h, :seen] * torch.sigmoid(gate[t, 6 * h:6 * h + 6].double())
            close(out[t, 6 * h:6 * h + 6], want, f"token {t}")
            assert (lse[t, 6 * h:6 * h + 6].double() - l).abs().max().item() <= LSE
    at = torch.tensor([0, 17, 63, 64, 1000, 30011, 65535, 65599], device="cuda")
    first = (at - (m - c)).clamp_min(0)
    for h in range(4):
        x = torch.exp(q[:, 6 * h:6 * h + 6].double().reshape(-1, 256) @ k64[h, at].T / 16.0 - lse[:, 6 * h:6 * h + 6].double().reshape(-1, 1))
        x = x.masked_fill(torch.arange(6 * c, device="cuda")[:, None] // 6 < first, 0.0).sum(0) + (at < m - c)
        # (65536 terms in fp32: by blocks of 256 rows, and 1536 of those)
        assert ((mass[0, h, at].double() - x).abs() <= 2e-4 * x).all()


@pytest.mark.parametrize("n", [1, 3, 70, 130])
def test_no_tokens(gpu, n):
    """Chunks that are all of them empty: nothing is written, by any plan."""
    b = Batch(ops.Q8_0, [100] * n, ld=33)
    for rows, max_len in ((40, 100), (40, 2048), (600, 2048)):
        _, _, out, lse = prefill(b, [rows // 2] * (n + 1), n, rows, max_len)
        assert (out == 7.0).all() and (lse == 7.0).all()
        mass = torch.full((n, 4, 33 * 64), 3.0, device="cuda")
        weights(b, torch.ones((rows, 24, 256), device="cuda"), torch.zeros((rows, 24), device="cuda"), [0] * (n + 1), n, rows, max_len, mass)
        assert (mass == 3.0).all()
        pool = b.kv.k.clone()
        data, q = prep_inputs(rows), torch.full((rows, 24, 256), 7.0, device="cuda")
        ops.attn_prep_rows_batch(*data, b.pages, None, i32([rows] * (n + 1)), n, rows, THETA, EPS, b.kvt, b.kv, q, q)
        torch.cuda.synchronize()
        assert (q == 7.0).all() and torch.equal(pool, b.kv.k)
