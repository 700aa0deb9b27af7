"""A prompt brought into the pages by the prefill operators: on a compacted pool the pages of a new sequence follow each other,
so a layer whose pointers begin at the first of them is the sequence's own contiguous cache."""
import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from test_gpu_attn_batch import EPS, THETA, close, i32

pytestmark = pytest.mark.gpu


def from_position(kv, pos):
    """The pool from position pos on (the head stride stays the pool's)."""
    at = lambda t: None if t is None else t.data_ptr() + pos * t.shape[2] * t.element_size()
    return ops.KVLayer(kv.kvt, kv.capacity, at(kv.k), at(kv.v), at(kv.ks), at(kv.vs))


@pytest.mark.parametrize("prompt, chunk, last", [(700, 300, False), (1, 1, False), (65, 64, True)])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_prompt_prefilled_in_its_pages(gpu, kvt, prompt, chunk, last):
    """Compact, room, prep and prefill through the offset layer in chunks, then forks that decode: cache rows and prefill
    outputs have the bits of a contiguous cache, no other pool byte changes, and the decode is that of one sequence.
    (last: the prompt's pages are the last of the pool.)"""
    page, n = 64, 3
    need = -(-(prompt + 1) // page)
    n_pages = 5 + need if last else 30 + need
    pages = ops.KVPages.allocate(n + 3, 1024, n_pages, page)
    kv, flat = ops.KVLayer.allocate(kvt, n_pages * page), ops.KVLayer.allocate(kvt, prompt + 1)
    pool = [t for t in (kv.k, kv.v, kv.ks, kv.vs) if t is not None]
    for t in pool:
        t.view(torch.uint8).fill_(0x11)
    work = torch.empty(ops.kv_pages_work_bytes(pages), dtype=torch.uint8, device="cuda")
    status, n_live = i32([9]), i32([0])
    # two sequences that stay and one between them that goes: 3 + 2 pages in use
    for s, m in ((4, 130), (0, 60), (5, 100)):
        ops.kv_pages_extend(pages, i32([s]), i32([m]), [kv], kvt, status, work)
    ops.kv_pages_trim(pages, i32([0]))
    ops.kv_pages_compact(pages, [kv], kvt, n_live, work)
    before = [t.clone() for t in pool]
    ops.kv_pages_extend(pages, i32([0]), i32([prompt]), [kv], kvt, status, work)
    torch.cuda.synchronize()
    held = -(-prompt // page)
    row = pages.table[0, :held].tolist()
    assert int(status) == 0 and int(n_live) == 5 and row == list(range(5, 5 + held))
    start = row[0] * page

    w = 1 + 0.1 * seeded_normal((256,), 7)
    qg, k, v = seeded_normal((prompt, 24, 512), 1), seeded_normal((prompt, 4, 256), 2), seeded_normal((prompt, 4, 256), 3)
    new = lambda m, dt=torch.float32: torch.empty((m, 24, 256), dtype=dt, device="cuda")
    ops.attn_prefill_reserve(chunk, prompt)
    for p0 in range(0, prompt, chunk):
        m = min(chunk, prompt - p0)
        r, rope, outs = slice(p0, p0 + m), torch.empty((m, 64), device="cuda"), []
        ops.rope_table(p0, m, THETA, rope)
        for layer in (from_position(kv, start), flat):
            q, gate, out = new(m), new(m), new(m, torch.float16)
            ops.attn_prep_rows(qg[r], k[r], v[r], w, w, m, p0, rope, EPS, kvt, layer, q, gate)
            ops.attn_prefill(q, gate, layer, kvt, m, p0, out)
            outs.append(out)
        torch.cuda.synchronize()
        assert torch.equal(*outs)
    for t, b, f in zip(pool, before, [t for t in (flat.k, flat.v, flat.ks, flat.vs) if t is not None]):
        b[:, start:start + prompt] = f[:, :prompt]
        assert torch.equal(t, b)

    # samples of the prompt decode a token each
    ops.kv_pages_fork(pages, i32([0] * (n - 1)), i32(list(range(1, n))), work)
    ops.kv_pages_trim(pages, i32([4, 5]))
    ops.kv_pages_extend(pages, i32(list(range(n))), i32([1] * n), [kv], kvt, status, work)
    QG, K, V = seeded_normal((n, 24, 512), 11), seeded_normal((n, 4, 256), 12), seeded_normal((n, 4, 256), 13)
    q, gate, out = new(n), new(n), new(n, torch.float16)
    scratch = torch.empty(ops.attn_batch_work_bytes(n, 1, prompt, 1024), dtype=torch.uint8, device="cuda")
    ops.attn_prep_batch(QG, K, V, w, w, pages, None, n, 1, THETA, EPS, kvt, kv, q, gate)
    ops.attn_decode_batch(q, gate, kv, kvt, pages, None, n, 1, prompt, 1024, out, scratch)
    torch.cuda.synchronize()
    assert int(status) == 0 and pages.len.tolist()[:n] == [prompt + 1] * n
    dec, q1, g1, want = torch.empty(ops.attn_work_bytes(prompt + 1) // 4 + 1, device="cuda"), new(1), new(1), new(1)
    for b in range(n):
        src = [ops.RowSrc.device(t[b], x) for t, x in ((QG, 24 * 512), (K, 1024), (V, 1024))]
        ops.attn_prep_multi(*src, w, w, prompt, prompt, 1, THETA, EPS, kvt, flat, q1, g1)
        ops.attn_decode(q1, g1, flat, kvt, prompt + 1, dec, want)
        torch.cuda.synchronize()
        assert torch.equal(q1[0], q[b])
        close(out[b], want[0], f"sample {b}")
