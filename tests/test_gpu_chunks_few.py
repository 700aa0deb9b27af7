"""Chunks of one or two tokens beside longer ones, where sequences are long enough to be cut: their keys are walked by themselves, in
steps of 256 positions.  Tolerances as for the chunks in general."""
import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from test_gpu_attn_batch import Batch, i32
from test_gpu_chunks import attention, check, close, offsets, prefill, LSE

pytestmark = pytest.mark.gpu
LONG = 2048  # (a bound of the lengths from which on they are cut)


@pytest.mark.parametrize("lens, counts, page", [
    ([1], [1], 16), ([2], [2], 64), ([1], [2], 64), ([0], [1], 64), ([255, 256, 257], [1, 2, 1], 16), ([512, 513], [2, 1], 128),
    ([2047], [1], 1024), ([1300, 40, 700, 0, 1], [1, 2, 1, 1, 2], 32), ([900, 30, 600, 256], [1, 130, 2, 22], 64),
    ([1500, 3, 1400, 1024, 17], [1, 3, 500, 2, 0], 256)], ids=lambda v: str(v).replace(" ", "") if isinstance(v, list) else v)
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_attention(gpu, kvt, lens, counts, page):
    b = Batch(kvt, lens, page=page, ld=LONG // page)
    out, lse = check(b, counts, pad=3, max_len=LONG)
    assert torch.equal(check(b, counts, pad=3, max_len=LONG, lse=False)[0], out)


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_sequences_named(gpu, kvt):
    """Any order, a sequence twice, unknown ones (zeros), a bound below a length."""
    b = Batch(kvt, [800, 77, 1410, 0, 33])
    check(b, [2, 1, 1, 20, 1, 0, 2], seqs=[2, 0, -1, 2, 9, 1, 3], pad=1)
    check(b, [1, 2, 40, 1], seqs=[2, 4, 0, 2], max_len=700)


def test_many_chunks(gpu):
    """More than a wave plans by itself, and as many as a call takes; more of them than slices."""
    b = Batch(ops.Q8_0, [(i * 37) % 1500 for i in range(150)])
    check(b, [(0, 1, 2, 5)[i % 4] for i in range(150)])
    b = Batch(ops.Q4_0, [17 + i % 40 for i in range(1024)], page=16, ld=64)
    check(b, [(i * 7) % 3 for i in range(1024)], max_len=1024)


def test_long_and_images(gpu):
    """Tokens at 40000 positions beside a chunk whose keys are brought into LDS's form once."""
    check(Batch(ops.Q4_0, [40000, 3000, 39000, 2], page=256), [1, 600, 2, 1])


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_not_finite(gpu, kvt):
    """K or V that is not finite shows where it is seen: of two tokens the first does not see the last position."""
    b = Batch(kvt, [300, 290], ld=LONG // 64)
    off = offsets([2, 1])
    q, gate, clean, _ = prefill(b, off, 2, 3, LONG)
    bad = 299
    slot = int(b.pages.table[0, bad // b.page]) * b.page + bad % b.page
    mark = torch.zeros((3, 24, 256), dtype=torch.bool, device="cuda")
    for what in "vk":
        values, scales = (b.kv.v, b.kv.vs) if what == "v" else (b.kv.k, b.kv.ks)
        keep = values[1, slot].clone(), None if scales is None else scales[1, slot].clone()
        if kvt == ops.F16:
            values[1, slot].view(torch.int16)[5] = 0x7E00
            dims = [5]
        else:
            scales[1, slot, 2] = 0x7E00
            dims = list(range(64, 96))
        _, _, out, lse = prefill(b, off, 2, 3, LONG, q=q, gate=gate)
        mark[:] = False
        mark[1, 6:12, dims if what == "v" else slice(None)] = True
        assert torch.isnan(out[mark]).all() and torch.equal(out[~mark], clean[~mark])
        assert torch.isnan(lse[1, 6:12]).all() == (what == "k")
        values[1, slot] = keep[0]
        if keep[1] is not None:
            scales[1, slot] = keep[1]


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_pages_outside_the_pool(gpu, kvt):
    b = Batch(kvt, [700, 64], page=32, ld=LONG // 32)
    for e, bad in ((2, -1), (7, 1 << 30), (21, b.pages.ref.numel())):
        b.pages.table[0, e] = bad
    b.pages.table[1, 0] = b.pages.table[1, 1] = -1  # (nothing is left of it)
    q, gate, out, lse = prefill(b, [0, 2, 3], 2, 3, LONG)
    gone = torch.zeros(700, dtype=torch.bool)
    gone[64:96] = gone[224:256] = gone[672:] = True
    K, V = b.values(0)
    K, V, kept = K[:, ~gone], V[:, ~gone], (~gone).cumsum(0)
    want, want_lse = attention(q[:2], gate[:2], lambda t: (K, V), [int(kept[698 + t]) for t in range(2)])
    close(out[:2], want, "holes")
    assert (lse[:2].double().cpu() - want_lse).abs().max() <= LSE
    assert (out[2] == 0).all() and (lse[2] == -torch.inf).all()


def test_scores_of_a_million(gpu):
    b = Batch(ops.F16, [5000, 4000])
    check(b, [2, 1], q=3000.0 * seeded_normal((3, 24, 256), 3), lse=False)


def test_streams_and_graphs(gpu):
    """Two calls at once, and a captured one that follows the device's numbers as chunks become long and short."""
    n, rows, m = 4, 200, 1000
    b = Batch(ops.Q8_0, [900, 350, 64, 800], ld=16)
    q, gate = seeded_normal((rows, 24, 256), 1), seeded_normal((rows, 24, 256), 2)
    off, size = i32(offsets([1, 2, 1, 100])), ops.attn_prefill_batch_work_bytes(n, rows, m)
    new = lambda: (torch.zeros((rows, 24, 256), dtype=torch.float16, device="cuda"), torch.zeros((rows, 24), device="cuda"),
                   torch.empty(size, dtype=torch.uint8, device="cuda"))

    def call(o, stream=None):
        ops.attn_prefill_batch(q, gate, b.kv, b.kvt, b.pages, None, off, n, rows, m, o[0], o[2], lse=o[1], stream=stream)

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
    for lens, cs in (([900, 350, 64, 800], [1, 2, 1, 100]), ([200, 350, 10, 999], [2, 2, 2, 1]), ([0, 1, 64, 900], [1, 1, 40, 150]),
                     ([900, 900, 900, 900], [0, 1, 0, 1])):
        off.copy_(i32(offsets(cs)))
        b.pages.len.copy_(i32([min(x, y) for x, y in zip(lens, b.lens)]))
        for o in (second, third):
            o[0].zero_()
            o[1].zero_()
        graph.replay()
        torch.cuda.synchronize()
        call(third)
        torch.cuda.synchronize()
        assert torch.equal(second[0], third[0]) and torch.equal(second[1], third[1])
        assert bool(third[0].abs().sum() > 0)


@pytest.mark.parametrize("n", [64, 65, 128, 129])
def test_numbers_of_chunks(gpu, n):
    """Where plans are made by a wave, by two and by a workgroup of 1024: chunks of none to 30 tokens, one of 300."""
    counts = [(i * 11) % 31 if i % 3 == 0 else i % 3 for i in range(n)]
    counts[n // 2] = 300
    b = Batch(ops.Q8_0, [max(c, (i * 53) % 640) for i, c in enumerate(counts)])
    check(b, counts, pad=2)


def test_offsets_past_32_bits(gpu):
    """A pool whose rows lie past 4 GiB of their head's, and heads past 8 GiB: two tokens, and a chunk that is read through images."""
    kvt, page = ops.F16, 1024
    small = Batch(kvt, [3000], page=page)
    n_pages = 8400
    kv = ops.KVLayer.allocate(kvt, n_pages * page)
    pages = ops.KVPages.allocate(1, 3 * page, n_pages, page)
    last = [n_pages - 1, n_pages - 3, n_pages - 2]
    pages.table[0, :3] = i32(last)
    pages.len.fill_(3000)
    for e, pg in enumerate(last):
        old = int(small.pages.table[0, e])
        for dst, src in ((kv.k, small.kv.k), (kv.v, small.kv.v)):
            dst[:, pg * page:(pg + 1) * page] = src[:, old * page:(old + 1) * page]
    want = [prefill(small, [0, c], 1, c, 3000)[2:] for c in (2, 300)]
    small.kv, small.pages = kv, pages
    for c, (out, lse) in zip((2, 300), want):
        got = prefill(small, [0, c], 1, c, 3000)[2:]
        assert torch.equal(got[0], out) and torch.equal(got[1], lse)


def test_images_without_room(gpu):
    """Three long chunks, of which the scratch has room for one's images: each as in a call of its own, both within the tolerance."""
    counts, lens = [300, 310, 290], [70000, 66000, 68000]
    b, rows = Batch(ops.Q4_0, lens, page=1024), sum(counts)
    off = offsets(counts)
    q, gate, out, lse = prefill(b, off, 3, rows, max(lens))
    for i, c in enumerate(counts):
        at = slice(off[i], off[i + 1])
        _, _, alone, alone_lse = prefill(b, [0, c], 1, c, max(lens), seqs=[i], q=q[at].contiguous(), gate=gate[at].contiguous())
        close(out[at], alone, f"chunk {i}", max_abs=4e-3, rel_l2=1e-3)
        assert (lse[at] - alone_lse).abs().max().item() <= 2 * LSE
