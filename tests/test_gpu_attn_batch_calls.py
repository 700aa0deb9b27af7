"""Calls of the batched attention that the other tests do not make."""
import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from test_gpu_attn_batch import Batch, close, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nq, shared, max_len", [(1, 0, 130), (3, 0, 130), (8, 100, 131), (3, 0, 2), (5, 100, 100)])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_longer_sequences_count_as_cut_to_max_len(gpu, kvt, nq, shared, max_len):
    """A sequence of more than max_len positions has the bits that it has after kv_pages_trim to max_len."""
    b = Batch(kvt, [300, 101, 129, 131, 260], shared=100)
    _, _, longer = b.run(nq, shared, max_len)
    ops.kv_pages_trim(b.pages, i32([0, 1, 2, 3, 4]), i32([min(m, max_len) for m in b.lens]))
    _, _, cut = b.run(nq, shared, max_len)
    assert torch.isfinite(cut).all() and torch.equal(longer, cut)
    b.lens = [min(m, max_len) for m in b.lens]
    b.check(nq, shared, max_len=max_len)


@pytest.mark.parametrize("lens, shared, nq", [([5000, 7001], 0, 1),               # many register states: a workgroup per row
                                              ([300, 411, 4200], 0, 5),
                                              ([210 + i for i in range(40)], 200, 1),   # few tile states: a wave per row
                                              ([4100 + i for i in range(9)], 4096, 1)])  # many: a workgroup per row
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_act_q8_of_every_combine(gpu, kvt, lens, shared, nq):
    """ActQ8 rows from register and tile states, by the combine of a wave and of a workgroup per row: within a step of what the
    values say, and the sums of their own codes."""
    b = Batch(kvt, lens, shared=shared)
    oq = ops.ActQ8.allocate(len(lens) * nq * 6144)
    out = b.check(nq, shared, oq=oq)
    x = out.double().view(-1, 32)
    d, q = oq.d.double(), oq.q.double().view(-1, 32)
    # the fp16 output is off its fp32 value by up to 2^-11 of it, d by as much of amax / 127
    assert ((x.abs().amax(1) / 127 - d).abs() <= 2.0**-11 * x.abs().amax(1) / 127 + 2.0**-25).all()
    assert ((q * d[:, None] - x).abs() <= d[:, None] * 0.5001 + 2.0**-11 * x.abs() + 2.0**-25).all()
    assert torch.allclose(oq.s.double(), d * q.sum(1), rtol=1e-6, atol=0)


def test_calls_in_flight_on_two_streams(gpu):
    """Calls of different sizes queued on two streams, with nothing between them that waits, a workspace for each stream: every
    output has the bits of the call by itself."""
    b = Batch(ops.Q8_0, [3000 + 17 * i for i in range(40)], shared=2048)
    calls = [(40, 1, 2048), (9, 4, 2048), (3, 8, 0), (40, 1, 100)]
    most, new = max(b.lens), lambda n, nq: torch.empty((n * nq, 24, 256), dtype=torch.float16, device="cuda")
    ins = [[(seeded_normal((n * nq, 24, 256), 10 * s + k), seeded_normal((n * nq, 24, 256), 10 * s + k + 5))
            for k, (n, nq, _) in enumerate(calls)] for s in range(2)]
    outs = [[[new(n, nq) for n, nq, _ in calls] for _ in range(4)] for s in range(2)]
    size = max(ops.attn_batch_work_bytes(n, nq, sh, most) for n, nq, sh in calls)
    work = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]

    def call(s, k, out):
        n, nq, sh = calls[k]
        ops.attn_decode_batch(*ins[s][k], b.kv, b.kvt, b.pages, None, n, nq, sh, most, out, work[s])

    want = [[new(n, nq) for n, nq, _ in calls] for s in range(2)]
    for s in range(2):
        for k in range(len(calls)):
            call(s, k, want[s][k])
            torch.cuda.synchronize()
    for rep in range(4):
        for k in range(len(calls)):
            for s in range(2):
                with torch.cuda.stream(streams[s]):
                    call(s, (k + s) % len(calls), outs[s][rep][(k + s) % len(calls)])
    torch.cuda.synchronize()
    for s in range(2):
        for rep in range(4):
            assert all(torch.equal(a, w) for a, w in zip(outs[s][rep], want[s]))


@pytest.mark.parametrize("x", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("lens, shared, nq, s, at", [
    ([70, 300], 0, 8, 1, 299),                                    # own positions: the last of eight queries sees it
    ([70, 300, 13], 0, 5, 1, 296),
    ([300, 64, 65], 0, 1, 0, 17),                                 # every row of its sequence
    ([100, 300], 256, 1, 1, 250),                                 # a prefix of which one row has only a part
    ([250, 251, 90, 300, 0], 256, 1, 3, 250),
    ([0, 3, 40, 100, 250, 251, 252, 300, 301, 256, 255, 17], 256, 1, 7, 250),
    ([0, 3, 40, 100, 250, 251, 252, 300, 301, 256, 255, 17], 256, 1, 7, 0),
    ([256] * 6 + [255], 256, 8, 0, 255),                          # everything shared, eight queries
    ([600 - 50 * i for i in range(12)], 590, 3, 0, 333)])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_values_that_are_not_finite_stay_in_the_rows_that_see_them(gpu, kvt, lens, shared, nq, s, at, x):
    """A V value, then a K value (of a quantized type: a block's scale) at position `at` of sequence s that is not finite: the
    rows that see it are not finite there (for an infinite K where its score is infinity; with a score of -infinity the key
    weighs nothing), all others have the bits that they have with a finite one."""
    page, kvh, dim = 32, 2, 41
    b = Batch(kvt, lens, shared=shared, page=page)
    most = max(lens)
    _, _, clean = b.run(nq, shared, most)
    slot = int(b.pages.table[s, at // page]) * page + at % page
    # the position is every row's whose sequence holds that page there
    same = b.pages.table[:, at // page] == b.pages.table[s, at // page]
    sees = torch.tensor([bool(same[i]) and at < m - nq + t + 1 for i, m in enumerate(lens) for t in range(nq)], device="cuda")
    assert sees.any() and not sees.all()
    heads = torch.zeros(24, dtype=torch.bool, device="cuda")
    heads[6 * kvh:6 * kvh + 6] = True
    hit = sees[:, None] & heads
    for which in ("v", "k"):
        buf, col = (getattr(b.kv, which), dim) if kvt == ops.F16 else (getattr(b.kv, which + "s"), dim // 32)
        buf = buf.view(torch.float16)
        old = buf[kvh, slot, col].clone()
        buf[kvh, slot, col] = x
        _, _, out = b.run(nq, shared, most)
        buf[kvh, slot, col] = old
        seen = out[hit]
        if which == "v":
            assert not torch.isfinite(seen[:, dim]).any()
        elif x != x:
            assert torch.isnan(seen).all()
        assert torch.equal(out[~hit], clean[~hit])
