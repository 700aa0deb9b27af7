"""The attention weight that positions gather from chunks of tokens, against its definition in 64 bits.

Tolerance: a weight's relative error is that of exp(score - lse), the absolute error of score - lse.  A score is a sum of 256
products in fp32, each partial sum rounded by at most 2^-24 of sum |q_i k_i| / 16, about 10 for N(0,1): at worst
256 * 2^-24 * 10 = 1.6e-4, at random sqrt(256) times less than that and below 1e-5 in the norm; the parts of Q leave 2^-22 * 10;
lse (given in fp32, at most 16) 2^-24 * 16, the exponential and its argument another 2^-22 * 16, each fp32 sum 2^-24 of itself a
term.  2e-4 for any element, 1e-5 in the norm."""
import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from test_gpu_attn_batch import Batch, i32
from test_gpu_chunks import offsets, prefill

pytestmark = pytest.mark.gpu


def log_sums(b, q, order, counts, max_len):
    """lse of the chunks' rows and, per chunk, exp(score - lse) in 64 bits summed: [4][len]"""
    lse, sums, at = [], [], 0
    for s, c in zip(order, counts):
        m = min(b.lens[s], max_len) if 0 <= s < len(b.lens) else 0
        K = b.values(s)[0][:, :m] if m else torch.zeros((4, 0, 256), dtype=torch.float64)
        x = q[at:at + c].double().cpu().view(c, 4, 6, 256)
        sc = torch.einsum("tghd,gjd->tghj", x, K) / 16.0
        hidden = torch.arange(m) > (m - c + torch.arange(c))[:, None]
        sc = sc.masked_fill(hidden[:, None, None], -torch.inf)
        l = torch.logsumexp(sc, -1) if m else torch.full((c, 4, 6), -torch.inf, dtype=torch.float64)
        lse.append(l.reshape(c, 24))
        l32 = l.float().double()
        p = torch.where(torch.isinf(l32)[..., None], 0.0, torch.exp(sc - torch.where(torch.isinf(l32), 0.0, l32)[..., None]))
        sums.append(p.sum((0, 2)))
        at += c
    return torch.cat(lse), sums


def weights(b, q, lse, off, n, rows, max_len, mass, seqs=None, work=None):
    if work is None:
        work = torch.full((ops.attn_weights_batch_work_bytes(n, rows, max_len),), 0xFF, dtype=torch.uint8, device="cuda")
    ops.attn_weights_batch(q, lse, b.kv, b.kvt, b.pages, None if seqs is None else i32(seqs), i32(off), n, rows, max_len, mass, work)
    torch.cuda.synchronize()


def near(got, want, what):
    got, want = got.double().cpu(), want.double().cpu()
    d = (got - want).abs()
    rel = (d.norm() / want.norm().clamp_min(1e-30)).item()
    worst = (d - 2e-4 * want.abs()).max().item()
    print(f"{what}: rel-L2 {rel:.2e}", flush=True)
    assert worst <= 1e-30 and rel <= 1e-5, f"{what}: rel-L2 {rel:.3e}, {worst:.3e}"


def check(b, counts, seqs=None, pad=0, max_len=None, counted=None, seed=5):
    """counted: which chunks add (of several of a sequence the last one)."""
    off, n = offsets(counts), len(counts)
    order, max_len = list(range(len(b.lens))) if seqs is None else seqs, max_len or max(b.lens)
    T, rows = off[-1], off[-1] + pad
    q = seeded_normal((rows, 24, 256), seed)
    lse, sums = log_sums(b, q, order, counts, max_len)
    lse_gpu = torch.full((rows, 24), float("nan"), device="cuda")
    lse_gpu[:T] = lse.float().cuda()
    ld = b.pages.table.shape[1] * b.page
    before = seeded_normal((len(b.lens), 4, ld), 9).abs()
    mass = before.clone()
    weights(b, q, lse_gpu, off, n, rows, max_len, mass, seqs)
    want = before.double().cpu()
    for i, (s, c) in enumerate(zip(order, counts)):
        if c == 0 or not 0 <= s < len(b.lens) or (counted is not None and i not in counted):
            continue
        m = min(b.lens[s], max_len)
        want[s, :, max(0, m - c):m] = 0.0
        want[s, :, :m] += sums[i]
    near(mass, want, f"{KV_NAMES[b.kvt]} {b.lens} chunks {counts}")
    return mass


SIZES = [([1], [1], 16), ([64], [64], 16), ([65], [3], 64), ([63, 129, 700], [1, 40, 1], 32), ([300], [43], 64),
         ([700, 250], [333, 90], 256), ([40, 513, 96, 5], [1, 300, 0, 9], 16), ([2100, 64], [5, 64], 1024)]


@pytest.mark.parametrize("lens, counts, page", SIZES, ids=lambda v: str(v).replace(" ", "") if isinstance(v, list) else v)
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_weights(gpu, kvt, lens, counts, page):
    check(Batch(kvt, lens, page=page), counts, pad=3)


@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_sequences_named(gpu, kvt):
    """Any order, unknown sequences, a sequence twice (the last chunk with tokens counts), a bound below a length."""
    b = Batch(kvt, [200, 77, 410, 0, 33])
    check(b, [3, 50, 1, 20, 4, 0, 2], seqs=[2, 0, -1, 2, 9, 0, 3], counted=[1, 3])
    check(b, [30, 3, 90], seqs=[2, 4, 0], max_len=128)
    check(Batch(kvt, [17 + i % 40 for i in range(1024)], page=16), [(i * 7) % 3 for i in range(1024)])


def test_log_sums_of_the_attention(gpu):
    """As they are used together: attention of a chunk, then the weights with its log sums: every row's weights sum to 1."""
    for kvt in KVTS:
        b = Batch(kvt, [900, 60])
        counts = [70, 1]
        q, _, _, lse = prefill(b, offsets(counts), 2, 71, 900)
        mass = torch.zeros((2, 4, b.pages.table.shape[1] * b.page), device="cuda")
        weights(b, q, lse, offsets(counts), 2, 71, 900, mass)
        total = mass.double().sum(-1).cpu()
        want = torch.tensor([[6.0 * 70], [6.0]]).expand(2, 4).double()
        assert ((total - want).abs() <= 4e-4 * want).all(), total  # (twice the bound of a score's error: in lse, and here)
        # the last tokens alone, with other offsets into the same rows: a window of 10
        window = torch.zeros_like(mass)
        weights(b, q, lse, [60, 70, 71], 2, 71, 900, window)
        assert ((window.double().sum(-1).cpu() - torch.tensor([[60.0], [6.0]])).abs() <= 0.024).all()


def test_holes_and_values_that_are_not_finite(gpu):
    """Positions of a foreign page gather nothing; a K value that is not finite shows at its own position and nowhere else."""
    for kvt in KVTS:
        b = Batch(kvt, [400, 64], page=32)
        q = seeded_normal((53, 24, 256), 3)
        off = [0, 50, 53]
        b.pages.table[0, 2] = -1
        lse = torch.full((53, 24), 8.0, device="cuda")
        ld = b.pages.table.shape[1] * 32
        clean = torch.ones((2, 4, ld), device="cuda")
        weights(b, q, lse, off, 2, 53, 400, clean)
        assert (clean[0, :, 64:96] == 1.0).all() and (clean[0, :, :64] > 1.0).all() and (clean[0, :, 400:] == 1.0).all()
        slot = int(b.pages.table[0, 11]) * 32 + 30  # position 382: tokens from 32 on see it
        if kvt == ops.F16:
            b.kv.k[2, slot].view(torch.int16)[200] = 0x7E00
        else:
            b.kv.ks[2, slot, 6] = 0x7E00
        mass = torch.ones((2, 4, ld), device="cuda")
        weights(b, q, lse, off, 2, 53, 400, mass)
        bad = torch.zeros_like(mass, dtype=torch.bool)
        bad[0, 2, 382] = True
        assert torch.isnan(mass[bad]).all() and torch.equal(mass[~bad], clean[~bad])


def test_streams_and_graphs(gpu):
    """The same bits on other streams and from a captured graph that follows the device's numbers."""
    kvt, n, rows = ops.Q8_0, 3, 400
    b = Batch(kvt, [900, 350, 64], ld=1024)
    q, lse = seeded_normal((rows, 24, 256), 1), 7.0 + seeded_normal((rows, 24), 2)
    off, size = i32(offsets([300, 1, 64])), ops.attn_weights_batch_work_bytes(n, rows, 1000)
    new = lambda: (torch.zeros((3, 4, b.pages.table.shape[1] * b.page), device="cuda"), torch.empty(size, dtype=torch.uint8, device="cuda"))

    def call(o, stream=None):
        ops.attn_weights_batch(q, lse, b.kv, kvt, b.pages, None, off, n, rows, 1000, *o, stream=stream)

    first, second, third = new(), new(), new()
    call(first)
    call(first)
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(2):
        call(second, streams[0])
        call(third, streams[1])
    torch.cuda.synchronize()
    assert torch.equal(second[0], first[0]) and torch.equal(third[0], first[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(second)
    for lens, cs in (([900, 350, 64], [300, 1, 64]), ([200, 350, 10], [7, 100, 10]), ([0, 1, 64], [0, 1, 40])):
        off.copy_(i32(offsets(cs)))
        b.pages.len.copy_(i32(lens))
        second[0].fill_(0.5)
        third[0].fill_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        call(third)
        torch.cuda.synchronize()
        assert torch.equal(second[0], third[0]) and bool((third[0] != 0.5).any())
