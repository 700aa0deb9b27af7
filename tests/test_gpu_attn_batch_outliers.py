"""Batched decode attention over caches with outlier keys (1% of the key rows eight times as large), against the definition in
64 bits, in every kernel that the sizes lead to.

Such keys have scores with a standard deviation of 8, so an error of a score enters the output at full weight: with Q / 16 or
d * code rounded to fp16 a score is off by up to 1e-2 and an output by 4e-3 to 6e-3.  The scores have to be exact up to fp32
accumulation (256 products of fp16 numbers, 2^-24 each).  Then P, V and the output are off by at most half a step of fp16,
2^-11 relative each: |error| <= 2^-10 sum_j p_j |v_j| + 2^-11 |out|.  `close` allows 3 * 2^-11 |out| + 2e-3, and
2^-10 (sum_j p_j |v_j| - |out|) is below 2e-3 as long as the sum of p_j |v_j| is not 2 larger than |out|; V ~N(0,1) has a mean
magnitude of 0.8, and a key that outweighs the others adds to both alike."""
import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES, seeded_normal
from pageref import batch_attention
from test_gpu_attn_batch import Batch, close

pytestmark = pytest.mark.gpu


class Outliers(Batch):
    """A Batch whose keys are eight times as large at 1% of the (position, KV head) pairs."""

    def __init__(self, kvt, lens, shared=0, page=64, seed=5):
        super().__init__(kvt, lens, shared, page, seed)
        K0, V0 = seeded_normal((max(shared, 1), 4, 256), seed + 2000), seeded_normal((max(shared, 1), 4, 256), seed + 2001)
        g = torch.Generator(device="cuda").manual_seed(seed + 2002)
        big = lambda K: torch.where(torch.rand(K.shape[:2], generator=g, device="cuda")[..., None] < 0.01, 8.0 * K, K)
        K0 = big(K0)
        for i, m in enumerate(lens):
            K = torch.cat([K0[:min(shared, m)], big(seeded_normal((max(0, m - shared), 4, 256), seed + 3000 + i))])
            V = torch.cat([V0[:min(shared, m)], seeded_normal((max(0, m - shared), 4, 256), seed + 5000 + i)])
            cache = self.caches[i]
            ops.kv_append(K, V, 0, m, kvt, cache)
            at = torch.arange(m, device="cuda")
            slot = self.pages.table[i].long()[at // page] * page + at % page
            for dst, src in ((self.kv.k, cache.k), (self.kv.v, cache.v), (self.kv.ks, cache.ks), (self.kv.vs, cache.vs)):
                if dst is not None:
                    dst[:, slot] = src[:, :m]


CASES = {"own positions": ([9000, 3001, 12000], 0, 1), "own positions, 8 queries": ([5003, 2500], 0, 8),
         "two sequences over a prefix": ([8200, 8300], 8192, 1), "five over a prefix": ([8200 + 7 * i for i in range(5)], 8192, 1),
         "forty over a prefix": ([8200 + 7 * i for i in range(40)], 8192, 1),
         "7 queries over a prefix": ([4100 + 17 * i for i in range(5)], 4093, 7)}


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_outlier_keys(gpu, kvt, case):
    lens, shared, nq = CASES[case]
    Outliers(kvt, lens, shared, page=16 if nq == 7 else 64).check(nq, shared, what=f"{KV_NAMES[kvt]} {case}")


@pytest.mark.parametrize("n, nq, shared", [(170, 8, 131072), (128, 1, 0)])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_many_keys_far_below_the_largest_score(gpu, kvt, n, nq, shared):
    """One key with a score 17.4 above those of 131071 others, as the first token of a prompt may have it: each of the others
    weighs 2.8e-8, less than half of fp16's least number, but together they move the output from -1 to -0.993.

    The states that hold the first key have the whole range (prefix) or a wave's quarter of it.  Tolerance: an MFMA adds 32
    keys in at most 4 sums, each off by half a step of 2^-24, O and l alike; the output is off by 2^-12, and the weights of
    the others, which together are 4e-3, by 2^-9 at most (their fp16 numbers have 9 bits)."""
    page, pages, most = 64, 64, 131072
    kv, pg = ops.KVLayer.allocate(kvt, pages * page), ops.KVPages.allocate(n, most, pages, page)
    K, V = torch.zeros((pages * page, 4, 256), device="cuda"), torch.ones((pages * page, 4, 256), device="cuda")
    K[0], V[0] = 1.0875, -1.0
    ops.kv_append(K, V, 0, pages * page, kvt, kv)
    table = torch.randint(1, pages, (n, most // page), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    table[:] = table[:1]
    table[:, 0] = 0
    pg.table.copy_(table)
    pg.len.fill_(most)
    q, gate = torch.ones((n * nq, 24, 256), device="cuda"), torch.full((n * nq, 24, 256), 30.0, device="cuda")
    out = torch.empty((n * nq, 24, 256), dtype=torch.float16, device="cuda")
    work = torch.empty(ops.attn_batch_work_bytes(n, nq, shared, most), dtype=torch.uint8, device="cuda")
    ops.attn_decode_batch(q, gate, kv, kvt, pg, None, n, nq, shared, most, out, work)
    torch.cuda.synchronize()
    b = Batch.__new__(Batch)
    b.kvt, b.caches, b._rows = kvt, [kv], {}
    k64, v64 = b.values(0)
    top, rest = k64[0, 0].sum() / 16, k64[0, 1].sum() / 16
    assert 17.35 < top - rest < 17.45
    tol = 8 * (most if shared else most // 4) / 32 * 2.0**-24 + 2.0**-12 + 4e-3 * 2.0**-9
    for t in range(nq):
        others = (most - nq + t) * torch.exp(rest - top)
        want = (v64[0, 0, 0] + others * v64[0, 1, 0]) / (1 + others)
        err = (out.view(n, nq, 24, 256)[:, t].double().cpu() - want).abs().max().item()
        print(f"{KV_NAMES[kvt]} {n} x {nq}, query {t}: off by {err:.2e} of {tol:.2e}", flush=True)
        assert err <= tol


@pytest.mark.parametrize("base", [60000, 59968, 52544, 33024])
@pytest.mark.parametrize("lens, shared, nq", [([3000, 200], 0, 1), ([700], 0, 8), ([2900, 2800], 2700, 1),
                                              ([2900 - 10 * i for i in range(9)], 2700, 1)])
def test_scores_of_a_million(gpu, lens, shared, nq, base):
    """Scores of 1.0 to 1.9 million that differ by 0 to 10, all of them whole numbers that fp32 holds: a state's reference times
    log2(e) is off by up to 0.1 there, and the states of a row, each with its own, have to weigh the same all the same.
    F16 keys of 255 equal numbers and a small one; half of the queries look the other way (scores below minus a million)."""
    b = Batch(ops.F16, lens, shared=shared)
    n = len(lens)
    for i, m in enumerate(lens):
        g = torch.Generator(device="cuda").manual_seed(900 + i)
        g0 = torch.Generator(device="cuda").manual_seed(899)
        own = torch.randint(0, 11, (m, 4), generator=g, device="cuda")
        own[:min(shared, m)] = torch.randint(0, 11, (max(shared, 1), 4), generator=g0, device="cuda")[:min(shared, m)]
        K = torch.full((m, 4, 256), float(base), device="cuda")
        K[..., 255] = 8.0 * own
        ops.kv_append(K, None, 0, m, ops.F16, b.caches[i])
        at = torch.arange(m, device="cuda")
        b.kv.k[:, b.pages.table[i].long()[at // b.page] * b.page + at % b.page] = b.caches[i].k[:, :m]
    q, gate = torch.full((n * nq, 24, 256), 2.0, device="cuda"), seeded_normal((n * nq, 24, 256), 4)
    q[:, ::2] = -2.0
    q[..., 255] = 2.0
    out = torch.empty((n * nq, 24, 256), dtype=torch.float16, device="cuda")
    work = torch.empty(ops.attn_batch_work_bytes(n, nq, shared, max(lens)), dtype=torch.uint8, device="cuda")
    ops.attn_decode_batch(q, gate, b.kv, b.kvt, b.pages, None, n, nq, shared, max(lens), out, work)
    torch.cuda.synchronize()
    want = batch_attention(q, gate, lambda t: b.values(t // nq), [lens[t // nq] - nq + t % nq + 1 for t in range(n * nq)])
    close(out, want, f"{lens} shared {shared}, {base}")
