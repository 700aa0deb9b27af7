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
from test_gpu_attn_batch import Batch

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
