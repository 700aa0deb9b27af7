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
