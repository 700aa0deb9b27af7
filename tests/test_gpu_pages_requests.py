"""Several fork or trim requests for one sequence in a call: the last of those that count is carried out, whatever ignored
requests stand behind it, also when a workgroup has only some of them (16 requests a workgroup)."""
import random

import pytest
import torch

import qwengine_amd.ops as ops
from pageref import PageRef
from test_gpu_pages import Both, i32

pytestmark = pytest.mark.gpu


class Counted(Both):
    """The requests that count, the last for each sequence, given to the definition one by one."""

    def fork(self, src, dst):
        n = len(self.ref.len)
        last = {d: s for s, d in zip(src, dst) if 0 <= d < n and s < n}
        ops.kv_pages_fork(self.pages, i32(src), i32(dst), self.work)
        self.ref.fork(list(last.values()), list(last))
        self.same()

    def trim(self, seqs, lens):
        last = {s: m for s, m in zip(seqs, lens) if 0 <= s < len(self.ref.len) and 0 <= m <= self.ref.len[s]}
        ops.kv_pages_trim(self.pages, i32(seqs), i32(lens))
        self.ref.trim(list(last), list(last.values()))
        self.same()


def test_ignored_requests_cancel_no_others(gpu):
    b = Counted(ops.Q8_0, 5, 4, 24, 16)
    assert b.extend([0, 1, 2], [33, 40, 7]) == 0
    b.fork([0, 99], [3, 3])
    assert b.ref.len[3] == 33
    b.fork([1, 0, 5, 5], [4, 3, 4, 3])
    assert b.ref.len[3:] == [33, 40]
    b.fork([1, -1, 7], [3, 3, 3])                      # src < 0 counts: 3 is left empty
    assert b.ref.len[3] == 0
    b.trim([1, 1], [5, 41])
    assert b.ref.len[1] == 5
    b.trim([0, 0, 0, 2], [30, 20, -1, 8])
    assert b.ref.len[0] == 20 and b.ref.len[2] == 7


def test_requests_of_many_workgroups(gpu):
    """Requests for few sequences, a third of them ignored, over as many workgroups as a call can have."""
    rng, n_seq = random.Random(7), 1024
    b = Counted(ops.Q4_0, n_seq, 20, 600, 16, n_layers=1)
    few = [3, 500, 1023]
    assert b.extend(few + [8], [300, 320, 161, 100]) == 0
    for k in range(6):
        seqs = [rng.choice(few) for _ in range(1000)]
        lens = [rng.choice([rng.randint(0, b.ref.len[s]), b.ref.len[s] + rng.randint(1, 9), -1]) for s in seqs]
        b.trim(seqs, lens)
        dst = [rng.choice(few) for _ in range(1000)]
        src = [rng.choice([8, rng.choice(few), n_seq + rng.randint(0, 9)]) for _ in dst]
        b.fork(src, dst)
        assert b.extend(few, [40, 1, 100]) == 0
