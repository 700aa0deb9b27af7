"""The page operators on the GPU against their definition (tests/pageref.py): tables, lengths, counts and the moved page
contents have to be equal."""
import random

import pytest
import torch

import qwengine_amd.ops as ops
from kvutil import KVTS, KV_NAMES
from pageref import PageRef

pytestmark = pytest.mark.gpu


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def pools(kvt, slots, n_layers, seed):
    """Layers with random bytes in every buffer (F16 and scales too: a move copies any bits)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    layers = [ops.KVLayer.allocate(kvt, slots) for _ in range(n_layers)]
    for kv in layers:
        for t in (kv.k, kv.v, kv.ks, kv.vs):
            if t is not None:
                b = t.view(torch.uint8)
                b.copy_(torch.randint(0, 256, b.shape, generator=g, device="cuda", dtype=torch.uint8))
    return layers


def work_for(pages):
    return torch.full((ops.kv_pages_work_bytes(pages) // 4,), -77, dtype=torch.int32, device="cuda")


class Both:
    """The operators on the GPU and in the definition, compared after every call."""

    def __init__(self, kvt, n_seq, ld, n_pages, page, n_layers=2, slack=0, seed=1):
        self.kvt, self.pages = kvt, ops.KVPages.allocate(n_seq, ld * page, n_pages, page)
        self.layers = pools(kvt, n_pages * page + slack, n_layers, seed)
        self.work, self.status, self.n_live = work_for(self.pages), i32([99]), i32([99])
        self.ref = PageRef.of(self.pages, self.layers)

    def same(self, check=True):
        torch.cuda.synchronize()
        self.ref.same(self.pages, self.layers)
        if check:
            self.ref.check()

    def extend(self, seqs, add):
        ops.kv_pages_extend(self.pages, i32(seqs), i32(add), self.layers, self.kvt, self.status, self.work)
        want = self.ref.extend(seqs, add)
        self.same()
        assert int(self.status) == want
        return want

    def fork(self, src, dst):
        ops.kv_pages_fork(self.pages, i32(src), i32(dst), self.work)
        self.ref.fork(src, dst)
        self.same()

    def trim(self, seqs, lens=None):
        ops.kv_pages_trim(self.pages, i32(seqs), None if lens is None else i32(lens))
        self.ref.trim(seqs, lens)
        self.same()

    def compact(self):
        ops.kv_pages_compact(self.pages, self.layers, self.kvt, self.n_live, self.work)
        want = self.ref.compact()
        self.same()
        assert int(self.n_live) == want
        return want


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("kvt", KVTS, ids=lambda k: KV_NAMES[k])
def test_life_of_forks(gpu, kvt, page):
    b = Both(kvt, 6, 5, 24, page, slack=page + 3)
    assert b.extend([2], [page + 5]) == 0
    b.fork([2, 2, 2], [0, 1, 5])                       # a shared, partly filled last page
    assert b.extend([0, 2], [1, 2]) == 0               # two copies, the others keep the page
    assert b.extend([1, 5], [page, 0]) == 0            # the last but one holder copies; add 0 changes nothing
    assert b.extend([5], [3]) == 0                     # the last holder keeps it
    b.trim([1], [page])                                # to a page's end
    assert b.extend([1], [1]) == 0
    b.fork([0, 1], [1, 0])                             # a permutation
    b.fork([-1, 5], [2, 3])                            # one freed, one forked
    assert b.compact() == sum(r > 0 for r in b.ref.ref)
    b.trim([0, 1, 2, 3, 4, 5])
    assert b.compact() == 0


def test_all_sharers_of_a_page_at_once(gpu):
    """Of the sequences that share a partly filled page, the last of the call keeps it: one page less than copies."""
    b = Both(ops.Q8_0, 5, 3, 8, 16)
    assert b.extend([4], [20]) == 0
    b.fork([4, 4, 4, 4], [3, 2, 1, 0])
    assert b.extend([1, 0, 4, 2, 3], [1, 1, 1, 1, 1]) == 0
    assert sum(r > 0 for r in b.ref.ref) == 6


def test_refused_extends_change_nothing(gpu):
    b = Both(ops.Q4_0, 4, 4, 6, 32)
    assert b.extend([0, 1], [40, 64]) == 0
    assert b.extend([0, 1, 2], [1, 1, 64]) == 1        # 0 + 1 + 2 pages of the 2 that are free
    assert b.extend([3, 4], [1, 1]) == -2              # no such sequence
    assert b.extend([3, -1], [1, 1]) == -2
    assert b.extend([0, 2, 0], [1, 1, 1]) == -3        # named twice
    assert b.extend([0, 1], [-1, 1]) == -1
    assert b.extend([0], [89]) == -1                   # past the row: 4 pages of 32
    assert b.extend([0], [2**31 - 1]) == -1
    assert b.extend([0], [88]) == 0
    assert b.extend([2], [1]) == 1                     # nothing is left
    assert b.extend([2], [0]) == 0
    assert b.extend([], []) == 0


def test_ignored_forks_and_trims(gpu):
    b = Both(ops.F16, 5, 4, 16, 16)
    b.extend([0, 1, 2], [33, 16, 7])
    b.fork([0, 1, 2], [3, 3, 3])                       # several with the same dst: the last one counts
    b.fork([0, 5, 1], [5, 4, -1])                      # dst or src that is no sequence
    b.fork([0], [0])                                   # onto itself
    b.fork([4], [0])                                   # an empty source
    b.trim([1, 1], [5, 9])                             # the last one counts
    b.trim([1, 2, 7, -1], [17, -1, 0, 0])              # longer than it is, negative, no sequence
    b.trim([1], [0])


@pytest.mark.parametrize("n_pages", [1, 2, 15, 16, 4097, 9000])
def test_compact_of_any_pool(gpu, n_pages):
    rng = random.Random(n_pages)
    b = Both(ops.Q4_0, 7, n_pages, n_pages, 16, n_layers=1)
    left = n_pages
    for s in range(7):                                 # random lengths over scattered pages, some shared
        left -= (m := rng.randint(0, left))
        if m:
            b.extend([s], [m * 16 - rng.randint(0, 15)])
    for s in rng.sample(range(7), 3):
        b.trim([s], [rng.randint(0, b.ref.len[s])])
    b.fork([0, 1], [5, 6])
    n = b.compact()
    assert all(r > 0 for r in b.ref.ref[:n]) and not any(b.ref.ref[n:])
    assert b.compact() == n


def test_many_requests(gpu):
    """The most requests of a call, all sharing one last page, and a row of many pages at once."""
    n = ops.PAGES_MAXN
    b = Both(ops.Q4_0, n + 1, 70, 3000, 16, n_layers=1)
    assert b.extend([n], [1000]) == 0
    b.fork([n] * n, list(range(n)))
    assert b.extend(list(range(n)), [1 + i % 20 for i in range(n)]) == 0
    free = sum(r == 0 for r in b.ref.ref)
    assert 0 < free < 2 * n and b.extend(list(range(n)), [32] * n) == 2 * n - free
    b.fork([(i * 7 + 3) % n for i in range(n)], list(range(n)))
    b.trim(list(range(0, n, 2)))


@pytest.mark.parametrize("seed", range(4))
def test_random_lives(gpu, seed):
    rng = random.Random(seed)
    kvt, page = rng.choice(KVTS), rng.choice([16, 32, 64])
    n_seq = rng.randint(2, 9)
    b = Both(kvt, n_seq, 6, rng.randint(8, 30), page, n_layers=rng.choice([1, 3]), seed=seed)
    for _ in range(40):
        k = rng.randint(1, n_seq)
        some = rng.sample(range(n_seq), k)
        op = rng.choice(["extend"] * 4 + ["fork"] * 2 + ["trim", "free", "compact"])
        if op == "extend":
            b.extend(some, [rng.choice([0, 1, 1, 3, page, 2 * page]) for _ in some])
        elif op == "fork":
            b.fork([rng.randint(-1, n_seq - 1) for _ in some], some)
        elif op == "trim":
            b.trim(some, [rng.randint(0, b.ref.len[s]) for s in some])
        elif op == "free":
            b.trim(some[:1])
        else:
            b.compact()


def test_bad_tables_stay_inside(gpu):
    """Page numbers outside the pool and lengths outside the row, as a broken table may hold them: nothing outside the
    tables and the pool is touched, and the sound sequences keep their pages."""
    page, n_pages = 16, 8
    pages = ops.KVPages.allocate(4, 3 * page, n_pages, page)
    layers = pools(ops.Q8_0, n_pages * page, 1, 3)
    work, status, n_live = work_for(pages), i32([0]), i32([0])
    ops.kv_pages_extend(pages, i32([0]), i32([20]), layers, ops.Q8_0, status, work)
    pages.table[1] = i32([99, -5, 7])
    pages.len[1], pages.len[2], pages.len[3] = 40, -3, 10**6
    ops.kv_pages_extend(pages, i32([1]), i32([1]), layers, ops.Q8_0, status, work)  # its last page (7) is free: ref 0
    torch.cuda.synchronize()
    assert int(status) == 0
    ops.kv_pages_extend(pages, i32([2]), i32([1]), layers, ops.Q8_0, status, work)
    torch.cuda.synchronize()
    assert int(status) == -1
    ops.kv_pages_fork(pages, i32([1, 3]), i32([2, 3]), work)
    ops.kv_pages_trim(pages, i32([1, 2, 3]))
    ops.kv_pages_compact(pages, layers, ops.Q8_0, n_live, work)
    torch.cuda.synchronize()
    assert pages.table[0].tolist()[:2] == [0, 1] and pages.len.tolist()[0] == 20
    assert pages.ref.tolist()[:2] == [1, 1]


def test_captured_step_follows_the_tables(gpu):
    """Room, fork and trim in one captured graph, replayed while the tables change between the replays."""
    b = Both(ops.Q8_0, 4, 6, 24, 16)
    b.extend([0], [21])
    seqs, one, src, dst = i32([1, 2]), i32([1, 1]), i32([0, 0]), i32([1, 2])

    def step():
        ops.kv_pages_trim(b.pages, seqs)
        ops.kv_pages_fork(b.pages, src, dst, b.work)
        ops.kv_pages_extend(b.pages, seqs, one, b.layers, b.kvt, b.status, b.work)
        ops.kv_pages_compact(b.pages, b.layers, b.kvt, b.n_live, b.work)

    def ref():
        b.ref.trim([1, 2])
        b.ref.fork([0, 0], [1, 2])
        assert b.ref.extend([1, 2], [1, 1]) == 0
        return b.ref.compact()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    ref()
    b.same()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        graph.replay()
        n = ref()
        b.same()
        assert int(b.n_live) == n and int(b.status) == 0
        b.extend([0], [9])                             # the program's own work between the replays


def test_nothing_past_the_work_buffer(gpu):
    """The operators write no byte behind kv_pages_work_bytes, at their largest number of requests and moves."""
    n, page = 1024, 16
    pages = ops.KVPages.allocate(n, 3 * page, 3 * n, page)
    layers = pools(ops.Q4_0, 3 * n * page, 1, 3)
    need = ops.kv_pages_work_bytes(pages)
    work = torch.full((need + 4096,), 0xAB, dtype=torch.uint8, device="cuda")
    status, n_live = i32([9]), i32([0])
    seqs = torch.arange(n, dtype=torch.int32, device="cuda")
    pages.table[0, 0], pages.len[0], pages.ref[0] = 0, 5, 1
    ops.kv_pages_fork(pages, torch.zeros_like(seqs), seqs, work)          # everyone shares page 0 ...
    ops.kv_pages_extend(pages, seqs, torch.full_like(seqs, 20), layers, ops.Q4_0, status, work)  # ... and leaves it
    torch.cuda.synchronize()
    assert int(status) == 0 and pages.len.tolist() == [25] * n and int((pages.ref > 0).sum()) == 2 * n
    ops.kv_pages_trim(pages, seqs[: n // 2].contiguous())
    ops.kv_pages_compact(pages, layers, ops.Q4_0, n_live, work)
    torch.cuda.synchronize()
    assert int(n_live) == n and int(pages.table.max()) == n - 1 and (work[need:] == 0xAB).all()
