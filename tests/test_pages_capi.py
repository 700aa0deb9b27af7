"""Batched, paged operators on the CPU: what they refuse before anything is launched, and the host's cut of a batch decode
(qwengine_amd/csrc/batch_plan.hpp)."""
import os
import subprocess

import pytest
import torch

import qwengine_amd.ops as ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x100000  # a non-null, aligned 'device pointer' that is never dereferenced: every call is rejected on the host


class FakePages:
    def __init__(self, n_seq=4, ld=8, n_pages=16, page=64, table=P, len=P, ref=P):
        self.v = ops._KVPagesC(table, len, ref, n_seq, ld, n_pages, page)

    def c(self):
        return self.v


def layer(kvt="q8_0", cap=1024, k=P, ks=P):
    f16 = kvt == "f16"
    return ops.KVLayer(ops._kvt(kvt), cap, k, P, None if f16 else ks, None if f16 else P)


def extend(pages=None, seqs=P, add=P, n=2, layers=None, kvt="q8_0", status=P, work=P):
    ops.kv_pages_extend(pages or FakePages(), seqs, add, layers if layers is not None else [layer(kvt)], kvt, status, work,
                        n=n, stream=0)


def fork(pages=None, src=P, dst=P, n=2, work=P):
    ops.kv_pages_fork(pages or FakePages(), src, dst, work, n=n, stream=0)


def trim(pages=None, seqs=P, lens=None, n=2):
    ops.kv_pages_trim(pages or FakePages(), seqs, lens, n=n, stream=0)


def compact(pages=None, layers=None, kvt="q8_0", n_live=P, work=P):
    ops.kv_pages_compact(pages or FakePages(), layers if layers is not None else [layer(kvt)], kvt, n_live, work, stream=0)


def prep(pages=None, seqs=None, n=2, nq=1, kvt="q8_0", kv=None, bufs=None):
    b = bufs or [P] * 7
    ops.attn_prep_batch(*b[:5], pages or FakePages(), seqs, n, nq, 1e7, 1e-6, kvt, kv or layer(kvt), b[5], b[6], stream=0)


def decode(pages=None, seqs=None, n=2, nq=1, shared=0, max_len=100, kvt="q8_0", kv=None, bufs=None, oq=None):
    b = bufs or [P] * 4
    ops.attn_decode_batch(b[0], b[1], kv or layer(kvt), kvt, pages or FakePages(), seqs, n, nq, shared, max_len, b[2], b[3],
                          oq, stream=0)


BAD_PAGES = [FakePages(table=None), FakePages(len=None), FakePages(ref=None), FakePages(n_seq=0), FakePages(ld=0),
             FakePages(n_pages=0), FakePages(page=0), FakePages(page=8), FakePages(page=48), FakePages(page=2048),
             FakePages(page=-64)]


@pytest.mark.parametrize("pages", BAD_PAGES, ids=range(len(BAD_PAGES)))
@pytest.mark.parametrize("call", [extend, fork, trim, compact, prep, decode], ids=lambda f: f.__name__)
def test_bad_page_tables(call, pages):
    with pytest.raises(ops.QwaError, match="page tables"):
        call(pages)
    assert ops.kv_pages_work_bytes(pages) == 0


@pytest.mark.parametrize("call", [extend, compact, prep, decode], ids=lambda f: f.__name__)
def test_bad_pools(call):
    one = (lambda kv: {"layers": [kv]}) if call in (extend, compact) else (lambda kv: {"kv": kv})
    with pytest.raises(ops.QwaError, match="capacity"):
        call(**one(layer(cap=1023)))
    with pytest.raises(ops.QwaError, match="aligned"):
        call(**one(layer(k=P + 8)))
    with pytest.raises(ops.QwaError, match="aligned"):
        call(**one(layer(ks=P + 8)))
    with pytest.raises(ops.QwaError, match="value buffers"):
        call(**one(layer(k=None)))
    with pytest.raises(ops.QwaError, match="scale buffers"):
        call(**one(layer(ks=None)))
    with pytest.raises(ops.QwaError, match="KV type"):
        call(kvt=7, **one(layer()))


def test_page_operator_arguments():
    for call in (extend, fork, trim):
        with pytest.raises(ops.QwaError, match="requests"):
            call(n=-1)
        with pytest.raises(ops.QwaError, match="requests"):
            call(n=1025, pages=FakePages(n_seq=5000))
    with pytest.raises(ops.QwaError, match="5 requests for 4 sequences"):
        fork(n=5)
    fork(n=0, src=None, dst=None)
    trim(n=0, seqs=None)
    for kw in ({"seqs": None}, {"add": None}, {"status": None}, {"work": None}):
        with pytest.raises(ops.QwaError, match="null"):
            extend(**kw)
    for kw in ({"src": None}, {"dst": None}, {"work": None}):
        with pytest.raises(ops.QwaError, match="null"):
            fork(**kw)
    with pytest.raises(ops.QwaError, match="null"):
        trim(seqs=None)
    for kw in ({"n_live": None}, {"work": None}):
        with pytest.raises(ops.QwaError, match="null"):
            compact(**kw)
    for call in (extend, fork, compact):
        with pytest.raises(ops.QwaError, match="aligned"):
            call(work=P + 4)
    for call in (extend, compact):
        for layers in ([], [layer()] * 33):
            with pytest.raises(ops.QwaError, match="layers"):
                call(layers=layers)


def test_batch_call_arguments():
    for call in (prep, decode):
        for nq in (0, 9, -1):
            with pytest.raises(ops.QwaError, match="queries"):
                call(nq=nq)
        for n in (0, -3, 1025):
            with pytest.raises(ops.QwaError, match="sequences"):
                call(n=n, seqs=P)
        with pytest.raises(ops.QwaError, match="5 batch rows for 4"):
            call(n=5)
        for i in range(7 if call is prep else 4):
            for v, what in ((None, "null"), (P + 4, "aligned")):
                bufs = [P] * 7
                bufs[i] = v
                if call is decode:
                    bufs = bufs[:4]
                with pytest.raises(ops.QwaError, match=what):
                    call(bufs=bufs)
    for shared, most in ((-1, 100), (101, 100), (0, 0), (0, -5), (0, 513), (0, 262145)):
        with pytest.raises(ops.QwaError, match="max_len"):
            decode(shared=shared, max_len=most)
        if most != 513:
            assert ops.attn_batch_work_bytes(2, 1, shared, most) == 0
    with pytest.raises(ops.QwaError, match="ActQ8"):
        decode(oq=ops.ActQ8(P, None, P))
    assert ops.attn_batch_work_bytes(0, 1, 0, 10) == 0 and ops.attn_batch_work_bytes(1, 9, 0, 10) == 0


def test_tensor_arguments_are_checked():
    """Tensors of another type, of too few entries or in host memory never reach the library."""
    i64 = torch.zeros(4, dtype=torch.int64)
    i32 = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ops.QwaError, match="seqs"):
        extend(seqs=i64)
    with pytest.raises(ops.QwaError, match="4 entries, 5 wanted"):
        extend(seqs=i32, n=5)
    with pytest.raises(ops.QwaError, match="not in GPU memory"):
        extend(seqs=i32)
    with pytest.raises(ops.QwaError, match="q: "):
        decode(bufs=[torch.zeros(4, dtype=torch.float16), P, P, P])
    with pytest.raises(ops.QwaError, match="2 sequences with 3 lengths"):
        ops.KVPages(torch.zeros((2, 4), dtype=torch.int32), torch.zeros(3, dtype=torch.int32), i32, 64).c()


def test_tensor_sizes_and_layer_types_are_checked():
    """Buffers of too few rows, and layers of another type than the call's, never reach the library."""
    f32 = lambda n: torch.zeros(n)
    rows = 2 * 6144
    for i in range(2):
        bufs = [P] * 4
        bufs[i] = f32(rows - 1)
        with pytest.raises(ops.QwaError, match=f"{rows - 1} entries, {rows} wanted"):
            decode(bufs=bufs)
    with pytest.raises(ops.QwaError, match="out16: 6144 entries"):
        decode(bufs=[P, P, torch.zeros(6144, dtype=torch.float16), P])
    for i, want in enumerate([2 * rows, 2048, 2048, 256, 256, rows, rows]):
        bufs = [P] * 7
        bufs[i] = f32(want - 1)
        with pytest.raises(ops.QwaError, match=f"{want - 1} entries, {want} wanted"):
            prep(bufs=bufs)
    with pytest.raises(ops.QwaError, match="oq.d"):
        decode(oq=ops.ActQ8(P, f32(rows // 32 - 1), P))
    with pytest.raises(ops.QwaError, match="oq.q: torch.int8 wanted"):
        decode(oq=ops.ActQ8(f32(rows), P, P))
    for call in (prep, decode):
        with pytest.raises(ops.QwaError, match="layer of KV type"):
            call(kvt="q4_0", kv=layer("q8_0"))
    for call in (extend, compact):
        with pytest.raises(ops.QwaError, match="layer of KV type"):
            call(kvt="f16", layers=[layer("f16"), layer("q8_0")])
        with pytest.raises(ops.QwaError, match="not in GPU memory"):
            call(layers=[ops.KVLayer.allocate("q8_0", 1024, device="cpu")])
        sparse = ops.KVLayer.allocate("q8_0", 2048, device="cpu")
        sparse.vs = sparse.vs[:, ::2]
        with pytest.raises(ops.QwaError, match="contiguous"):
            call(layers=[sparse])


PLAN = r'''
#include <stdio.h>
#include "batch_plan.hpp"
using namespace qwa;
#define CHECK(c, ...) do { if (!(c)) { fprintf(stderr, __VA_ARGS__); return 1; } } while (0)
int main() {
    const int ns[] = {1, 2, 3, 7, 31, 128, 1000, 1024}, lens[] = {1, 15, 16, 127, 128, 129, 4093, 33000, MAX_POS};
    for (int n : ns) for (int nq = 1; nq <= MAXQ; nq++) for (int most : lens) for (int sh : lens) {
        for (int shared : {0, sh}) {
            if (shared > most) continue;
            const BatchPlan p = batch_plan(n, nq, shared, most);
            const BatchWork w = batch_work(p, n, nq);
            const size_t rows = (size_t)n * nq * NH;
            CHECK(p.groups * p.rt_own * 16 >= nq * GRP && p.rt_own <= BT_MAXRT, "rows of a sequence\n");
            CHECK(shared == 0 || (p.nt > 0) != (p.ns_shared > 0), "the shared positions: one kind of workgroup\n");
            CHECK(p.nt == 0 || p.blocks * BT_TROWS >= n * nq * GRP, "rows of the batch\n");
            CHECK(p.nt * (long long)PF_TILE < shared + PF_TILE, "an empty range\n");
            CHECK(p.groups_shared * p.rt_shared * 16 >= n * nq * GRP, "rows of the batch\n");
            CHECK(p.nt > 0 || (long long)p.ns_shared * p.len_shared >= shared, "shared\n");
            CHECK(p.ns_shared == 0 || (long long)(p.ns_shared - 1) * p.len_shared < shared, "an empty range\n");
            CHECK(p.len_shared % 16 == 0, "a range that begins inside 16 keys\n");
            CHECK((most > shared) == (p.wgs > 0), "own\n");
            CHECK(p.wgs + p.ns_shared + p.nt >= 1, "no range\n");
            CHECK((long long)p.blocks * p.nt * NKV < 1LL << 31 && (long long)p.wgs * NKV * p.groups < 1LL << 31 &&
                  (long long)p.ns_shared * NKV * p.groups_shared < 1LL << 31, "grid\n");
            const size_t own = p.wgs ? (size_t)NKV * (p.wgs + n) * nq * GRP : 0;
            CHECK(w.bytes >= rows * (p.nt * (HD * 2 + 16) + p.ns_shared * (HD * 4 + 8)) + own * (HD * 4 + 8) + 4 * (n + 1) &&
                  w.tile_ml % 16 == 0 && w.o % 16 == 0 && w.ml % 8 == 0 && w.own_o % 16 == 0 && w.own_ml % 8 == 0 &&
                  w.begin % 4 == 0, "work buffer\n");
        }
    }
    // slices and segments: every step lies in the slice that the combine looks for it in, segment numbers are unique
    for (int wgs : {1, 2, 7, 192}) for (int total : {1, 2, 5, 191, 192, 193, 2048, 2097152}) {
        const int slices = std::min(wgs, total);
        for (int w = 0; w < slices; w++) {
            const long long lo = (long long)w * total / slices, hi = (long long)(w + 1) * total / slices;
            CHECK(lo < hi, "empty slice\n");
            for (long long x : {lo, (lo + hi) / 2, hi - 1})
                if (x < hi) CHECK(((x + 1) * slices - 1) / total == w, "step %lld of %d in slice %d\n", x, total, w);
        }
    }
    return 0;
}
'''


def test_batch_plan(tmp_path):
    src = tmp_path / "plan.cpp"
    src.write_text(PLAN)
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-O1", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "qwengine_amd", "csrc"), str(src), "-o", exe], check=True)
    subprocess.run([exe], check=True)
