"""The operators on chunks and evictions on the CPU: what they refuse before anything is launched, and the host's bounds of how the
device cuts a call (qwengine_amd/csrc/chunk_plan.hpp)."""
import ctypes
import os
import subprocess

import pytest
import torch

import qwengine_amd.ops as ops
from test_pages_capi import BAD_PAGES, P, ROOT, FakePages, layer


def prep(pages=None, seqs=None, off=P, n=2, rows=9, kvt="q8_0", kv=None, bufs=None):
    b = bufs or [P] * 7
    ops.attn_prep_rows_batch(*b[:5], pages or FakePages(), seqs, off, n, rows, 1e7, 1e-6, kvt, kv or layer(kvt), b[5], b[6],
                             stream=0)


def prefill(pages=None, seqs=None, off=P, n=2, rows=9, max_len=100, kvt="q8_0", kv=None, bufs=None, lse=None):
    b = bufs or [P] * 4
    ops.attn_prefill_batch(b[0], b[1], kv or layer(kvt), kvt, pages or FakePages(), seqs, off, n, rows, max_len, b[2], b[3],
                           lse=lse, stream=0)


def weights(pages=None, seqs=None, off=P, n=2, rows=9, max_len=100, kvt="q8_0", kv=None, bufs=None, lse=P, mass=P):
    b = bufs or [P] * 2
    ops.attn_weights_batch(b[0], lse, kv or layer(kvt), kvt, pages or FakePages(), seqs, off, n, rows, max_len, mass, b[1],
                           stream=0)


def evict(pages=None, seqs=P, keep=P, n=2, recent=3, max_keep=20, layers=None, kvt="q8_0", kv=None, mass=P, dropped=P, status=P,
          work=P):
    layers = [kv or layer(kvt)] if layers is None else layers
    ops.kv_pages_evict(pages or FakePages(), seqs, keep, recent, max_keep, layers, kvt, mass, dropped, status, work, n=n, stream=0)


CHUNKS = [prep, prefill, weights]
named = pytest.mark.parametrize("call", CHUNKS + [evict], ids=lambda f: f.__name__)
chunks = pytest.mark.parametrize("call", CHUNKS, ids=lambda f: f.__name__)


@named
def test_bad_page_tables(call):
    for pages in BAD_PAGES:
        with pytest.raises(ops.QwaError, match="page tables"):
            call(pages)
        assert ops.kv_pages_evict_work_bytes(pages, 2, 1, 20) == 0


@named
def test_bad_pools(call):
    for kv, what in ((layer(cap=1023), "capacity"), (layer(k=P + 8), "aligned"), (layer(ks=P + 8), "aligned"),
                     (layer(k=None), "value buffers"), (layer(ks=None), "scale buffers"), (layer("f16"), "layer of KV type")):
        with pytest.raises(ops.QwaError, match=what):
            call(kv=kv)
    with pytest.raises(ops.QwaError, match="KV type"):
        call(kvt=7, kv=layer())


@chunks
def test_chunk_arguments(call):
    for n in (0, -3, 1025):
        with pytest.raises(ops.QwaError, match="sequences"):
            call(n=n, seqs=P)
    with pytest.raises(ops.QwaError, match="5 batch rows for 4"):
        call(n=5)
    for rows in (0, -1, 65537):
        with pytest.raises(ops.QwaError, match="rows"):
            call(rows=rows)
    with pytest.raises(ops.QwaError, match="null"):
        call(off=None)
    for i in range({prep: 7, prefill: 4, weights: 2}[call]):
        for v, what in ((None, "null"), (P + 4, "aligned")):
            bufs = [P] * {prep: 7, prefill: 4, weights: 2}[call]
            bufs[i] = v
            with pytest.raises(ops.QwaError, match=what):
                call(bufs=bufs)
    if call is not prep:
        for most in (0, -5, 513, 262145):
            with pytest.raises(ops.QwaError, match="max_len"):
                call(max_len=most)
    if call is weights:
        for kw in ({"lse": None}, {"mass": None}):
            with pytest.raises(ops.QwaError, match="null"):
                weights(**kw)


def test_evict_arguments():
    for n in (-1, 1025):
        with pytest.raises(ops.QwaError, match="requests"):
            evict(n=n)
    for most in (-1, 262145):
        with pytest.raises(ops.QwaError, match="max_keep"):
            evict(max_keep=most)
    with pytest.raises(ops.QwaError, match="recent"):
        evict(recent=-1)
    for kw in ("seqs", "keep", "mass", "dropped", "status", "work"):
        with pytest.raises(ops.QwaError, match="null"):
            evict(**{kw: None})
    for kw in ("mass", "work"):
        with pytest.raises(ops.QwaError, match="aligned"):
            evict(**{kw: P + 4})
    for layers in ([], [layer()] * 33):
        with pytest.raises(ops.QwaError, match="layers"):
            evict(layers=layers)


def test_tensors_are_checked():
    """Tensors of another type, of too few entries or in host memory never reach the library."""
    f32, i32 = torch.zeros, torch.zeros(2, dtype=torch.int32)
    for call in CHUNKS:
        with pytest.raises(ops.QwaError, match="off: 2 entries, 3 wanted"):
            call(off=i32)
        with pytest.raises(ops.QwaError, match="off: torch.int32 wanted"):
            call(off=torch.zeros(3, dtype=torch.int64))
        with pytest.raises(ops.QwaError, match="seqs: not in GPU memory"):
            call(seqs=i32)
    for i, want in enumerate([9 * 12288, 9 * 1024, 9 * 1024, 256, 256, 9 * 6144, 9 * 6144]):
        bufs = [P] * 7
        bufs[i] = f32(want - 1)
        with pytest.raises(ops.QwaError, match=f"{want - 1} entries, {want} wanted"):
            prep(bufs=bufs)
    for i in range(2):
        bufs = [P] * 4
        bufs[i] = f32(9 * 6144 - 1)
        with pytest.raises(ops.QwaError, match="wanted"):
            prefill(bufs=bufs)
    with pytest.raises(ops.QwaError, match="out16: torch.float16 wanted"):
        prefill(bufs=[P, P, f32(9 * 6144), P])
    for call in (prefill, weights):
        with pytest.raises(ops.QwaError, match="lse: 215 entries, 216 wanted"):
            call(lse=f32(215))
    want = 4 * 4 * 8 * 64  # sequences, heads, positions of a table row
    with pytest.raises(ops.QwaError, match=f"mass: {want - 1} entries, {want} wanted"):
        weights(mass=f32(want - 1))
    with pytest.raises(ops.QwaError, match=f"mass: {2 * want - 1} entries, {2 * want} wanted"):
        evict(layers=[layer(), layer()], mass=f32(2 * want - 1))
    for kw in ("seqs", "keep", "dropped"):
        with pytest.raises(ops.QwaError, match=f"{kw}: 2 entries, 3 wanted"):
            evict(n=3, **{kw: i32})


def test_small_workspaces_are_refused():
    L, pc, kv = ops.lib(), ctypes.byref(FakePages().c()), ctypes.byref(layer().c())
    calls = [
        (ops.attn_prefill_batch_work_bytes(2, 9, 100), lambda size: L.qwa_attn_prefill_batch(
            P, P, kv, ops.Q8_0, pc, None, P, 2, 9, 100, P, None, P, size, None)),
        (ops.attn_weights_batch_work_bytes(2, 9, 100), lambda size: L.qwa_attn_weights_batch(
            P, P, kv, ops.Q8_0, pc, None, P, 2, 9, 100, P, P, size, None)),
        (ops.kv_pages_evict_work_bytes(FakePages(), 2, 1, 20), lambda size: L.qwa_kv_pages_evict(
            pc, P, P, 2, 3, 20, kv, 1, ops.Q8_0, P, P, P, P, size, None))]
    for need, call in calls:
        assert need > 0
        for size in (0, 1, need // 2, need - 1):
            assert call(size) == 2  # QWA_ERR_RANGE
            assert f"workspace of {size} bytes, the call needs {need}" in L.qwa_last_error().decode()


def test_sizes_of_invalid_calls():
    for size in (ops.attn_prefill_batch_work_bytes, ops.attn_weights_batch_work_bytes):
        for args in ((0, 9, 100), (1025, 9, 100), (2, 0, 100), (2, 65537, 100), (2, 9, 0), (2, 9, 262145)):
            assert size(*args) == 0
        # a larger call's buffer does for a smaller one
        assert 0 < size(1, 1, 1) <= size(2, 9, 100) <= size(3, 1000, 5000) <= size(1024, 65536, 262144)
    for args in ((-1, 1, 20), (1025, 1, 20), (2, 0, 20), (2, 33, 20), (2, 1, -1), (2, 1, 262145)):
        assert ops.kv_pages_evict_work_bytes(FakePages(), *args) == 0


PLAN = r'''
#include <stdio.h>
#include <random>
#include <vector>
#include "chunk_plan.hpp"
using namespace qwa;
#define CHECK(c, ...) do { if (!(c)) { fprintf(stderr, __VA_ARGS__); return 1; } } while (0)
int main() {
    std::mt19937 r(5);
    auto upto = [&](int m) { return (int)(r() % (unsigned)(m + 1)); };
    for (int round = 0; round < 4000; round++) {
        const int n = 1 + upto(round % 3 == 0 ? 1023 : 20), rows = 1 + upto(round % 5 == 0 ? 65535 : 3000), most = 1 + upto(round % 2 ? 500 : 40000);
        const ChunkPlan p = chunk_plan(n, rows, most);
        const WeightsPlan q = weights_plan(n, rows, most);
        const ChunkWork w = chunk_work(p);
        const WeightsWork x = weights_work(q, most);
        // chunks as the device may find them: their rows are disjoint
        int left = rows;
        long long blocks = 0, images = 0, wblocks = 0, parts = 0, multi = 0;
        for (int b = 0; b < n; b++) {
            int c = round % 7 == 0 ? rows / n : round % 7 == 1 ? (b == 0 ? rows : 0) : upto(left);
            if (c > left) c = left;
            left -= c;
            const int nb = (GRP * c + CH_ROWS - 1) / CH_ROWS, wb = (GRP * c + CW_ROWS - 1) / CW_ROWS;
            blocks += nb;
            images += nb >= CH_IMG_BLOCKS;
            wblocks += wb;
            if (wb > 1) parts += wb, multi++;
            CHECK(nb == 0 || std::min(CH_ROWS, GRP * c) <= p.rows, "rows of a block\n");
        }
        CHECK(blocks <= p.blocks && images <= p.images, "%lld blocks, %lld with images: %d, %d\n", blocks, images, p.blocks, p.images);
        CHECK(wblocks <= q.blocks && parts <= q.parts && multi <= q.parts / 2, "weights: %lld blocks, %lld places\n", wblocks, parts);
        CHECK(p.images == 0 || p.tiles >= (most + PF_TILE - 1) / PF_TILE, "room for one sequence\n");
        CHECK(p.slices >= 1 && p.slices <= CH_SLICES && q.slices >= 1 && q.slices <= CH_SLICES, "slices\n");
        // tiles fit 32 bits
        CHECK((long long)p.blocks * ((MAX_POS + PF_TILE - 1) / PF_TILE) < 1LL << 31, "tiles\n");
        CHECK(w.o % 16 == 0 && w.ml % 16 == 0 && w.blocks % 16 == 0 && w.list % 16 == 0 && w.head % 16 == 0, "alignment\n");
        CHECK(x.blocks % 16 == 0 && x.list % 16 == 0 && x.head % 16 == 0, "alignment\n");
        CHECK(w.bytes >= (size_t)NKV * p.tiles * sizeof(ChunkImage) + (size_t)NKV * p.slices * 2 * p.rows * (HD * 4 + 16), "bytes\n");
    }
    return 0;
}
'''


def test_chunk_plan(tmp_path):
    src = tmp_path / "plan.cpp"
    src.write_text(PLAN)
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-O1", "-I", os.path.join(ROOT, "include"), "-I",
                    os.path.join(ROOT, "qwengine_amd", "csrc"), str(src), "-o", exe], check=True)
    subprocess.run([exe], check=True)
