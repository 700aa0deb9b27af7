"""The measured calls of the batched, paged side of the framework: decode attention of a batch over a paged KV cache whose
sequences share a prefix, the prep that appends a batch's new rows, and the operators on the cache's pages.

The model has 16 attention layers (24 query / 4 KV heads, head_dim 256).  A page is `page` consecutive positions of a
layer's cache; the page tables [sequence][page of the sequence] serve every layer.  A used pool is scattered, so the
sequences' pages are a random permutation of the pool's.  Cache contents are synthetic: K / V ~N(0,1) with 1% of the key
rows scaled by 8, quantized as the append does it.
"""
import math

import torch

own = False

DEV = "cuda"
NH, NKV, HD, GRP, QD = 24, 4, 256, 6, 6144
VB = {"f16": 512, "q8_0": 256, "q4_0": 128}            # value bytes of one row of 256
POS_BYTES = {"f16": 4096, "q8_0": 2176, "q4_0": 1152}  # K + V values and scales of one position, all KV heads
EPS, THETA = 1e-6, 1e7


# ---- the cases ------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a handful of short chats: launches and latency
        {"name": "decode_3_q8_0", "kind": "decode", "kv": "q8_0", "page": 64, "n": 3, "nq": 1, "shared": 0, "own": 301},
        # a service's system prompt and its users' questions: the prefix counts once, the batch is mid-sized
        {"name": "decode_32_shared_8192_q8_0", "kind": "decode", "kv": "q8_0", "page": 64, "n": 32, "nq": 1,
         "shared": 8192, "own": 700},
        # many samples over one long document: the largest shared part, bound by the matrix cores
        {"name": "decode_128_shared_32768_q4_0", "kind": "decode", "kv": "q4_0", "page": 64, "n": 128, "nq": 1,
         "shared": 32768, "own": 1021},
        # unrelated ragged conversations: nothing is shared, bound by the cache's bytes
        {"name": "decode_24_ragged_16384_q4_0", "kind": "decode", "kv": "q4_0", "page": 128, "n": 24, "nq": 1,
         "shared": 0, "own": 16384},
        # speculative verify of 6 drafted tokens in several chats over one prompt that ends inside a page
        {"name": "verify7_5_shared_4093_f16", "kind": "decode", "kv": "f16", "page": 16, "n": 5, "nq": 7,
         "shared": 4093, "own": 513},
        # one decoded token in each of a few chats: norm, rotation, append
        {"name": "prep_6_q8_0", "kind": "prep", "kv": "q8_0", "page": 64, "n": 6, "nq": 1, "own": 300},
        # a verify step's rows of a large batch
        {"name": "prep_200x4_f16", "kind": "prep", "kv": "f16", "page": 32, "n": 200, "nq": 4, "own": 90},
        # three samples of one answer: the samples of the last request are dropped, the prompt is forked, and room for
        # the next token is made, which copies the partly filled last page for each sample
        {"name": "fork_3_of_517_q8_0", "kind": "fork", "kv": "q8_0", "page": 64, "layers": 16, "n": 3, "len": 517,
         "add": 1, "pages": 64},
        # the same for a large batch of samples of a long prompt, with room for a block of drafted tokens
        {"name": "fork_100_of_20011_f16", "kind": "fork", "kv": "f16", "page": 64, "layers": 16, "n": 100,
         "len": 20011, "add": 7, "pages": 768},
        # a small pool with a few holes
        {"name": "compact_48_q8_0", "kind": "compact", "kv": "q8_0", "page": 32, "layers": 2, "n": 4, "pages": 48,
         "used": 0.5},
        # a large pool that requests have come to and gone from for a while
        {"name": "compact_1500_q4_0", "kind": "compact", "kv": "q4_0", "page": 64, "layers": 16, "n": 40,
         "pages": 1500, "used": 0.55},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["decode"] * 5 + ["prep", "fork", "compact"])
    kv = rng.choice(list(VB))
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "decode":
        nq = rng.choice([1, 1, 1, 1, 2, 3, 5, 8])
        n = max(1, _log(rng, 1, 128) // nq)
        shared = 0 if rng.random() < 0.35 else _log(rng, 16, 32768)
        cap = min(16384, 200_000_000 // (n * POS_BYTES[kv]))
        return {"kind": kind, "kv": kv, "page": page, "n": n, "nq": nq, "shared": shared,
                "own": max(nq, _log(rng, 1, cap))}
    if kind == "prep":
        nq = rng.choice([1, 1, 2, 4, 7, 8])
        return {"kind": kind, "kv": kv, "page": page, "n": _log(rng, 1, 1000 // nq), "nq": nq,
                "own": max(nq, _log(rng, 8, 200))}
    if kind == "fork":
        n, length, add = _log(rng, 1, 120), _log(rng, 3, 20000), rng.choice([1, 1, 2, 7, 8, 60])
        return {"kind": kind, "kv": kv, "page": page, "layers": rng.choice([1, 4, 16]), "n": n, "len": length,
                "add": add, "pages": length // page + 1 + n * (add // page + 2) + _log(rng, 1, 64)}
    layers = rng.choice([1, 2, 4, 16])
    most = int(1_700_000_000 // (layers * page * POS_BYTES[kv]))
    n = _log(rng, 2, 40)
    return {"kind": kind, "kv": kv, "page": page, "layers": layers, "n": n, "pages": _log(rng, max(16, 2 * n), max(64, min(4000, most))),
            "used": rng.choice([0.3, 0.5, 0.7, 0.9])}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + salt) % (1 << 62))


def _rn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _quantize(x, kv):
    """Rows x [...][256] as the cache stores them: (value bytes [...][vb], fp16 scales [...][8] or None)."""
    if kv == "f16":
        return x.half().view(torch.uint8), None
    b = x.unflatten(-1, (8, 32))
    if kv == "q8_0":
        d = b.abs().amax(-1) / 127.0
        y = b * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))[..., None]
        q = (torch.sign(y) * torch.floor(y.abs() + 0.5)).to(torch.int8).view(torch.uint8)
        return q.flatten(-2), d.half()
    big = b.gather(-1, b.abs().argmax(-1, keepdim=True))[..., 0]
    d = big / -8.0
    y = b * torch.where(d != 0, 1.0 / d, torch.zeros_like(d))[..., None]
    q = (y + 8.5).to(torch.int32).clamp_(0, 15).to(torch.uint8)
    return (q[..., 0::2] | (q[..., 1::2] << 4)).flatten(-2), d.half()


def _pool(c, slots, g, layers=1, fill=True):
    """K and V of `layers` layers: values [2][layers][4][slots][vb], fp16 scales [2][layers][4][slots][8] or None."""
    vals = torch.zeros((2, layers, NKV, slots, VB[c["kv"]]), dtype=torch.uint8, device=DEV)
    scales = None if c["kv"] == "f16" else torch.zeros((2, layers, NKV, slots, 8), dtype=torch.float16, device=DEV)
    if fill:
        for i in range(2 * layers):
            for p in range(0, slots, 32768):
                m = min(32768, slots - p)
                x = _rn(g, NKV, m, HD)
                if i < layers:
                    x[torch.rand((NKV, m), generator=g, device=DEV) < 0.01] *= 8.0
                q, s = _quantize(x, c["kv"])
                vals[i // layers, i % layers, :, p:p + m] = q
                if s is not None:
                    scales[i // layers, i % layers, :, p:p + m] = s
    return vals, scales


def _ceil(a, b):
    return -(-a // b)


def _batch(c, seed):
    """Tables of n sequences over a scattered pool, the first c["shared"] positions in the same pages: (table [n][ld],
    len [n], pages).  Lengths are ragged: the longest has c["own"] positions of its own, the shortest about a third."""
    g = torch.Generator().manual_seed(seed % (1 << 62))
    n, nq, page, shared = c["n"], c["nq"], c["page"], c.get("shared", 0)
    lens = [shared + max(nq, c["own"] - (i * 2 * c["own"]) // (3 * n)) for i in range(n)]
    order = torch.randperm(n, generator=g).tolist()
    lens = [lens[i] for i in order]
    whole = shared // page                                # shared pages; a partly shared one is held as a copy each
    need = whole + sum(_ceil(m, page) - whole for m in lens)
    pages = need + need // 8 + 1
    perm = torch.randperm(pages, generator=g).tolist()
    ld = max(_ceil(m, page) for m in lens)
    table, at = [], whole
    for m in lens:
        k = _ceil(m, page) - whole
        table.append(perm[:whole] + perm[at:at + k] + [-1] * (ld - whole - k))
        at += k
    return _i32(table), _i32(lens), pages, max(lens)


def _share_partial(c, s):
    """The partly shared page's rows are the same in every sequence's copy of it."""
    page, shared = c["page"], c["shared"]
    r = shared % page
    if r:
        at = s["table"][:, shared // page].long()[:, None] * page + torch.arange(r, device=DEV)
        for t in (s["vals"], s["scales"]):
            if t is not None:
                t[:, :, :, at] = t[:, :, :, at[:1]].expand_as(t[:, :, :, at]).clone()


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = {"case": c}
    if c["kind"] in ("decode", "prep"):
        s["table"], s["len"], pages, s["max_len"] = _batch(c, seed)
        n, nq = c["n"], c["nq"]
        s["pages"] = pages
        s["vals"], s["scales"] = _pool(c, pages * c["page"], g, fill=c["kind"] == "decode")
        s["q"], s["gate"] = _rn(g, n * nq, NH, HD), _rn(g, n * nq, NH, HD)
        if c["kind"] == "decode":
            _share_partial(c, s)
            s["out"] = torch.empty((n * nq, NH, HD), dtype=torch.float16, device=DEV)
        else:
            s["qg"] = _rn(g, n * nq, NH, 2 * HD)
            s["k"], s["v"] = _rn(g, n * nq, NKV, HD), _rn(g, n * nq, NKV, HD)
            s["qn"] = 0.5 + torch.rand(HD, generator=g, device=DEV)
            s["kn"] = 0.5 + torch.rand(HD, generator=g, device=DEV)
            pos = (s["len"][:, None] - nq + torch.arange(nq, device=DEV)).long()
            s["slots"] = (s["table"].long().gather(1, pos // c["page"]) * c["page"] + pos % c["page"]).flatten()
        s["ref"] = torch.bincount(s["table"][s["table"] >= 0].flatten(), minlength=pages).int()
        return s
    cpu = torch.Generator().manual_seed(seed % (1 << 62))
    page, P, L = c["page"], c["pages"], c["layers"]
    perm = torch.randperm(P, generator=cpu)
    if c["kind"] == "fork":
        # sequence 0 holds the prompt, sequences 1..n are its samples
        k = _ceil(c["len"], page)
        table = torch.full((c["n"] + 1, _ceil(c["len"] + c["add"], page) + 1), -1, dtype=torch.int32)
        table[0, :k] = perm[:k].int()
        lens = torch.zeros(c["n"] + 1, dtype=torch.int32)
        lens[0] = c["len"]
        s["src"] = torch.zeros(c["n"], dtype=torch.int32, device=DEV)
        s["dst"] = torch.arange(1, c["n"] + 1, dtype=torch.int32, device=DEV)
        s["add"] = torch.full((c["n"],), c["add"], dtype=torch.int32, device=DEV)
        s["status"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    else:
        # n sequences of random lengths hold `used` of the pages, scattered; the second half share their first page
        n, used = c["n"], max(c["n"], int(P * c["used"]))
        cuts = torch.sort(torch.randperm(used - 1, generator=cpu)[:n - 1] + 1).values.tolist()
        table = torch.full((n, used - n + 1), -1, dtype=torch.int32)  # the longest that one of them can be
        lens = torch.zeros(n, dtype=torch.int32)
        for i, (a, b) in enumerate(zip([0] + cuts, cuts + [used])):
            table[i, :b - a] = perm[a:b].int()
            lens[i] = (b - a) * page - int(torch.randint(0, page, (1,), generator=cpu))
        table[n // 2:, 0] = table[n // 2, 0]
        s["n_live"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    ref = torch.bincount(table[table >= 0].flatten().long(), minlength=P).int()
    # tables, lengths and counts in one buffer, as an engine uploads them
    meta = torch.cat([table.flatten(), lens, ref]).to(DEV)
    s["meta"], s["meta0"] = meta, meta.clone()
    a, b = table.numel(), table.numel() + lens.numel()
    s["table"], s["len"], s["ref"] = meta[:a].view(table.shape), meta[a:b], meta[b:]
    s["vals"], s["scales"] = _pool(c, P * page, g, layers=L, fill=False)
    # page contents: any codes; scales and F16 values are finite
    if c["kv"] == "f16":
        s["vals"].view(torch.float16).copy_(torch.randint(-2048, 2048, (1 << 20,), generator=g, device=DEV).half().repeat(
            s["vals"].numel() // 2 // (1 << 20) + 1)[:s["vals"].numel() // 2].view(s["vals"].view(torch.float16).shape))
    else:
        s["vals"].copy_(torch.randint(0, 256, s["vals"].shape, generator=g, device=DEV, dtype=torch.uint8))
        s["scales"].copy_(0.01 * torch.randn(s["scales"].shape, generator=g, device=DEV))
    return s


# ---- one pass, by the framework -------------------------------------------------------------------------------------
def _handle(s):
    """The objects that a user's program keeps: the layers, the pages, the workspaces."""
    if "pg" not in s:
        import qwengine_amd.ops as ops
        c = s["case"]
        kvt = ops.KV_TYPES[c["kv"]]
        cap, v, d = s["vals"].shape[3], s["vals"], s["scales"]
        bits = lambda t: None if t is None else t.view(torch.int16)
        s["kvt"] = kvt
        s["layers"] = [ops.KVLayer(kvt, cap, v[0, i], v[1, i], bits(d if d is None else d[0, i]),
                                   bits(d if d is None else d[1, i])) for i in range(v.shape[1])]
        s["pg"] = ops.KVPages(s["table"], s["len"], s["ref"], c["page"])
        if c["kind"] == "decode":
            size = ops.attn_batch_work_bytes(c["n"], c["nq"], c["shared"], s["max_len"])
        elif c["kind"] == "prep":
            size = 0
        else:
            size = ops.kv_pages_work_bytes(s["pg"])
        s["work"] = torch.empty(size, dtype=torch.uint8, device=DEV)
    return s["layers"], s["pg"], s["work"]


def _run_own(s):
    import qwengine_amd.ops as ops
    c = s["case"]
    layers, pg, work = _handle(s)
    if c["kind"] == "decode":
        ops.attn_decode_batch(s["q"], s["gate"], layers[0], s["kvt"], pg, None, c["n"], c["nq"], c["shared"], s["max_len"],
                              s["out"], work)
    elif c["kind"] == "prep":
        ops.attn_prep_batch(s["qg"], s["k"], s["v"], s["qn"], s["kn"], pg, None, c["n"], c["nq"], THETA, EPS, s["kvt"],
                            layers[0], s["q"], s["gate"])
    elif c["kind"] == "fork":
        ops.kv_pages_trim(pg, s["dst"], None)
        ops.kv_pages_fork(pg, s["src"], s["dst"], work)
        ops.kv_pages_extend(pg, s["dst"], s["add"], layers, s["kvt"], s["status"], work)
    else:
        ops.kv_pages_compact(pg, layers, s["kvt"], s["n_live"], work)


# ---- the same in elementary operations ------------------------------------------------------------------------------
def _values(vals, scales, kv):
    """Rows in 32 bits."""
    if kv == "f16":
        return vals.view(torch.float16).float()
    if kv == "q8_0":
        q = vals.view(torch.int8).float()
    else:
        q = torch.stack([vals & 15, vals >> 4], -1).flatten(-2).float() - 8.0
    return (q.unflatten(-1, (8, 32)) * scales.float()[..., None]).flatten(-2)


def _rows(s, slots):
    """K and V rows of the slots: [2][4][*slots][256] in 32 bits."""
    d = None if s["scales"] is None else s["scales"][:, 0][:, :, slots]
    return _values(s["vals"][:, 0][:, :, slots], d, s["case"]["kv"])


def _plain_decode(s):
    c, page = s["case"], s["case"]["page"]
    n, nq, shared, most = c["n"], c["nq"], c["shared"], s["max_len"]
    lens = s["len"].long()
    slot = lambda row, j: row[..., j // page].clamp_min(0) * page + j % page
    table = s["table"].long()
    first = table[lens.argmax()]
    a, b = torch.arange(shared, device=DEV), torch.arange(shared, most, device=DEV)
    K0, V0 = _rows(s, slot(first, a))                        # [4][shared][256]
    K1, V1 = _rows(s, slot(table, b))                        # [4][n][own][256]
    x = s["q"].view(n, nq, NKV, GRP, HD).permute(2, 0, 1, 3, 4) / 16.0
    rows = x.reshape(NKV, n, nq * GRP, HD)
    S0 = (rows.reshape(NKV, n * nq * GRP, HD) @ K0.transpose(1, 2)).view(NKV, n, nq * GRP, shared)
    S = torch.cat([S0, rows @ K1.transpose(2, 3)], -1)
    sees = lens[:, None] - nq + torch.arange(nq, device=DEV) + 1
    masked = torch.arange(most, device=DEV) >= sees[..., None]               # [n][nq][most]
    S = S.masked_fill(masked.repeat_interleave(GRP, 1)[None], -math.inf)
    top = S.amax(-1, keepdim=True).clamp_min(-3e38)
    P = torch.exp(S - top)
    den = P.sum(-1, keepdim=True)
    P0, P1 = P[..., :shared], P[..., shared:]
    O = (P0.reshape(NKV, n * nq * GRP, shared) @ V0).view(NKV, n, nq * GRP, HD) + P1 @ V1
    O = torch.where(den > 0, O / den.clamp_min(1e-30), 0.0)
    O = O.view(NKV, n, nq, GRP, HD).permute(1, 2, 0, 3, 4).reshape(n * nq, NH, HD)
    s["out"].copy_(O / (1.0 + torch.exp(-s["gate"])))


def _plain_prep(s):
    c = s["case"]
    n, nq, page = c["n"], c["nq"], c["page"]
    pos = s["len"][:, None].long() - nq + torch.arange(nq, device=DEV)
    i = torch.arange(32, device=DEV, dtype=torch.float64)
    ang = (pos.flatten().double()[:, None] * THETA ** (-i / 32.0))[:, None]
    cos, sin = torch.cos(ang), torch.sin(ang)

    def prep(x, w):  # in 64 bits: the quantizer's borders
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
        lo, hi = x[..., :32], x[..., 32:64]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., 64:]], -1).float()

    s["q"].copy_(prep(s["qg"][..., :HD], s["qn"]))
    s["gate"].copy_(s["qg"][..., HD:])
    x = torch.stack([prep(s["k"], s["kn"]), s["v"]]).transpose(1, 2)          # [2][4][n nq][256]
    slots = (s["table"].long().gather(1, pos // page) * page + pos % page).flatten()
    q, d = _quantize(x.contiguous(), c["kv"])
    s["vals"][:, 0][:, :, slots] = q
    if d is not None:
        s["scales"][:, 0][:, :, slots] = d


def _plain_fork(s):
    c, page = s["case"], s["case"]["page"]
    table, lens, ref = s["table"], s["len"], s["ref"]
    src, dst, add = s["src"].long(), s["dst"].long(), s["add"].long()
    at = torch.arange(table.shape[1], device=DEV)
    held = lambda rows: at < ((lens[rows].long() + page - 1) // page)[:, None]
    # the samples' old pages are given back, the prompt's are held once more for each sample
    m = held(dst)
    ref.index_add_(0, table[dst][m].long(), torch.full((1,), -1, dtype=torch.int32, device=DEV).expand(int(m.sum())))
    m, rows = held(src), table[src]
    ref.index_add_(0, rows[m].long(), torch.ones(1, dtype=torch.int32, device=DEV).expand(int(m.sum())))
    rows = torch.where(m, rows, -1)
    # room: a page for each begun page past the present ones, and one for a partly filled last page that others hold
    have = lens[src].long()
    last = rows.gather(1, ((have - 1).clamp_min(0) // page)[:, None])[:, 0].long()
    part = (have % page != 0) & (add > 0) & (ref[last.clamp_min(0)] > 1)
    grow = (have + add + page - 1) // page - (have + page - 1) // page
    need = grow + part
    free = (ref == 0).nonzero()[:, 0]
    who = torch.repeat_interleave(torch.arange(c["n"], device=DEV), need)
    begin = need.cumsum(0) - need
    k = torch.arange(who.numel(), device=DEV)
    got = free[:who.numel()]
    where = (have + page - 1)[who] // page - part.long()[who] + (k - begin[who])
    copied = part[who] & (k == begin[who])
    old = last[who[copied]]
    rows[who, where] = got.int()
    ref[got] = 1
    ref.index_add_(0, old, torch.full((1,), -1, dtype=torch.int32, device=DEV).expand(old.numel()))
    table[dst] = rows
    lens[dst] = (have + add).int()
    r = torch.arange(page, device=DEV)
    filled = r < (have % page)[who[copied]][:, None]
    frm, to = ((p[:, None] * page + r)[filled] for p in (old, got[copied]))
    s["vals"][:, :, :, to] = s["vals"][:, :, :, frm]
    if s["scales"] is not None:
        s["scales"][:, :, :, to] = s["scales"][:, :, :, frm]
    s["status"].zero_()


def _plain_compact(s):
    page, table, lens, ref = s["case"]["page"], s["table"], s["len"], s["ref"]
    live = ref > 0
    at = torch.arange(ref.numel(), device=DEV)
    count = live.sum()
    frm, to = (live & (at >= count)).nonzero()[:, 0], (~live & (at < count)).nonzero()[:, 0]
    new = at.clone()
    new[frm] = to
    held = torch.arange(table.shape[1], device=DEV) < ((lens.long() + page - 1) // page)[:, None]
    table.copy_(torch.where(held, new[table.long().clamp_min(0)].int(), table))
    ref[to] = ref[frm]
    ref[frm] = 0
    s["n_live"].copy_(count)
    for t in (s["vals"], s["scales"]):
        if t is not None:
            t = t.view(*t.shape[:3], -1, page, t.shape[-1])
            t[:, :, :, to] = t[:, :, :, frm]


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "compact":
        s["meta"].copy_(s["meta0"])  # the pool as the requests left it; the pages to move still hold their rows
    if own:
        _run_own(s)
    else:
        {"decode": _plain_decode, "prep": _plain_prep, "fork": _plain_fork, "compact": _plain_compact}[kind](s)
    if kind == "decode":
        return {"out": s["out"]}
    if kind == "prep":  # the appended rows as the values they stand for
        v, d = s["vals"][:, 0][:, :, s["slots"]], s["scales"]
        if c["kv"] == "f16":
            v = v.view(torch.float16)
        elif c["kv"] == "q8_0":
            v = (v.view(torch.int8).unflatten(-1, (8, 32)) * d[:, 0][:, :, s["slots"]][..., None]).flatten(-2)
        else:
            v = torch.stack([v & 15, v >> 4], -1).view(torch.int8).flatten(-2) - 8
            v = (v.unflatten(-1, (8, 32)) * d[:, 0][:, :, s["slots"]][..., None]).flatten(-2)
        return {"q": s["q"], "gate": s["gate"], "rows": v}
    # page contents are moved, never computed: their codes have to be equal
    vals = s["vals"].view(torch.float16) if c["kv"] == "f16" else s["vals"]
    extra = {"status": s["status"]} if kind == "fork" else {"n_live": s["n_live"]}
    return {"table": s["table"], "len": s["len"], "ref": s["ref"], "vals": vals, "scales": s["scales"], **extra}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "decode":
        n, nq, page, shared = c["n"], c["nq"], c["page"], c["shared"]
        mine = [max(nq, c["own"] - (i * 2 * c["own"]) // (3 * n)) for i in range(n)]
        keys = sum(shared * nq + sum(m - nq + t + 1 for t in range(nq)) for m in mine)
        return {"bytes": (shared + sum(mine)) * POS_BYTES[c["kv"]] + n * nq * QD * (4 + 4 + 2) + 4 * n,
                "flops": 4.0 * QD * keys}
    if c["kind"] == "prep":
        tokens = c["n"] * c["nq"]
        return {"bytes": tokens * (2 * 4 * QD * 2 + 2 * 4 * NKV * HD + POS_BYTES[c["kv"]]), "flops": tokens * QD * 8.0}
    row = c["layers"] * POS_BYTES[c["kv"]]
    if c["kind"] == "fork":
        k = _ceil(c["len"], c["page"])
        return {"bytes": 2.0 * c["n"] * (c["len"] % c["page"]) * row + 4 * (k + 2 * c["n"] * (k + 2) + 2 * c["pages"]),
                "flops": 0.0}
    used = max(c["n"], int(c["pages"] * c["used"]))
    return {"bytes": 2.0 * (used * (c["pages"] - used) / c["pages"]) * c["page"] * row + 4 * (2 * used + 2 * c["pages"]),
            "flops": 0.0}


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------
def _row64(s, layer, which, head, slots):
    """Cache rows in 64 bits, one KV head: [slots][256]."""
    kv = s["case"]["kv"]
    b = s["vals"][which, layer, head][slots]
    if kv == "f16":
        return b.view(torch.float16).double()
    d = s["scales"][which, layer, head][slots].double().repeat_interleave(32, -1)
    if kv == "q8_0":
        return b.view(torch.int8).double() * d
    out = torch.empty((b.shape[0], HD), dtype=torch.float64, device=DEV)
    out[:, 0::2], out[:, 1::2] = (b % 16).double() - 8, (b // 16).double() - 8
    return out * d


def exact(case, seed):
    c, s = case, prepare(case, seed)
    page = c["page"]
    table, lens = s["table"].cpu().tolist(), s["len"].cpu().tolist()
    if c["kind"] == "decode":
        n, nq = c["n"], c["nq"]
        out = torch.zeros((n * nq, NH, HD), dtype=torch.float64, device=DEV)
        for b in range(n):
            j = torch.arange(lens[b], device=DEV)
            slots = s["table"][b].long()[j // page] * page + j % page
            for h in range(NKV):
                K, V = _row64(s, 0, 0, h, slots), _row64(s, 0, 1, h, slots)
                x = s["q"][b * nq:(b + 1) * nq, h * GRP:(h + 1) * GRP].double().reshape(-1, HD)
                sc = (x @ K.T / math.sqrt(HD)).view(nq, GRP, -1)
                for t in range(nq):
                    sc[t, :, lens[b] - nq + t + 1:] = -math.inf
                o = torch.softmax(sc, -1).view(nq * GRP, -1) @ V
                out[b * nq:(b + 1) * nq, h * GRP:(h + 1) * GRP] = o.view(nq, GRP, HD)
        return {"out": out * torch.sigmoid(s["gate"].double())}
    if c["kind"] == "prep":
        n, nq = c["n"], c["nq"]
        pos = torch.tensor([lens[b] - nq + t for b in range(n) for t in range(nq)], dtype=torch.float64, device=DEV)
        i = torch.arange(32, device=DEV, dtype=torch.float64)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), pos[:, None] * THETA ** (-2.0 * i / 64.0))

        def prep(x, w):
            x = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS) * w.double()
            z = torch.complex(x[..., :32], x[..., 32:64]) * turn[:, None]
            return torch.cat([z.real, z.imag, x[..., 64:]], -1)

        rows = None
        if c["kv"] == "f16":
            rows = torch.stack([prep(s["k"], s["kn"]), s["v"].double()]).transpose(1, 2).contiguous()
        return {"q": prep(s["qg"][..., :HD], s["qn"]), "gate": s["qg"][..., HD:].double(), "rows": rows}
    # the pages: a literal account, sequence by sequence
    ref = s["ref"].cpu().tolist()
    moves = []  # (from, to, rows)
    if c["kind"] == "fork":
        for d in s["dst"].cpu().tolist():
            table[d] = list(table[0])
            lens[d] = lens[0]
            for p in table[0][:_ceil(lens[0], page)]:
                ref[p] += 1
        for d in s["dst"].cpu().tolist():
            take = lambda: next(p for p, r in enumerate(ref) if r == 0)
            k = _ceil(lens[d], page)
            if lens[d] % page and ref[table[d][k - 1]] > 1:
                p, q = table[d][k - 1], take()
                ref[p] -= 1
                ref[q], table[d][k - 1] = 1, q
                moves.append((p, q, lens[d] % page))
            for i in range(k, _ceil(lens[d] + c["add"], page)):
                table[d][i] = take()
                ref[table[d][i]] = 1
            lens[d] += c["add"]
        extra = {"status": 0}
    else:
        live = [p for p, r in enumerate(ref) if r]
        holes = [p for p in range(len(live)) if ref[p] == 0]
        new = {p: p for p in live}
        new.update(zip([p for p in live if p >= len(live)], holes))
        moves = [(p, q, page) for p, q in new.items() if p != q]
        table = [[new[p] if i < _ceil(m, page) else p for i, p in enumerate(row)] for row, m in zip(table, lens)]
        for p, q, _ in moves:
            ref[q], ref[p] = ref[p], 0
        extra = {"n_live": len(live)}
    vals = s["vals"].view(torch.float16) if c["kv"] == "f16" else s["vals"]
    for p, q, m in moves:
        for t in (vals, s["scales"]):
            if t is not None:
                t[:, :, :, q * page:q * page + m] = t[:, :, :, p * page:p * page + m]
    wide = lambda t: None if t is None else t.double() if t.is_floating_point() else t
    return {"table": _i32(table), "len": _i32(lens), "ref": _i32(ref), "vals": wide(vals), "scales": wide(s["scales"]),
            **extra}
