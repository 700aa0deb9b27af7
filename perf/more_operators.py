"""The measured calls of prompts and evictions on the paged side of the framework: the prep and the attention of a batch of
chunks (any number of new tokens for each sequence) over a paged KV cache, the attention weight that its positions gather,
and the eviction of the positions that gathered least.

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
# Chunk cases: `n` chunks of at most `chunk` and at least about half as many tokens, and `ones` sequences that decode a
# token; the sequence of the first chunk has `past` positions before it, the last sequence of the batch about a third of them.
def listed():
    return [
        # the next turn of two short chats: launches and latency
        {"name": "prefill_2x20_at_300_q8_0", "kind": "prefill", "kv": "q8_0", "page": 64, "n": 2, "chunk": 20, "ones": 0,
         "past": 300, "lse": False},
        # a serving step: a prompt's chunk goes along with the tokens that the other sequences decode
        {"name": "prefill_1x499_and_23x1_at_8192_q4_0", "kind": "prefill", "kv": "q4_0", "page": 64, "n": 1, "chunk": 499,
         "ones": 23, "past": 8192, "lse": False},
        # new prompts of different lengths, with the rows' log sums for the weights
        {"name": "prefill_6x1021_at_0_f16", "kind": "prefill", "kv": "f16", "page": 32, "n": 6, "chunk": 1021, "ones": 0,
         "past": 0, "lse": True},
        # the next chunk of a long document: the largest, bound by the matrix cores
        {"name": "prefill_1x1024_at_32768_q8_0", "kind": "prefill", "kv": "q8_0", "page": 64, "n": 1, "chunk": 1024,
         "ones": 0, "past": 32768, "lse": False},
        # the rows of the small call: norm, rotation, append
        {"name": "prep_2x20_at_300_q8_0", "kind": "prep", "kv": "q8_0", "page": 64, "n": 2, "chunk": 20, "ones": 0,
         "past": 300},
        # those of a step of prompts and decoded tokens
        {"name": "prep_5x700_and_40x1_at_900_q4_0", "kind": "prep", "kv": "q4_0", "page": 128, "n": 5, "chunk": 700,
         "ones": 40, "past": 900},
        # the weights of the last questions' tokens in a few chats
        {"name": "weights_3x32_at_1000_q8_0", "kind": "weights", "kv": "q8_0", "page": 64, "n": 3, "chunk": 32, "ones": 0,
         "past": 1000},
        # those of a decoded token in each of a batch of long sequences: bound by the keys' bytes
        {"name": "weights_16x1_at_16000_f16", "kind": "weights", "kv": "f16", "page": 64, "n": 0, "chunk": 1, "ones": 16,
         "past": 16000},
        # those of a prompt's whole chunk: bound by the matrix cores
        {"name": "weights_1x1000_at_16384_q4_0", "kind": "weights", "kv": "q4_0", "page": 64, "n": 1, "chunk": 1000,
         "ones": 0, "past": 16384},
        # two chats cut to a small budget: launches and latency
        {"name": "evict_2_of_600_to_256_q8_0", "kind": "evict", "kv": "q8_0", "page": 64, "layers": 16, "n": 2,
         "len": 600, "keep": 256, "recent": 32, "shared": 0},
        # one long document cut to an eighth
        {"name": "evict_1_of_32768_to_4096_q4_0", "kind": "evict", "kv": "q4_0", "page": 64, "layers": 16, "n": 1,
         "len": 32768, "keep": 4096, "recent": 256, "shared": 0},
        # a batch that a common prompt was forked to, cut to a quarter: pages that others hold are left to them
        {"name": "evict_6_of_8000_to_2000_f16", "kind": "evict", "kv": "f16", "page": 64, "layers": 16, "n": 6,
         "len": 8000, "keep": 2000, "recent": 128, "shared": 1000},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _cost(c):
    """(tokens, (query, key) pairs, entries of the scores of the sequences with a chunk, padded to the longest)"""
    shape = _shape(c)
    pairs = sum(k * (m - k) + k * (k + 1) // 2 for k, m in shape)
    return sum(k for k, _ in shape), pairs, (c["n"] * c["chunk"] + c["ones"]) * NH * (c["past"] + c["chunk"])


def draw(rng):
    kind = rng.choice(["prefill"] * 4 + ["weights"] * 2 + ["prep", "evict"])
    kv = rng.choice(list(VB))
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "evict":
        layers, n = rng.choice([1, 4, 16]), _log(rng, 1, 16)
        most = max(256, min(32768, int(2e9 // (layers * n * POS_BYTES[kv]))))
        length = _log(rng, 100, most)
        keep = _log(rng, 16, max(17, length // 2))
        return {"kind": kind, "kv": kv, "page": page, "layers": layers, "n": n, "len": length, "keep": keep,
                "recent": rng.choice([0, 1, keep // 8, keep // 2]), "shared": rng.choice([0, 0, length // 10])}
    while True:
        c = {"kind": kind, "kv": kv, "page": page, "n": _log(rng, 1, 12), "chunk": _log(rng, 1, 1024),
             "ones": rng.choice([0, 0, _log(rng, 1, 48)]), "past": rng.choice([0, _log(rng, 16, 32768), _log(rng, 16, 32768)])}
        if kind == "prefill":
            c["lse"] = rng.random() < 0.5
        tokens, pairs, scores = _cost(c)
        if kind == "prep" and tokens <= 3500 and c["past"] <= 4096 or kind != "prep" and pairs <= 3.3e7 and scores <= 1.2e9 and \
                (c["n"] + c["ones"]) * (c["past"] + c["chunk"]) <= 300000:
            return c


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed, salt=0):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + salt) % (1 << 62))


def _rn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _ceil(a, b):
    return -(-a // b)


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


def _pool(c, slots, g):
    """K and V of one layer: values [2][4][slots][vb], fp16 scales [2][4][slots][8] or None."""
    vals = torch.empty((2, NKV, slots, VB[c["kv"]]), dtype=torch.uint8, device=DEV)
    scales = None if c["kv"] == "f16" else torch.empty((2, NKV, slots, 8), dtype=torch.float16, device=DEV)
    for i in range(2):
        for p in range(0, slots, 32768):
            m = min(32768, slots - p)
            x = _rn(g, NKV, m, HD)
            if i == 0:
                x[torch.rand((NKV, m), generator=g, device=DEV) < 0.01] *= 8.0
            q, d = _quantize(x, c["kv"])
            vals[i, :, p:p + m] = q
            if d is not None:
                scales[i, :, p:p + m] = d
    return vals, scales


def _shape(c):
    """(tokens, positions with them) of each sequence, before the batch is shuffled"""
    n, m = c["n"], c["n"] + c["ones"]
    counts = [max(1, c["chunk"] - i * c["chunk"] // (2 * n)) for i in range(n)] + [1] * c["ones"]
    return [(k, k + c["past"] - (2 * i * c["past"]) // (3 * m)) for i, k in enumerate(counts)]


def _prepare_chunks(c, s, seed):
    cpu, g = torch.Generator().manual_seed(seed % (1 << 62)), _gen(seed)
    shape = _shape(c)
    shape = [shape[i] for i in torch.randperm(len(shape), generator=cpu).tolist()]
    page = c["page"]
    need = [_ceil(m, page) for _, m in shape]
    pages = sum(need) + sum(need) // 8 + 1
    perm, table, at = torch.randperm(pages, generator=cpu).tolist(), [], 0
    for k in need:
        table.append(perm[at:at + k] + [-1] * (max(need) - k))
        at += k
    off = [0]
    for k, _ in shape:
        off.append(off[-1] + k)
    rows = _ceil(off[-1], 8) * 8  # the step's buffers; the rows behind the last sequence's are nobody's
    s["table"], s["len"], s["off"] = _i32(table), _i32([m for _, m in shape]), _i32(off)
    s["ref"] = torch.bincount(s["table"][s["table"] >= 0].flatten(), minlength=pages).int()
    s["rows"], s["max_len"], s["tokens"], s["n"] = rows, max(m for _, m in shape), off[-1], len(shape)
    s["vals"], s["scales"] = _pool(c, pages * page, g)
    # the sequences with a chunk and those with one token, each kind padded to its longest: batch rows, tokens, positions
    s["groups"] = []
    for kind in (False, True):
        b = [i for i, (k, _) in enumerate(shape) if (k == 1) == kind]
        if b:
            s["groups"].append((torch.tensor(b, device=DEV), max(shape[i][0] for i in b), max(shape[i][1] for i in b)))
    if c["kind"] == "prep":
        s["qg"], s["k"], s["v"] = _rn(g, rows, NH, 2 * HD), _rn(g, rows, NKV, HD), _rn(g, rows, NKV, HD)
        s["qn"] = 0.5 + torch.rand(HD, generator=g, device=DEV)
        s["kn"] = 0.5 + torch.rand(HD, generator=g, device=DEV)
        s["q"], s["gate"] = torch.zeros((rows, NH, HD), device=DEV), torch.zeros((rows, NH, HD), device=DEV)
        s["seq"] = torch.repeat_interleave(torch.arange(s["n"], device=DEV), torch.tensor([k for k, _ in shape], device=DEV))
        first = s["len"].long() - s["off"][1:].long()
        s["pos"] = first[s["seq"]] + torch.arange(s["tokens"], device=DEV)
        s["slots"] = s["table"].long()[s["seq"], s["pos"] // page] * page + s["pos"] % page
        return
    s["q"], s["gate"] = _rn(g, rows, NH, HD), _rn(g, rows, NH, HD)
    if c["kind"] == "prefill":
        s["out"] = torch.zeros((rows, NH, HD), dtype=torch.float16, device=DEV)
        s["lse"] = torch.zeros((rows, NH), device=DEV) if c["lse"] else None
        return
    # what the attention of these tokens left, and the weights that the positions gathered before
    s["lse"] = torch.zeros((rows, NH), device=DEV)
    for group in s["groups"]:
        S, real, at = _scores(s, group)
        s["lse"][at[real]] = torch.logsumexp(S, -1)[real]
    ld = s["table"].shape[1] * page
    s["mass"] = 0.01 * torch.exp(2.0 * _rn(g, s["n"], NKV, ld))


def _prepare_evict(c, s, seed):
    cpu, g = torch.Generator().manual_seed(seed % (1 << 62)), _gen(seed)
    n, page, L = c["n"], c["page"], c["layers"]
    lens = [c["len"] - (i * c["len"]) // (3 * n) for i in range(n)]
    lens = [lens[i] for i in torch.randperm(n, generator=cpu).tolist()]
    whole = min(c["shared"], min(lens)) // page if n > 1 else 0
    need = [_ceil(m, page) - whole for m in lens]
    fresh = _ceil(c["keep"], page) * n  # room for the copies of shared pages
    pages = whole + sum(need) + fresh
    perm, table, at = torch.randperm(pages, generator=cpu).tolist(), [], whole
    ld = max(need) + whole
    for k in need:
        table.append(perm[:whole] + perm[at:at + k] + [-1] * (ld - whole - k))
        at += k
    table = torch.tensor(table, dtype=torch.int32)
    ref = torch.bincount(table[table >= 0].flatten().long(), minlength=pages).int()
    # tables, lengths and counts in one buffer, as an engine uploads them
    s["meta"] = torch.cat([table.flatten(), torch.tensor(lens, dtype=torch.int32), ref]).to(DEV)
    s["meta0"] = s["meta"].clone()
    a, b = table.numel(), table.numel() + n
    s["table"], s["len"], s["ref"] = s["meta"][:a].view(table.shape), s["meta"][a:b], s["meta"][b:]
    s["seqs"] = torch.randperm(n, generator=cpu).int().to(DEV)
    s["keep"] = _i32([c["keep"] - i * c["keep"] // (4 * n) for i in range(n)])
    s["dropped"], s["status"] = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    # a few positions draw most of the weight, some none at all
    mass = torch.exp(2.0 * _rn(g, L, n, NKV, ld * page))
    s["mass0"] = mass.masked_fill_(torch.rand(mass.shape, generator=g, device=DEV) < 0.05, 0.0)
    s["mass"] = s["mass0"].clone()
    # page contents: any codes; scales and F16 values are finite
    s["vals"] = torch.empty((2, L, NKV, pages * page, VB[c["kv"]]), dtype=torch.uint8, device=DEV)
    s["scales"] = None
    if c["kv"] == "f16":
        flat = s["vals"].view(torch.float16).view(-1)
        part = torch.randint(-2048, 2048, (min(flat.numel(), (1 << 22) + 256),), generator=g, device=DEV).half()
        flat.copy_(part.repeat(flat.numel() // part.numel() + 1)[:flat.numel()])
    else:
        s["vals"].random_(0, 256, generator=g)
        s["scales"] = (0.01 * _rn(g, 2, L, NKV, pages * page, 8)).half()


def prepare(case, seed):
    s = {"case": case}
    (_prepare_evict if case["kind"] == "evict" else _prepare_chunks)(case, s, seed)
    return s


# ---- one pass, by the framework -------------------------------------------------------------------------------------
def _handle(s):
    """The objects that a user's program keeps: the layers, the pages, the workspaces."""
    if "pg" not in s:
        import qwengine_amd.ops as ops
        c = s["case"]
        s["kvt"] = ops.KV_TYPES[c["kv"]]
        v, d = s["vals"], s["scales"]
        if c["kind"] != "evict":
            v, d = v[:, None], None if d is None else d[:, None]
        bits = lambda t: None if t is None else t.view(torch.int16)
        s["layers"] = [ops.KVLayer(s["kvt"], v.shape[3], v[0, i], v[1, i], bits(d if d is None else d[0, i]),
                                   bits(d if d is None else d[1, i])) for i in range(v.shape[1])]
        s["pg"] = ops.KVPages(s["table"], s["len"], s["ref"], c["page"])
        size = 0
        if c["kind"] == "prefill":
            size = ops.attn_prefill_batch_work_bytes(s["n"], s["rows"], s["max_len"])
        elif c["kind"] == "weights":
            size = ops.attn_weights_batch_work_bytes(s["n"], s["rows"], s["max_len"])
        elif c["kind"] == "evict":
            size = ops.kv_pages_evict_work_bytes(s["pg"], c["n"], c["layers"], c["keep"])
        s["work"] = torch.empty(size, dtype=torch.uint8, device=DEV)
    return s["layers"], s["pg"], s["work"]


def _run_own(s):
    import qwengine_amd.ops as ops
    c = s["case"]
    layers, pg, work = _handle(s)
    if c["kind"] == "prefill":
        ops.attn_prefill_batch(s["q"], s["gate"], layers[0], s["kvt"], pg, None, s["off"], s["n"], s["rows"], s["max_len"],
                               s["out"], work, lse=s["lse"])
    elif c["kind"] == "prep":
        ops.attn_prep_rows_batch(s["qg"], s["k"], s["v"], s["qn"], s["kn"], pg, None, s["off"], s["n"], s["rows"], THETA, EPS,
                                 s["kvt"], layers[0], s["q"], s["gate"])
    elif c["kind"] == "weights":
        ops.attn_weights_batch(s["q"], s["lse"], layers[0], s["kvt"], pg, None, s["off"], s["n"], s["rows"], s["max_len"],
                               s["mass"], work)
    else:
        ops.kv_pages_evict(pg, s["seqs"], s["keep"], c["recent"], c["keep"], layers, s["kvt"], s["mass"], s["dropped"],
                           s["status"], work)


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


def _group_rows(s, group, which):
    """K (0) or V (1) rows of a group's sequences: [4][sequences][positions][256] in 32 bits."""
    b, _, most = group
    page, j = s["case"]["page"], torch.arange(most, device=DEV)
    slots = s["table"].long()[b][:, (j // page)].clamp_min(0) * page + j % page
    d = None if s["scales"] is None else s["scales"][which][:, slots]
    return _values(s["vals"][which][:, slots], d, s["case"]["kv"])


def _scores(s, group):
    """A group's scores [sequences][tokens][24][positions], -inf where a token does not see the position; which of its
    [sequences][tokens] there are; their rows."""
    b, tokens, most = group
    first, last, lens = s["off"][b].long(), s["off"][b + 1].long(), s["len"][b].long()
    t = torch.arange(tokens, device=DEV)
    at = (first[:, None] + t).clamp_max(s["rows"] - 1)
    real = first[:, None] + t < last[:, None]
    x = s["q"][at].view(len(b), tokens, NKV, GRP, HD).permute(2, 0, 1, 3, 4).reshape(NKV, len(b), tokens * GRP, HD)
    S = (x / 16.0) @ _group_rows(s, group, 0).transpose(2, 3)
    S = S.view(NKV, len(b), tokens, GRP, most).permute(1, 2, 0, 3, 4).reshape(len(b), tokens, NH, most)
    sees = (lens - (last - first))[:, None] + t + 1
    hidden = (torch.arange(most, device=DEV) >= sees[..., None]) | ~real[..., None]
    return S.masked_fill_(hidden[:, :, None], -math.inf), real, at


def _plain_prefill(s):
    for group in s["groups"]:
        b, tokens, most = group
        S, real, at = _scores(s, group)
        top = S.amax(-1, keepdim=True).clamp_min(-3e38)
        P = torch.exp(S.sub_(top))
        den = P.sum(-1, keepdim=True)
        if s["lse"] is not None:
            s["lse"][at[real]] = (top + torch.log(den))[..., 0][real]
        rows = P.view(len(b), tokens, NKV, GRP, most).permute(2, 0, 1, 3, 4).reshape(NKV, len(b), tokens * GRP, most)
        O = (rows @ _group_rows(s, group, 1)).view(NKV, len(b), tokens, GRP, HD)
        O = O.permute(1, 2, 0, 3, 4).reshape(len(b), tokens, NH, HD) / den.clamp_min(1e-30)
        s["out"][at[real]] = (O[real] / (1.0 + torch.exp(-s["gate"][at[real]]))).half()


def _plain_prep(s):
    T, c = s["tokens"], s["case"]
    i = torch.arange(32, device=DEV, dtype=torch.float64)
    ang = (s["pos"].double()[:, None] * THETA ** (-i / 32.0))[:, None]
    cos, sin = torch.cos(ang), torch.sin(ang)

    def prep(x, w):  # in 64 bits: the quantizer's borders
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
        lo, hi = x[..., :32], x[..., 32:64]
        return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin, x[..., 64:]], -1).float()

    s["q"][:T] = prep(s["qg"][:T, :, :HD], s["qn"])
    s["gate"][:T] = s["qg"][:T, :, HD:]
    x = torch.stack([prep(s["k"][:T], s["kn"]), s["v"][:T]]).transpose(1, 2)  # [2][4][tokens][256]
    q, d = _quantize(x.contiguous(), c["kv"])
    s["vals"][:, :, s["slots"]] = q
    if d is not None:
        s["scales"][:, :, s["slots"]] = d


def _plain_weights(s):
    for group in s["groups"]:
        b, tokens, most = group
        S, real, at = _scores(s, group)
        P = torch.exp(S.sub_(s["lse"][at][..., None]))
        add = P.view(len(b), tokens, NKV, GRP, most).sum((1, 3))
        lens, first = s["len"][b].long(), s["len"][b].long() - (s["off"][b + 1] - s["off"][b]).long()
        j = torch.arange(most, device=DEV)
        old = s["mass"][b, :, :most]
        # the chunk's own positions begin with it
        new = torch.where(j < first[:, None, None], old, torch.zeros_like(old)) + add
        s["mass"][b, :, :most] = torch.where(j < lens[:, None, None], new, old)


def _plain_evict(s):
    c, page = s["case"], s["case"]["page"]
    table, lens, ref, mass = s["table"], s["len"], s["ref"], s["mass"]
    seqs, keep = s["seqs"].long(), s["keep"].long()
    have = lens[seqs].long()
    cut = have > keep
    # per layer, request and head: the last `recent` positions, then those of the largest weight, the lower one of equals
    j = torch.arange(mass.shape[-1], device=DEV)
    near = torch.minimum(keep, torch.full_like(keep, c["recent"]))
    m, r = have[:, None, None], near[:, None, None]
    key = torch.where(j >= m - r, math.inf, mass[:, seqs])
    order = torch.where(j >= m, -1.0, key).sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros(order.shape, dtype=torch.bool, device=DEV)
    kept.scatter_(-1, order, (j < keep[:, None, None]).expand(order.shape))
    kept &= cut[:, None, None]
    place = kept.cumsum(-1) - 1
    l, i, h, src = kept.nonzero(as_tuple=True)
    dst = place[l, i, h, src]
    # pages of the kept part that others hold are left to them
    e = torch.arange(table.shape[1], device=DEV)
    old, rows = table[seqs].long(), table[seqs].long()
    stay = (e < ((keep + page - 1) // page)[:, None]) & cut[:, None]
    used = (e < ((have + page - 1) // page)[:, None]) & cut[:, None]
    copied = stay & (ref[old.clamp_min(0)] > 1)
    free = (ref == 0).nonzero()[:, 0]
    gone = old[used & (copied | ~stay)]
    rows[copied] = free[:copied.sum()]
    ref.index_add_(0, gone, torch.full_like(gone, -1, dtype=torch.int32))
    ref[rows[copied]] = 1
    rows[used & ~stay] = -1
    table[seqs] = rows.int()
    lens[seqs] = torch.where(cut, keep, have).int()
    s["dropped"].copy_(torch.where(cut, have - keep, 0))
    s["status"].zero_()
    frm = old[i, src // page] * page + src % page
    to = rows[i, dst // page] * page + dst % page
    for t in (s["vals"], s["scales"]):
        if t is not None:
            t[:, l, h, to] = t[:, l, h, frm]
    mass[l, seqs[i], h, dst] = mass[l, seqs[i], h, src]


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "evict":
        # the sequences as the requests left them, with their weights; what the positions hold is moved, whatever it is
        s["meta"].copy_(s["meta0"])
        s["mass"].copy_(s["mass0"])
    if own:
        _run_own(s)
    else:
        {"prefill": _plain_prefill, "prep": _plain_prep, "weights": _plain_weights, "evict": _plain_evict}[kind](s)
    if kind == "prefill":
        return {"out": s["out"], "lse": s["lse"]}
    if kind == "weights":
        return {"mass": s["mass"]}
    if kind == "prep":  # the appended rows as the values they stand for
        v, d = s["vals"][:, :, s["slots"]], s["scales"]
        if c["kv"] == "f16":
            v = v.view(torch.float16)
        elif c["kv"] == "q8_0":
            v = (v.view(torch.int8).unflatten(-1, (8, 32)) * d[:, :, s["slots"]][..., None]).flatten(-2)
        else:
            v = torch.stack([v & 15, v >> 4], -1).view(torch.int8).flatten(-2) - 8
            v = (v.unflatten(-1, (8, 32)) * d[:, :, s["slots"]][..., None]).flatten(-2)
        return {"q": s["q"], "gate": s["gate"], "rows": v}
    # page contents and weights are moved, never computed: their bits have to be equal
    vals = s["vals"].view(torch.float16) if c["kv"] == "f16" else s["vals"]
    return {"table": s["table"], "len": s["len"], "ref": s["ref"], "vals": vals, "scales": s["scales"], "mass": s["mass"],
            "dropped": s["dropped"], "status": s["status"]}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "evict":
        n = c["n"]
        lens = sum(c["len"] - (i * c["len"]) // (3 * n) for i in range(n))
        keep = sum(c["keep"] - i * c["keep"] // (4 * n) for i in range(n))
        # the survivors read and written, the weights read, theirs written
        return {"bytes": c["layers"] * (2.0 * keep * POS_BYTES[c["kv"]] + 4 * NKV * (lens + keep)), "flops": 0.0}
    tokens, pairs, _ = _cost(c)
    keys = sum(m for _, m in _shape(c))
    if c["kind"] == "prep":
        return {"bytes": tokens * (2 * 4 * QD * 2 + 2 * 4 * NKV * HD + POS_BYTES[c["kv"]]), "flops": tokens * QD * 8.0}
    if c["kind"] == "prefill":
        return {"bytes": keys * POS_BYTES[c["kv"]] + tokens * (QD * (4 + 4 + 2) + (4 * NH if c["lse"] else 0)),
                "flops": 4.0 * QD * pairs}
    return {"bytes": keys * (POS_BYTES[c["kv"]] // 2 + 2 * 4 * NKV) + tokens * (QD * 4 + 4 * NH), "flops": 2.0 * QD * pairs}


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------
def _row64(s, which, head, slots):
    """Cache rows in 64 bits, one KV head: [slots][256]."""
    kv = s["case"]["kv"]
    b = s["vals"][which, head][slots]
    if kv == "f16":
        return b.view(torch.float16).double()
    d = s["scales"][which, head][slots].double().repeat_interleave(32, -1)
    if kv == "q8_0":
        return b.view(torch.int8).double() * d
    out = torch.empty((b.shape[0], HD), dtype=torch.float64, device=DEV)
    out[:, 0::2], out[:, 1::2] = (b % 16).double() - 8, (b // 16).double() - 8
    return out * d


def _exact_chunks(c, s):
    page, lens, off = c["page"], s["len"].cpu().tolist(), s["off"].cpu().tolist()
    out = torch.zeros((s["rows"], NH, HD), dtype=torch.float64, device=DEV)
    lse = torch.zeros((s["rows"], NH), dtype=torch.float64, device=DEV)
    mass = s["mass"].double() if c["kind"] == "weights" else None
    for b, m in enumerate(lens):
        k = off[b + 1] - off[b]
        j = torch.arange(m, device=DEV)
        slots = s["table"][b].long()[j // page] * page + j % page
        if mass is not None:
            mass[b, :, m - k:m] = 0.0
        for h in range(NKV):
            K, V = _row64(s, 0, h, slots), _row64(s, 1, h, slots)
            heads = slice(h * GRP, (h + 1) * GRP)
            for t0 in range(0, k, 256):
                r = slice(off[b] + t0, off[b] + min(k, t0 + 256))
                n = r.stop - r.start
                sc = torch.tensordot(s["q"][r, heads].double(), K, ([2], [1])) / math.sqrt(HD)  # [n][6][m]
                late = j > (m - k + t0 + torch.arange(n, device=DEV))[:, None]
                sc.masked_fill_(late[:, None], -math.inf)
                if mass is not None:
                    mass[b, h, :m] += torch.exp(sc - s["lse"][r, heads].double()[..., None]).sum((0, 1))
                    continue
                out[r, heads] = torch.tensordot(torch.softmax(sc, -1), V, ([2], [0]))
                lse[r, heads] = torch.logsumexp(sc, -1)
    if mass is not None:
        return {"mass": mass}
    return {"out": out * torch.sigmoid(s["gate"].double()), "lse": lse if c["lse"] else None}


def _exact_prep(c, s):
    T = s["tokens"]
    i = torch.arange(32, device=DEV, dtype=torch.float64)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * THETA ** (-2.0 * i / 64.0))

    def prep(x, w):
        x = x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + EPS) * w.double()
        z = torch.complex(x[..., :32], x[..., 32:64]) * turn[:, None]
        return torch.cat([z.real, z.imag, x[..., 64:]], -1)

    rows = None
    if c["kv"] == "f16":
        rows = torch.stack([prep(s["k"][:T], s["kn"]), s["v"][:T].double()]).transpose(1, 2).contiguous()
    q, gate = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    q[:T], gate[:T] = prep(s["qg"][:T, :, :HD], s["qn"]), s["qg"][:T, :, HD:]
    return {"q": q, "gate": gate, "rows": rows}


def _exact_evict(c, s):
    # a literal account, request by request and head by head
    page, L = c["page"], c["layers"]
    table, lens, ref = s["table"].cpu().tolist(), s["len"].cpu().tolist(), s["ref"].cpu().tolist()
    free, before = [p for p, r in enumerate(ref) if r == 0], list(ref)
    mass, out = s["mass0"].cpu().numpy(), s["mass0"].clone()
    vals = s["vals"].view(torch.float16) if c["kv"] == "f16" else s["vals"]
    dropped, moves = [], []
    for q, keep in zip(s["seqs"].cpu().tolist(), s["keep"].cpu().tolist()):
        m, near = lens[q], min(c["recent"], keep)
        dropped.append(max(0, m - keep))
        if m <= keep:
            continue
        row = list(table[q])
        for e in range(_ceil(m, page)):
            if e >= _ceil(keep, page):
                ref[row[e]] -= 1
                table[q][e] = -1
            elif before[row[e]] > 1:
                ref[row[e]] -= 1
                table[q][e] = free.pop(0)
                ref[table[q][e]] = 1
        old, new = _i32(row).long(), _i32(table[q]).long()
        to = torch.arange(keep, device=DEV)
        to = new[to // page] * page + to % page
        lens[q] = keep
        for l in range(L):
            for h in range(NKV):
                w = mass[l, q, h, :m - near]
                best = sorted((-w).argsort(kind="stable")[:keep - near].tolist()) + list(range(m - near, m))
                at = torch.tensor(best, device=DEV)
                out[l, q, h, :keep] = s["mass0"][l, q, h, at]
                moves.append((l, h, old[at // page] * page + at % page, to))
    for t in (vals, s["scales"]):
        if t is not None:
            was = [t[:, l, h, frm] for l, h, frm, _ in moves]
            for (l, h, _, to), x in zip(moves, was):
                t[:, l, h, to] = x
    wide = lambda t: None if t is None else t.double() if t.is_floating_point() else t
    return {"table": _i32(table), "len": _i32(lens), "ref": _i32(ref), "vals": wide(vals), "scales": wide(s["scales"]),
            "mass": out.double(), "dropped": _i32(dropped), "status": torch.zeros(1, dtype=torch.int32, device=DEV)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"prefill": _exact_chunks, "weights": _exact_chunks, "prep": _exact_prep, "evict": _exact_evict}[case["kind"]](case, s)
