"""Timed cases of the operators around a paged key/value cache: attention of a chunk of new tokens over the cache
(`paged.paged_attention_chunk`), rotary positions (`rotary.rotary_tables`, `rotary.rotary_embedding`) and the pages
themselves (`paged.copy_pages`, `fork_sequences`, `extend_sequences`, `free_sequences`, `compact_pages`).

`run` computes each in plain torch, or, where `own` is set, through the package.  `exact` restates the definitions in
64 bits, sequence by sequence."""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
H = torch.float16


def _package():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ascend-ops_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from ascend910a_extras import paged, rotary

    return paged, rotary


# ------------------------------------------------------------------------------------------------ cases
def listed():
    chunk = dict(op="chunk", one=0.0, window=0, lse=False)
    pages = dict(layers=4, row=1024, block=128)
    return [
        # four sequences that verify up to five drafted tokens each: the smallest call of a serving loop
        dict(chunk, name="chunk verify", seqs=4, new_lo=2, new_hi=5, past_lo=200, past_hi=1000, heads=32, kv_heads=8,
             dim=128, block=128, mix=1),
        # a batch in which most sequences decode one token while others still read their prompts; a sliding window,
        # small pages, a head size that is no power of two, log-sum-exp for a later join
        dict(chunk, name="chunk mixed window", seqs=24, new_lo=33, new_hi=500, past_lo=0, past_hi=2500, heads=16,
             kv_heads=16, dim=80, block=16, mix=2, one=0.6, window=1024, lse=True),
        # the last few tokens of one very long document
        dict(chunk, name="chunk long past", seqs=1, new_lo=16, new_hi=16, past_lo=131063, past_hi=131063, heads=32,
             kv_heads=8, dim=128, block=128, mix=3),
        # one chunk of a long prompt
        dict(chunk, name="chunk prefill", seqs=1, new_lo=4096, new_hi=4096, past_lo=28672, past_hi=28672, heads=32,
             kv_heads=8, dim=128, block=128, mix=4),
        # one decode step of 64 sequences: interleaved pairs in half of the head, q and k inside a fused projection
        dict(op="rotary", name="rotary decode", tokens=64, heads=32, kv_heads=8, dim=128, part=64, interleaved=True,
             fused=True, table="float16", positions=8192, build=False),
        # a prompt batch after the context was stretched: new tables, then the whole head rotated
        dict(op="rotary", name="rotary rescaled prefill", tokens=16384, heads=32, kv_heads=8, dim=128, part=128,
             interleaved=False, fused=True, table="float32", positions=32768, build=True),
        # a few pages handed from one sequence to another
        dict(op="copy", name="copy few pages", layers=2, row=256, block=16, pool=64, pairs=5),
        # a shared prefix duplicated over all layers
        dict(pages, op="copy", name="copy many pages", pool=640, pairs=301),
        # one beam search step of a single request: children take over from parents, get room, the old beams go
        dict(op="beam", name="beam few", layers=2, row=256, block=16, seqs=4, children=4, len_lo=20, len_hi=200,
             pool=96, mix=5),
        # the same step for a full batch with long contexts
        dict(pages, op="beam", name="beam many", seqs=64, children=128, len_lo=100, len_hi=2000, pool=1024, mix=6),
        # a small pool packed before it shrinks
        dict(op="compact", name="compact small pool", layers=2, row=256, block=16, pool=100, seqs=9, len_lo=1,
             len_hi=120, mix=7),
        # a pool with a thousand pages left full of holes by finished sequences
        dict(pages, op="compact", name="compact large pool", pool=1024, seqs=60, len_lo=100, len_hi=2000, mix=8),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["chunk", "chunk", "chunk", "rotary", "copy", "beam", "compact"])
    mix = rng.randrange(1 << 20)
    if op == "chunk":
        while True:
            kv_heads = rng.choice([1, 2, 4, 8, 16])
            new_hi = _log_int(rng, 1, 2048)
            past_hi = _log_int(rng, 1, 65536)
            c = dict(op="chunk", seqs=_log_int(rng, 1, 64), new_lo=max(1, new_hi // rng.choice([1, 2, 8])), new_hi=new_hi,
                     past_lo=rng.choice([0, past_hi // 2, past_hi]), past_hi=past_hi,
                     heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8]), kv_heads=kv_heads,
                     dim=rng.choice([64, 80, 96, 112, 128, 128, 160, 192, 256]), block=rng.choice([16, 32, 64, 128]), mix=mix,
                     one=rng.choice([0.0, 0.0, 0.5]), window=rng.choice([0, 0, rng.randrange(1, 5000)]),
                     lse=rng.random() < 0.5)
            padded = c["seqs"] * (new_hi * c["heads"] * (past_hi + new_hi) * 4 + 2 * (past_hi + new_hi) * kv_heads * c["dim"] * 4)
            if padded < 10e9 and work(c)["flops"] < 1.5e12:
                return c
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        build = rng.random() < 0.3
        return dict(op="rotary", tokens=_log_int(rng, 1, 8192), heads=kv_heads * rng.choice([1, 3, 4, 8]),
                    kv_heads=kv_heads, dim=dim, part=rng.choice([dim, dim // 2, dim // 4, 20]),
                    interleaved=rng.random() < 0.5, fused=rng.random() < 0.5, table=rng.choice(["float16", "float32"]),
                    positions=_log_int(rng, 500, 32768), build=build)
    big = rng.random() < 0.5
    c = dict(op=op, layers=rng.randrange(1, 5), row=rng.choice([256, 512, 1024] if big else [64, 128, 256]),
             block=rng.choice([64, 128] if big else [16, 32]))
    hi = _log_int(rng, 2 * c["block"], 2000 if big else 300)
    per = hi // c["block"] + 1
    if op == "copy":
        pairs = _log_int(rng, 1, 200)
        return dict(c, pool=2 * pairs + rng.randrange(1, 60), pairs=pairs)
    seqs = _log_int(rng, 1, 40)
    if op == "beam":
        children = _log_int(rng, 1, 80)
        return dict(c, seqs=seqs, children=children, len_lo=1, len_hi=hi, mix=mix,
                    pool=seqs * per + rng.choice([2 * children, children // 2]) + rng.randrange(9))  # at times too few pages
    return dict(c, pool=int(seqs * per * rng.uniform(1.2, 2.0)) + 2, seqs=seqs, len_lo=1, len_hi=hi, mix=mix)


def _chunk_lens(c):
    """New tokens and context lengths of the sequences."""
    r = random.Random(c["mix"])
    new = [1 if r.random() < c["one"] else r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["seqs"])]
    return new, [n + r.randint(c["past_lo"], c["past_hi"]) for n in new]


def _lens(c):
    r = random.Random(c["mix"])
    return [r.randint(c["len_lo"], c["len_hi"]) for _ in range(c["seqs"])]


def _parents(c):
    r = random.Random(c["mix"] + 1)
    return [r.randrange(c["seqs"]) for _ in range(c["children"])]


# ------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _normal(shape, g):
    return torch.randn(shape, generator=g, device=DEV, dtype=H)


def _page_rows(lens, block, pool, g):
    """A block table in which every sequence owns pages of its own, taken at random from the pool."""
    need = [-(-n // block) for n in lens]
    order = torch.randperm(pool, generator=g, device=DEV).int()
    width = max(need) + 1
    at = torch.tensor([[min(sum(need[:b]) + j, pool - 1) for j in range(width)] for b in range(len(lens))], device=DEV)
    live = torch.tensor([[j < n for j in range(width)] for n in need], device=DEV)
    return torch.where(live, order[at], torch.full_like(order[at], -1)), order[: sum(need)]


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=c, op=c["op"])
    if c["op"] == "chunk":
        new, ctx = _chunk_lens(c)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        need = [-(-n // c["block"]) for n in ctx]
        pool = sum(need) + 3
        order = torch.randperm(pool, generator=g, device=DEV).int()
        width = max(need)
        first = [sum(need[:b]) for b in range(len(need))]
        at = torch.tensor(first, device=DEV)[:, None] + torch.arange(width, device=DEV)
        s["tables"] = order[at.clamp(max=pool - 1)].contiguous()
        shape = (pool, c["kv_heads"] * c["dim"] // 16, c["block"], 16)
        s["kc"], s["vc"] = _normal(shape, g), _normal(shape, g)
        s["q"] = _normal((starts[-1], c["heads"], c["dim"]), g)
        s["ctx"], s["starts"] = _int(ctx), _int(starts)
        s["max_new"], s["max_ctx"] = max(new), max(ctx)
    elif c["op"] == "rotary":
        qd, kd = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
        if c["fused"]:
            qkv = _normal((c["tokens"], qd + 2 * kd), g)
            q, k, _ = qkv.split([qd, kd, kd], dim=1)
        else:
            q, k = _normal((c["tokens"], qd), g), _normal((c["tokens"], kd), g)
        s["q"], s["k"] = q.unflatten(1, (c["heads"], c["dim"])), k.unflatten(1, (c["kv_heads"], c["dim"]))
        s["pos"] = torch.randint(0, c["positions"], (c["tokens"],), generator=g, device=DEV, dtype=torch.int32)
        s["dtype"] = getattr(torch, c["table"])
        if not c["build"]:
            s["cos"], s["sin"] = (t.to(s["dtype"]) for t in _plain_tables(c))
    else:
        shape = (c["pool"], c["row"] // 16, c["block"], 16)
        s["kcs"] = [_normal(shape, g) for _ in range(c["layers"])]
        s["vcs"] = [_normal(shape, g) for _ in range(c["layers"])]
        if c["op"] == "copy":
            order = torch.randperm(c["pool"], generator=g, device=DEV).int()
            s["src"], s["dst"] = order[: c["pairs"]].contiguous(), order[c["pairs"]: 2 * c["pairs"]].contiguous()
        else:
            lens = _lens(c)
            s["tables"], owned = _page_rows(lens, c["block"], c["pool"], g)
            s["lens"] = _int(lens)
            s["counts"] = torch.zeros(c["pool"], dtype=torch.int32, device=DEV)
            s["counts"][owned.long()] = 1
            if c["op"] == "beam":
                parents = _parents(c)
                s["parents"] = _int(parents)
                s["wanted"] = _int([lens[p] + 1 for p in parents])
                s["rows"] = _int(list(range(c["seqs"])))
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return _own(state) if own else _plain(state)


def _own(s):
    paged, rotary = _package()
    c = s["case"]
    if s["op"] == "chunk":
        return paged.paged_attention_chunk(s["q"], s["kc"], s["vc"], s["tables"], s["ctx"], s["starts"],
                                           window=c["window"], return_lse=c["lse"])
    if s["op"] == "rotary":
        if not c["build"]:
            return rotary.rotary_embedding(s["q"], s["k"], s["pos"], s["cos"], s["sin"], interleaved=c["interleaved"])
        cos, sin = rotary.rotary_tables(c["positions"], c["part"], 10000.0, scaling="yarn", factor=8.0,
                                        original_max_position=4096, dtype=s["dtype"])
        return (cos, sin, *rotary.rotary_embedding(s["q"], s["k"], s["pos"], cos, sin, interleaved=c["interleaved"]))
    if s["op"] == "copy":
        paged.copy_pages(s["kcs"], s["vcs"], s["src"], s["dst"])
        return s["kcs"], s["vcs"]
    if s["op"] == "beam":
        rows, lens, counts = paged.fork_sequences(s["tables"], s["lens"], s["parents"], s["counts"], s["kcs"], s["vcs"])
        room, granted, counts = paged.extend_sequences(rows, lens, s["wanted"], counts, c["block"])
        counts = paged.free_sequences(s["tables"], s["lens"], s["rows"], counts, c["block"])
        return rows, lens, room, granted, counts, s["kcs"], s["vcs"]
    tables, counts, used = paged.compact_pages(s["tables"], s["lens"], s["counts"], s["kcs"], s["vcs"])
    return tables, counts, used, s["kcs"], s["vcs"]


def _plain(s):
    if s["op"] == "chunk":
        return _plain_chunk(s)
    if s["op"] == "rotary":
        return _plain_rotary(s)
    if s["op"] == "copy":
        src, dst = s["src"].long(), s["dst"].long()
        _plain_move(s, src, dst)
        return s["kcs"], s["vcs"]
    return _plain_beam(s) if s["op"] == "beam" else _plain_compact(s)


def _plain_chunk(s):
    c = s["case"]
    T, Hq, D = s["q"].shape
    Hkv, B = c["kv_heads"], c["seqs"]
    starts, ctx = s["starts"].long(), s["ctx"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(s["max_new"], device=DEV)
    rows = (starts[:-1, None] + i).clamp(max=T - 1)                                   # [B, max_new]
    q = s["q"].float()[rows].unflatten(2, (Hkv, Hq // Hkv)).permute(0, 2, 3, 1, 4)    # [B, Hkv, G, max_new, D]
    pages = s["tables"].long()

    def whole(cache):  # [B, Hkv, max_ctx, D]
        x = cache[pages].unflatten(2, (Hkv, D // 16)).permute(0, 2, 1, 4, 3, 5)
        return x.reshape(B, Hkv, -1, D)[:, :, : s["max_ctx"]].float()

    score = torch.matmul(q.flatten(2, 3), whole(s["kc"]).transpose(2, 3)).unflatten(2, (Hq // Hkv, -1))
    score.mul_(1 / math.sqrt(D))
    at = ctx[:, None] - new[:, None] + i
    j = torch.arange(s["max_ctx"], device=DEV)
    seen = j <= at[:, :, None]
    if c["window"]:
        seen &= j > at[:, :, None] - c["window"]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score.sub_(top).exp_()
    total = score.sum(-1, keepdim=True)
    out = torch.matmul(score.flatten(2, 3), whole(s["vc"])).unflatten(2, (Hq // Hkv, -1)) / total
    b = (torch.arange(T, device=DEV)[:, None] >= starts[1:]).sum(1)
    back = torch.arange(T, device=DEV) - starts[b]
    o = out[b, :, :, back].reshape(T, Hq, D).to(H)
    if not c["lse"]:
        return o
    return o, (top + torch.log(total))[..., 0][b, :, :, back].reshape(T, Hq)


def _plain_tables(c):
    """cos and sin in 64 bits; the ramp of the stretched frequencies where the case builds them."""
    half = c["part"] // 2
    f = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) * 2 / c["part"])
    a = 1.0
    if c["build"]:
        low, high = (c["part"] * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(10000.0)) for t in (32, 1))
        low, high = max(math.floor(low), 0), min(math.ceil(high), c["part"] - 1)
        ramp = ((torch.arange(half, dtype=torch.float64, device=DEV) - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / 8 * ramp + f * (1 - ramp)
        a = 0.1 * math.log(8) + 1
    angle = torch.arange(c["positions"], dtype=torch.float64, device=DEV)[:, None] * f
    return torch.cos(angle) * a, torch.sin(angle) * a


def _plain_rotary(s):
    c = s["case"]
    tables = tuple(t.to(s["dtype"]) for t in _plain_tables(c)) if c["build"] else (s["cos"], s["sin"])
    cos, sin = (t[s["pos"].long()].float()[:, None] for t in tables)

    def turn(x):
        y = x.float()
        part = y[..., : c["part"]]
        if c["interleaved"]:
            x1, x2 = part[..., 0::2], part[..., 1::2]
            both = torch.stack([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).flatten(-2)
        else:
            x1, x2 = part.chunk(2, -1)
            both = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
        return torch.cat([both, y[..., c["part"]:]], -1).to(H)

    out = turn(s["q"]), turn(s["k"])
    return (*tables, *out) if c["build"] else out


def _plain_move(s, src, dst):
    [cache.index_copy_(0, dst, cache[src]) for cache in s["kcs"] + s["vcs"]]


def _plain_free_pages(counts):
    """Page numbers, the free ones first, each kind ascending; and how many are free."""
    used = counts > 0
    return torch.argsort(used.int(), stable=True), (~used).sum()


def _plain_beam(s):
    c = s["case"]
    block, pool = c["block"], c["pool"]
    lens = s["lens"].long()
    width = s["tables"].size(1)
    j = torch.arange(width, device=DEV)
    # children
    parents = s["parents"].long()
    length = lens[parents]
    full, part = length // block, length % block
    order, free = _plain_free_pages(s["counts"])
    rank = torch.cumsum((part > 0).int(), 0) - 1
    ok = (part == 0) | (rank < free)
    fresh = order[rank.clamp(0, pool - 1)]
    old = s["tables"][parents].long()
    rows = torch.where(j < full[:, None], old, torch.full_like(old, -1))
    rows = torch.where((j == full[:, None]) & (part > 0)[:, None], fresh[:, None], rows)
    rows = torch.where(ok[:, None], rows, torch.full_like(rows, -1))
    child_lens = torch.where(ok, length, torch.zeros_like(length))
    counts = s["counts"].long().clamp(min=0)
    counts = counts.index_add(0, rows.flatten().clamp(min=0), (rows >= 0).flatten().long())
    takes = ok & (part > 0)
    last = torch.gather(old, 1, full.clamp(max=width - 1)[:, None])[:, 0]
    src, dst, live = last[takes], fresh[takes], (torch.arange(block, device=DEV) < part[takes][:, None])[:, None, :, None]
    [cache.index_copy_(0, dst, torch.where(live, cache[src], cache[dst])) for cache in s["kcs"] + s["vcs"]]
    # room for the next token
    wanted = s["wanted"].long()
    need = ((wanted + block - 1) // block - (child_lens + block - 1) // block).clamp(min=0)
    need = torch.where(wanted <= width * block, need, torch.zeros_like(need))
    order, free = _plain_free_pages(counts)
    before = torch.cumsum(need, 0) - need
    fits = (wanted > child_lens) & (wanted <= width * block) & ((need == 0) | (before + need <= free))
    have = (child_lens + block - 1) // block
    nth = j - have[:, None]
    grown = fits[:, None] & (nth >= 0) & (nth < need[:, None])
    room = torch.where(grown, order[(before[:, None] + nth).clamp(0, pool - 1)], rows)
    granted = torch.where(fits, wanted, child_lens)
    counts = counts.index_add(0, room.flatten().clamp(min=0), grown.flatten().long())
    # the old beams
    gone = s["tables"][s["rows"].long()].long()
    live = j < ((lens[s["rows"].long()] + block - 1) // block)[:, None]
    counts = counts.index_add(0, gone.flatten().clamp(min=0), -live.flatten().long()).clamp(min=0)
    return rows.int(), child_lens.int(), room.int(), granted.int(), counts.int(), s["kcs"], s["vcs"]


def _plain_compact(s):
    c = s["case"]
    used = s["counts"] > 0
    total = used.sum()
    page = torch.arange(c["pool"], device=DEV)
    src, dst = torch.nonzero(used & (page >= total))[:, 0], torch.nonzero(~used & (page < total))[:, 0]
    to = page.index_copy(0, src, dst)
    _plain_move(s, src, dst)
    counts = torch.zeros_like(s["counts"]).index_add(0, to, s["counts"].clamp(min=0))
    live = torch.arange(s["tables"].size(1), device=DEV) < ((s["lens"] + c["block"] - 1) // c["block"])[:, None]
    tables = torch.where(live, to[s["tables"].long().clamp(min=0)].int(), s["tables"])
    return tables, counts, total.int().reshape(1), s["kcs"], s["vcs"]


# ------------------------------------------------------------------------------------------------ floors
def work(case):
    c = case
    if c["op"] == "chunk":
        new, ctx = _chunk_lens(c)
        pairs = touched = 0
        for n, total in zip(new, ctx):
            w = c["window"] or total
            first = total - n  # position of the first new token; token i sees min(first + i + 1, w) keys
            bend = min(max(w - first, 0), n)
            pairs += bend * first + bend * (bend + 1) // 2 + (n - bend) * w
            touched += total - max(0, first - w + 1)
        rows = sum(new) * c["heads"]
        return {"bytes": 2 * c["dim"] * (2 * rows + 2 * touched * c["kv_heads"]) + (4 * rows if c["lse"] else 0),
                "flops": 4 * c["dim"] * c["heads"] * pairs}
    if c["op"] == "rotary":
        heads = c["heads"] + c["kv_heads"]
        entry = 2 if c["table"] == "float16" else 4
        table = c["positions"] if c["build"] else min(c["tokens"], c["positions"])
        return {"bytes": 4 * c["tokens"] * heads * c["dim"] + c["part"] * entry * table + 4 * c["tokens"],
                "flops": 3 * c["tokens"] * heads * c["part"]}
    token = 2 * c["row"] * 2 * c["layers"]  # bytes of one token in all caches
    if c["op"] == "copy":
        return {"bytes": 2 * c["pairs"] * c["block"] * token + 8 * c["pairs"], "flops": 0}
    lens = _lens(c)
    width = max(-(-n // c["block"]) for n in lens) + 1
    if c["op"] == "beam":
        copied = sum(lens[p] % c["block"] for p in _parents(c))
        ints = c["seqs"] * (width + 2) + c["children"] * (2 * width + 4) + 2 * c["pool"]
        return {"bytes": 2 * copied * token + 4 * ints, "flops": 0}
    # pages that move: on average the used share of those behind the first `used`
    used = sum(-(-n // c["block"]) for n in lens)
    moved = used * (c["pool"] - used) / c["pool"]
    return {"bytes": 2 * moved * c["block"] * token + 4 * (2 * c["seqs"] * width + c["seqs"] + 2 * c["pool"]), "flops": 0}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "chunk":
        return _exact_chunk(c, s)
    if c["op"] == "rotary":
        return _exact_rotary(c, s)
    caches = s["kcs"] + s["vcs"]
    if c["op"] == "copy":
        pairs = list(zip(s["src"].tolist(), s["dst"].tolist()))
        after = [_moved(x, pairs, c["block"]) for x in caches]
        return after[: c["layers"]], after[c["layers"]:]
    if c["op"] == "beam":
        return _exact_beam(c, s, caches)
    counts, tables, lens = s["counts"].tolist(), s["tables"].tolist(), s["lens"].tolist()
    used = sum(n > 0 for n in counts)
    holes = [p for p in range(used) if counts[p] <= 0]
    pairs = list(zip([p for p in range(used, c["pool"]) if counts[p] > 0], holes))
    to = dict(pairs)
    for src, dst in pairs:
        counts[dst], counts[src] = counts[src], 0
    for row, n in zip(tables, lens):
        for j in range(-(-n // c["block"])):
            row[j] = to.get(row[j], row[j])
    after = [_moved(x, pairs, c["block"]) for x in caches]
    return _int(tables), _int(counts), _int([used]), after[: c["layers"]], after[c["layers"]:]


def _moved(cache, pairs, tokens):
    """The cache after its pages (src, dst[, tokens]) were copied one after the other."""
    x = cache.clone()
    for src, dst, *n in pairs:
        n = n[0] if n else tokens
        x[dst, :, :n] = cache[src, :, :n]
    return x


def _exact_beam(c, s, caches):
    block = c["block"]
    counts, tables, lens = s["counts"].tolist(), s["tables"].tolist(), s["lens"].tolist()
    width = len(tables[0])
    free = [p for p in range(c["pool"]) if counts[p] <= 0]
    rows, out_lens, pairs = [], [], []
    for p in s["parents"].tolist():
        full, part = divmod(lens[p], block)
        row = tables[p][:full]
        if part:
            if not free:
                rows.append([-1] * width)
                out_lens.append(0)
                continue
            pairs.append((tables[p][full], free[0], part))
            row = row + [free.pop(0)]
        for page in row:
            counts[page] += 1
        rows.append(row + [-1] * (width - len(row)))
        out_lens.append(lens[p])
    room, granted, short = [list(r) for r in rows], list(out_lens), False
    free = [p for p in range(c["pool"]) if counts[p] <= 0]
    for i, want in enumerate(s["wanted"].tolist()):
        if want <= out_lens[i] or want > width * block:
            continue
        have = -(-out_lens[i] // block)
        need = -(-want // block) - have
        short = short or need > len(free)
        if need and short:  # rows are served in order: nothing for those behind the first that does not fit
            continue
        for k in range(need):
            room[i][have + k] = free.pop(0)
            counts[room[i][have + k]] += 1
        granted[i] = want
    for r in s["rows"].tolist():
        for j in range(-(-lens[r] // block)):
            counts[tables[r][j]] = max(0, counts[tables[r][j]] - 1)
    after = [_moved(x, pairs, block) for x in caches]
    return _int(rows), _int(out_lens), _int(room), _int(granted), _int(counts), after[: c["layers"]], after[c["layers"]:]


def _exact_rotary(c, s):
    R = c["part"]
    freqs = []
    for j in range(R // 2):
        f = math.exp(-2.0 * j / R * math.log(10000.0))
        if c["build"]:
            def where(turns):  # the pair whose wave turns so often within the original context
                return R * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))

            lo, hi = max(math.floor(where(32.0)), 0), min(math.ceil(where(1.0)), R - 1)
            mixed = min(max((j - lo) / (hi - lo if hi > lo else 0.001), 0.0), 1.0)
            f = f * (1 - mixed) + f / 8 * mixed
        freqs.append(f)
    scale = 1 + 0.1 * math.log(8) if c["build"] else 1.0
    turn = torch.polar(torch.tensor(scale, dtype=torch.float64, device=DEV),
                       torch.outer(torch.arange(c["positions"], device=DEV).double(), torch.tensor(freqs, device=DEV, dtype=torch.float64)))
    # the embedding is defined on the table's rounded entries
    rounded = torch.complex(turn.real.to(s["dtype"]).double(), turn.imag.to(s["dtype"]).double())
    by = rounded[s["pos"].long()][:, None]

    def rotate(x):
        y = x.double().clone()
        first, second = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    out = rotate(s["q"]), rotate(s["k"])
    return (turn.real.contiguous(), turn.imag.contiguous(), *out) if c["build"] else out


def _exact_chunk(c, s):
    new, ctx = _chunk_lens(c)
    D, group = c["dim"], c["heads"] // c["kv_heads"]
    o = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)
    begin = 0
    for b, (n, total) in enumerate(zip(new, ctx)):
        j = torch.arange(total, device=DEV)
        page, slot = s["tables"][b].long()[j // c["block"]], j % c["block"]
        k = s["kc"][page, :, slot].reshape(total, c["kv_heads"], D)
        v = s["vc"][page, :, slot].reshape(total, c["kv_heads"], D)
        where = torch.arange(total - n, total, device=DEV)[:, None]
        hidden = j > where
        if c["window"]:
            hidden |= where - j >= c["window"]
        for h in range(c["heads"]):
            x = s["q"][begin: begin + n, h].double() @ k[:, h // group].double().T * D ** -0.5
            x[hidden] = -math.inf
            lse[begin: begin + n, h] = torch.logsumexp(x, 1)
            o[begin: begin + n, h] = torch.softmax(x, 1) @ v[:, h // group].double()
        begin += n
    return (o, lse) if c["lse"] else o
