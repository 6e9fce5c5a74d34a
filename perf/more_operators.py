"""The operators of a paged key/value cache and of beam search as they are timed and compared: the plain forms
below in elementary torch operations, and the calls that a program makes of the library.

A cache's pools are [layers, pages, kv_heads, page, head_dim]. Position j of a sequence is row j % page of the page
that entry j / page of its table row names; a page may stand in several rows (refs counts them), and a table
entry of -1 names none. The rows of a step are packed: sequence s has rows starts[s] .. starts[s + 1] - 1, at cache
positions lens[s], lens[s] + 1, ...: one token, a run of them, or the nodes of a tree of drafted tokens, whose masks
say which of the sequence's rows each may see (bit i: row i).
"""
import math

import torch

own = False
DEV = torch.device("cuda", 0)
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # the next token of one conversation over an f32 cache: latency
        {"name": "attend_token", "kind": "attend", "slots": 1, "rows": 1, "len": 1500, "ragged": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "x": "f32", "cache": "f32", "tree": 0},
        # one token of each of many conversations of all lengths, a 16-bit model
        {"name": "attend_batch", "kind": "attend", "slots": 24, "rows": 1, "len": 8000, "ragged": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "x": "bf16", "cache": "bf16", "tree": 0},
        # small drafted trees of a few conversations: f32 activations over a half-size cache
        {"name": "attend_trees", "kind": "attend", "slots": 8, "rows": 26, "len": 4000, "ragged": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "x": "f32", "cache": "bf16", "tree": 1},
        # wide trees deep in long conversations
        {"name": "attend_trees_30000", "kind": "attend", "slots": 4, "rows": 64, "len": 30000, "ragged": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "x": "f16", "cache": "f16", "tree": 1},
        # the rows of one token rotated and appended, f32
        {"name": "append_token", "kind": "append", "slots": 1, "rows": 1, "len": 1500, "ragged": 0, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "x": "f32", "cache": "f32", "tree": 0},
        # trees of many conversations, positions by depth, into a 16-bit cache
        {"name": "append_trees", "kind": "append", "slots": 64, "rows": 64, "len": 4000, "ragged": 1, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "x": "f32", "cache": "bf16", "tree": 1},
        # four beams of one short text, reordered: a page each copied in every layer
        {"name": "fork_beams", "kind": "fork", "slots": 4, "sources": 2, "len": 300, "reserve": 1, "layers": 32,
         "kv_heads": 8, "dim": 128, "page": 16, "max_pages": 64, "cache": "bf16"},
        # many answers sampled from each of a few long prompts
        {"name": "fork_samples", "kind": "fork", "slots": 128, "sources": 4, "len": 6000, "reserve": 64, "layers": 8,
         "kv_heads": 8, "dim": 128, "page": 64, "max_pages": 256, "cache": "bf16"},
        # the accepted path of each drafted tree moved up behind its text, in every layer
        {"name": "accept_trees", "kind": "accept", "slots": 16, "rows": 64, "depth": 8, "len": 2000, "layers": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "cache": "bf16"},
        # a pool half of whose pages were freed, packed before it is cut
        {"name": "compact_pool", "kind": "compact", "slots": 32, "used": 1024, "pages": 2048, "layers": 8, "kv_heads": 8,
         "dim": 128, "page": 16, "cache": "f16"},
        # the next tokens of four beams over the vocabulary, their texts reordered
        {"name": "beam_4", "kind": "beam", "batch": 1, "beams": 4, "count": 4, "vocab": 128256, "x": "f32", "live": 4,
         "done": 0, "text": 512},
        # a batch of searches, twice as many candidates as beams, some beams done
        {"name": "beam_16x8", "kind": "beam", "batch": 16, "beams": 8, "count": 16, "vocab": 128256, "x": "bf16",
         "live": 8, "done": 1, "text": 2048},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = ((32, 8, 128), (16, 16, 128), (32, 4, 128), (8, 2, 64), (12, 4, 64), (8, 1, 64), (16, 2, 256))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "append", "fork", "accept", "compact", "beam", "beam"))
    heads, kv_heads, dim = rng.choice(HEADS)
    page = rng.choice((16, 32, 64, 128))
    cache = rng.choice(("f32", "bf16", "f16"))
    c = {"kind": kind}
    token = 2 * kv_heads * dim * SIZE[cache]  # a position's key and value rows in a layer
    if kind in ("attend", "append"):
        slots = _log(rng, 1, 32)
        rows = rng.choice((1, rng.randint(2, 24), _log(rng, 24, 64)))
        # (no more bytes, and no more products, than in the largest listed case)
        most = min(30000, 480000000 // (slots * token), 4 * 64 * 30000 * 32 * 128 // (slots * rows * heads * dim))
        return {**c, "slots": slots, "rows": rows, "len": _log(rng, 1, most), "ragged": rng.choice((0, 1)),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
                "x": rng.choice(("f32", cache, rng.choice(("bf16", "f16")))), "cache": cache,
                "tree": int(rows > 1 and rng.random() < 0.75)}
    if kind == "fork":
        slots = _log(rng, 2, 96)
        sources = rng.randint(1, max(1, slots // 2))
        length = _log(rng, 1, min(4000, 40000 // sources))
        reserve = rng.choice((0, 1, rng.randint(2, 64)))
        held = sources * length + slots * (3 * page + reserve)
        return {**c, "slots": slots, "sources": sources, "len": length, "reserve": reserve,
                "layers": rng.randint(1, max(1, min(16, 1000000000 // (held * token)))), "kv_heads": kv_heads,
                "dim": dim, "page": page, "max_pages": (length + 64) // page + rng.randint(2, 40), "cache": cache}
    if kind == "accept":
        rows = rng.randint(2, 64)
        slots, length = _log(rng, 1, 24), _log(rng, 1, 2000)
        return {**c, "slots": slots, "rows": rows, "depth": rng.randint(1, min(10, rows)), "len": length,
                "layers": rng.randint(1, max(1, min(32, 1000000000 // (slots * (length + rows) * token)))),
                "kv_heads": kv_heads, "dim": dim, "page": page, "cache": cache}
    if kind == "compact":
        page = min(page, 32)
        pages = _log(rng, 64, min(2048, 500000000 // (page * token)))
        return {**c, "slots": _log(rng, 1, 32), "used": rng.randint(1, pages), "pages": pages,
                "layers": rng.randint(1, max(1, min(8, 500000000 // (pages * page * token)))), "kv_heads": kv_heads,
                "dim": dim, "page": page, "cache": cache}
    beams = rng.randint(1, 16)
    return {**c, "batch": _log(rng, 1, 64 // beams), "beams": beams, "count": beams * rng.choice((1, 2)),
            "vocab": _log(rng, 500, 128256), "x": rng.choice(("f32", "bf16", "f16")),
            "live": rng.choice((1, beams)), "done": rng.choice((0, 1)), "text": _log(rng, 16, 2048)}


def _spread(most, n, ragged, ratio):
    """n sizes from 1 to most, the first the largest (all of them, where not ragged)."""
    return [most if not ragged or i == 0 else 1 + int((most - 1) * ((i * ratio) % 1.0)) for i in range(n)]


def _lens(c):
    return _spread(c["len"], c["slots"], c.get("ragged", 1), 0.6180339887)


def _rows(c):
    return _spread(c["rows"], c["slots"], c.get("ragged", 1), 0.4142135624)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _gen(seed, tag):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1009 + tag)
    return g


def _randn(seed, tag, shape, dtype=torch.float32, std=1.0):
    x = torch.empty(shape, device=DEV, dtype=dtype)
    x.normal_(0.0, std, generator=_gen(seed, tag))
    return x


def _perm(seed, tag, n):
    return torch.randperm(n, generator=_gen(seed, tag), device=DEV)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _tables(seed, lens, page, max_pages, pages):
    """Table rows of sequences of those lengths, their pages anywhere in the pool, and the pages' counts."""
    need = -(-torch.tensor(lens) // page)
    at = torch.cumsum(need, 0) - need
    j = torch.arange(max_pages)
    have = (j < need[:, None]).to(DEV)
    ids = _perm(seed, 11, pages)[(at[:, None] + j).clamp_max(pages - 1).to(DEV)]
    table = torch.where(have, ids, -1).int()
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[ids[have]] = 1
    return table, refs


def _pools(seed, c, layers, pages):
    shape = (layers, pages, c["kv_heads"], c["page"], c["dim"])
    return _randn(seed, 12, shape, DT[c["cache"]]), _randn(seed, 13, shape, DT[c["cache"]])


def _tree(seed, rows):
    """Parents (-1: the text) of each sequence's nodes, nodes after their parents, level by level."""
    g = torch.Generator().manual_seed(seed * 31 + 7)
    out = []
    for n in rows:
        u = torch.rand(n, generator=g).tolist()
        out.append([-1 if j < 3 else max(int(j * 0.25 + u[j] * j * 0.35) - 1, -1) for j in range(n)])
    return out


def _marks(parents):
    """(masks, depths) of the packed rows: a node sees itself and the nodes above it."""
    masks, depths = [], []
    for seq in parents:
        m, d = [], []
        for j, p in enumerate(seq):
            m.append((m[p] if p >= 0 else 0) | 1 << j)
            d.append(d[p] + 1 if p >= 0 else 0)
        masks += [v - (1 << 64) if v >> 63 else v for v in m]
        depths += d
    return torch.tensor(masks, dtype=torch.int64, device=DEV).unsqueeze(1), _ints(depths)


def _rotation(positions, dim):
    """cos / sin tables [positions, dim] (cat(freqs, freqs)), base 500000."""
    inv = 500000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    f = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv
    f = torch.cat([f, f], 1)
    return f.cos().float(), f.sin().float()


def _inputs(c, seed):
    s = {"case": c}
    kind = c["kind"]
    if kind == "beam":
        rows = c["batch"] * c["beams"]
        s["logits"] = _randn(seed, 1, (rows, c["vocab"]), std=2.5).to(DT[c["x"]])
        s["scores"] = -_randn(seed, 2, (rows,), std=3.0).abs() - 4.0
        beam = torch.arange(rows, device=DEV) % c["beams"]
        s["scores"][beam >= c["live"]] = -math.inf  # a first step: one beam of each search has begun
        s["finished"] = ((beam == 1) & (c["done"] == 1)).int()
        s["text"] = torch.randint(0, c["vocab"], (rows, c["text"]), generator=_gen(seed, 3), device=DEV,
                                  dtype=torch.int32)
        s["next"] = torch.zeros(c["batch"] * c["count"], c["text"], dtype=torch.int32, device=DEV)
        return s
    page = c["page"]
    if kind in ("attend", "append"):
        lens, rows = _lens(c), _rows(c)
        total = [a + b for a, b in zip(lens, rows)]
        s["max_rows"], s["max_len"] = max(rows), max(total)
        max_pages = -(-s["max_len"] // page)
        pages = sum(-(-t // page) for t in total) + 8
        s["table"], s["refs"] = _tables(seed, total, page, max_pages, pages)
        s["lens"] = _ints(lens)
        s["starts"] = _ints([sum(rows[:i]) for i in range(len(rows) + 1)])
        s["k"], s["v"] = _pools(seed, c, 1, pages)
        s["q"] = _randn(seed, 4, (sum(rows), c["heads"], c["dim"])).to(DT[c["x"]])
        s["masks"], s["depths"] = _marks(_tree(seed, rows)) if c["tree"] else (None, None)
        if kind == "append":
            s["new_k"], s["new_v"] = (_randn(seed, t, (sum(rows), c["kv_heads"], c["dim"])).to(DT[c["x"]])
                                      for t in (5, 6))
            s["cos"], s["sin"] = _rotation(s["max_len"], c["dim"])
        return s
    if kind == "fork":
        # a few texts of different lengths in the first slots, the other slots held by texts that end here
        n, src = c["slots"], c["sources"]
        lens = [c["len"] - (7 * i) % min(c["len"], 50) if i < src else min(c["len"], page) for i in range(n)]
        extra = n * (2 + -(-c["reserve"] // page))
        pages = sum(-(-v // page) for v in lens) + extra
        s["table"], s["refs"] = _tables(seed, lens, page, c["max_pages"], pages)
        s["lens"] = _ints(lens)
        s["parents"] = (_perm(seed, 5, n) % src).int()
        s["parents"][:src] = torch.arange(src, dtype=torch.int32, device=DEV)
        s["k"], s["v"] = _pools(seed, c, c["layers"], pages)
    elif kind == "accept":
        n = c["slots"]
        lens = _lens(c)
        total = [v + c["rows"] for v in lens]
        max_pages = -(-max(total) // page)
        pages = sum(-(-t // page) for t in total) + 8
        s["table"], s["refs"] = _tables(seed, total, page, max_pages, pages)
        s["lens"] = _ints(lens)
        s["kept"] = torch.zeros(n, dtype=torch.int32, device=DEV)
        # increasing paths; a node is where it stays, or behind all places that the path's nodes move to
        late = torch.rand((n, c["rows"]), generator=_gen(seed, 5), device=DEV)
        late[:, :c["depth"]] = 2.0
        late[:, 0] = -1.0
        pick = torch.sort(late, dim=1, stable=True).indices[:, :c["depth"]]
        s["path"] = torch.sort(pick, dim=1).values.int().contiguous()
        s["counts"] = (torch.arange(n, device=DEV) * 5 % c["depth"] + 1).int()
        s["counts"][0] = c["depth"]
        s["k"], s["v"] = _pools(seed, c, c["layers"], pages)
    else:  # compact
        n = c["slots"]
        each = max(1, c["used"] // n)
        lens = [each * page - (i * 3) % page for i in range(min(n, c["used"]))]
        lens += [0] * (n - len(lens))
        s["table"], s["refs"] = _tables(seed, lens, page, each + 2, c["pages"])
        s["lens"] = _ints(lens)
        s["k"], s["v"] = _pools(seed, c, c["layers"], c["pages"])
    # the step's new lists: the old ones stay as they are
    s["new"] = tuple(torch.zeros_like(s[x]) for x in ("table", "lens", "refs"))
    s["short"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] != "beam":  # the handle that such a program keeps
        from inference_amd import PagedKVCache
        s["cache"] = PagedKVCache(s["k"], s["v"], s["table"], s["lens"], s["refs"])
    return s


# ---------------------------------------------------------------------------
# the passes
# ---------------------------------------------------------------------------

def _padded(s):
    """(sequence, number in it) of every packed row, and the largest number of rows."""
    n = s["starts"].diff().long()
    r = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(s["starts"][1:].contiguous(), r.int(), right=True)
    return seq, r - s["starts"].long()[seq], n


def _whole(pool, table):
    """[sequences, kv_heads, positions, dim] of a layer's pages in 32 bits, as the table's rows name them."""
    p = pool[table.clamp_min(0).long()].float()
    return p.permute(0, 2, 1, 3, 4).flatten(2, 3).contiguous()


def _attend(s):
    c = s["case"]
    q, table, lens = s["q"].float(), s["table"], s["lens"].long()
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    seq, num, n = _padded(s)
    most = s["max_rows"]
    k, v = _whole(s["k"][0], table), _whole(s["v"][0], table)
    pos = torch.arange(k.shape[2], device=DEV)
    rel = pos - lens[:, None]  # number among the step's rows, of the positions from lens on
    rows = torch.zeros((c["slots"], most, heads, dim), device=DEV)
    rows[seq, num] = q
    rows = rows.view(c["slots"], most, kv, heads // kv, dim).permute(0, 2, 1, 3, 4).reshape(c["slots"], kv, -1, dim)
    seen = (rel < 0)[:, None, :].expand(-1, most, -1).clone()
    inside = ((rel >= 0) & (rel < n[:, None]))[:, None, :]
    if s["masks"] is None:
        seen |= inside & (rel[:, None, :] <= torch.arange(most, device=DEV)[:, None])
    else:
        bits = torch.zeros((c["slots"], most), dtype=torch.int64, device=DEV)
        bits[seq, num] = s["masks"][:, 0]
        seen |= inside & ((bits[:, :, None] >> rel[:, None, :].clamp(0, 63)) & 1).bool()
    g = heads // kv
    sc = rows @ k.transpose(2, 3).contiguous() * dim ** -0.5
    sc = sc.view(c["slots"], kv, most, g, -1).masked_fill(~seen[:, None, :, None, :], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m == -math.inf, 0.0, m))
    z = p.sum(-1, keepdim=True)
    o = p.view(c["slots"], kv, most * g, -1) @ v
    o = o.view(c["slots"], kv, most, g, dim) / torch.where(z == 0, 1.0, z)
    return o.permute(0, 2, 1, 3, 4).reshape(c["slots"], most, heads, dim)[seq, num].to(s["q"].dtype)


def _turn(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _append(s):
    c = s["case"]
    seq, num, _ = _padded(s)
    base = s["lens"].long()[seq]
    at = base + (num if s["depths"] is None else s["depths"].long())
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    where = base + num
    page = s["table"][seq, where // c["page"]].long()
    row = where % c["page"]
    s["k"][0, page, :, row] = _turn(s["new_k"].float(), cos, sin).to(s["k"].dtype)
    s["v"][0, page, :, row] = s["new_v"].float().to(s["v"].dtype)
    return _turn(s["q"].float(), cos, sin).to(s["q"].dtype), s["k"], s["v"]


def _held(table, lens, page):
    return torch.arange(table.shape[1], device=DEV) < (-(-lens // page))[:, None]


def _fork(s):
    c = s["case"]
    page, table, reserve = c["page"], s["table"].long(), c["reserve"]
    pages, wide = s["refs"].shape[0], table.shape[1]
    par = s["parents"].long()
    lens = s["lens"].long()[par]
    new = torch.where(_held(table, lens, page), table[par], -1)
    one = torch.ones((), dtype=torch.int64, device=DEV)
    refs = s["refs"].long().clone()
    refs.scatter_add_(0, table.clamp_min(0).flatten(), -(table >= 0).long().flatten())
    refs.scatter_add_(0, new.clamp_min(0).flatten(), (new >= 0).long().flatten())
    # the part-filled pages that will be written: the first of those who would write one alone keeps it, a page that
    # others hold for good is kept by none
    slot = torch.arange(c["slots"], device=DEV)
    last = (lens - 1).clamp_min(0) // page
    part = (lens % page != 0) & (reserve > 0)
    w = torch.where(part, new[slot, last], pages)
    writers = torch.zeros(pages + 1, dtype=torch.int64, device=DEV).scatter_add_(0, w, one.expand_as(w))
    first = torch.full((pages + 1,), c["slots"], device=DEV).scatter_reduce_(0, w, slot, "amin")
    alone = torch.cat([refs, refs[:1]])[w] == writers[w]
    copy = part & ~(alone & (first[w] == slot))
    held = -(-lens // page)
    need = -(-(lens + reserve) // page) - held if reserve else torch.zeros_like(held)
    free = torch.nonzero(refs == 0).flatten()
    take = copy.long() + need
    at = torch.cumsum(take, 0) - take
    refs.scatter_add_(0, w.clamp_max(pages - 1), -copy.long())
    refs[free[:int(take.sum())]] = 1
    dst = free[at.clamp_max(free.shape[0] - 1)]
    j = torch.arange(wide, device=DEV)
    more = (j >= held[:, None]) & (j < (held + need)[:, None])
    new = torch.where(more, free[(at + copy)[:, None].add(j - held[:, None]).clamp(0, free.shape[0] - 1)], new)
    new[slot, last] = torch.where(copy, dst, new[slot, last])
    # the pages' rows that are in use
    i = torch.nonzero(copy).flatten()
    rows = torch.arange(page, device=DEV)
    use = (rows < (lens[i] % page)[:, None])[:, None, :, None]
    src, to = table[par[i], last[i]], dst[i]
    for pool in (s["k"], s["v"]):
        pool[:, to] = torch.where(use, pool[:, src], pool[:, to])
    return new.int(), lens.int(), refs.int(), torch.zeros_like(s["short"]), s["k"], s["v"]


def _accept(s):
    c = s["case"]
    page, lens = c["page"], s["lens"].long()
    d = torch.arange(c["depth"], device=DEV)
    slot, d = torch.nonzero(d < s["counts"][:, None], as_tuple=True)
    src, dst = lens[slot] + s["path"].long()[slot, d], lens[slot] + d
    ps, pd = (s["table"].long()[slot, x // page] for x in (src, dst))
    for pool in (s["k"], s["v"]):
        pool[:, pd, :, dst % page] = pool[:, ps, :, src % page]
    return (lens + s["counts"]).int(), s["k"], s["v"]


def _compact(s):
    refs, table = s["refs"], s["table"].long()
    used = (refs != 0).sum()
    ids = torch.arange(refs.shape[0], device=DEV)
    src = torch.nonzero((refs != 0) & (ids >= used)).flatten()
    dst = torch.nonzero((refs == 0) & (ids < used)).flatten()
    to = ids.clone()
    to[src] = dst
    new = torch.where(table >= 0, to[table.clamp_min(0)], table)
    counts = refs.clone()
    counts[dst] = refs[src]
    counts[src] = 0
    for pool in (s["k"], s["v"]):
        pool[:, dst] = pool[:, src]
    return new.int(), counts, used.int().view(1), s["k"], s["v"]


def _beam(s):
    c = s["case"]
    b, w, n = c["batch"], c["beams"], c["count"]
    lg = torch.nan_to_num(s["logits"].double(), nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf)
    m = lg.amax(-1, keepdim=True)
    lse = m + torch.log(torch.exp(lg - m).sum(-1, keepdim=True))
    score = s["scores"].double().unsqueeze(1)
    sc = score + (lg - lse)
    done = (s["finished"] != 0).unsqueeze(1)
    end = torch.arange(c["vocab"], device=DEV) == 2  # a beam that is done goes on with its end alone
    sc = torch.where(done, torch.where(end, score, -math.inf), sc).view(b, -1)
    best, at = (x[:, :n] for x in torch.sort(sc, dim=1, descending=True, stable=True))
    none = best == -math.inf
    beam = at // c["vocab"] + torch.arange(b, device=DEV)[:, None] * w
    token = torch.where(none, -1, at % c["vocab"]).int()
    parent = torch.where(none, -1, beam).int()
    over = torch.where(none, 0, ((s["finished"][beam] != 0) | (token == 2)).int()).int()
    rows = parent.flatten().long()
    text = torch.where((rows >= 0)[:, None], s["text"][rows.clamp_min(0)], s["next"])
    return token, parent, best.float(), over, text


def run(s):
    c = s["case"]
    kind = c["kind"]
    if not own:
        return {"attend": _attend, "append": _append, "fork": _fork, "accept": _accept, "compact": _compact,
                "beam": _beam}[kind](s)
    if kind == "beam":
        import inference_amd as qa
        token, parent, score, over = qa.beam_select(s["logits"], s["scores"], c["beams"], c["count"],
                                                    finished=s["finished"], eos=2)
        return token, parent, score, over, qa.reorder_rows(s["text"], parent.view(-1), out=s["next"])
    cache = s["cache"]
    if kind == "attend":
        return cache.attention(0, s["q"], s["starts"], masks=s["masks"], max_rows=s["max_rows"], max_len=s["max_len"])
    if kind == "append":
        q = cache.append(0, s["new_k"], s["new_v"], s["starts"], q=s["q"], cos=s["cos"], sin=s["sin"],
                         depths=s["depths"])
        return q, s["k"], s["v"]
    if kind == "fork":
        cache.fork(s["parents"], reserve=c["reserve"], out=s["new"], shortage=s["short"])
        return (*s["new"], s["short"], s["k"], s["v"])
    if kind == "accept":
        cache.accept(s["path"], s["counts"], out=s["kept"])
        return s["kept"], s["k"], s["v"]
    used = cache.compact(out=(s["new"][0], s["new"][2]))
    return s["new"][0], s["new"][2], used, s["k"], s["v"]


def work(case):
    c = case
    kind = c["kind"]
    if kind == "beam":
        rows, cand = c["batch"] * c["beams"], c["batch"] * c["count"]
        return {"bytes": rows * (c["vocab"] * SIZE[c["x"]] + 8) + cand * (16 + 8 * c["text"]),
                "flops": 4 * rows * c["vocab"]}
    token = c["kv_heads"] * c["dim"] * SIZE[c["cache"]] * 2  # a position's key and value rows in a layer
    if kind in ("attend", "append"):
        lens, rows = _lens(c), _rows(c)
        q = 2 * c["heads"] * c["dim"] * SIZE[c["x"]] * sum(rows)
        if kind == "append":
            new = 2 * c["kv_heads"] * c["dim"] * SIZE[c["x"]] + 8 * c["dim"]
            return {"bytes": q + sum(rows) * (token + new), "flops": 3 * (c["heads"] + c["kv_heads"]) * c["dim"] * sum(rows)}
        return {"bytes": q + token * sum(a + b for a, b in zip(lens, rows)),
                "flops": 4 * c["heads"] * c["dim"] * sum(b * (a + b / 2) for a, b in zip(lens, rows))}
    lists = 8 * c["slots"]
    if kind == "fork":
        lens = [c["len"] - (7 * i) % min(c["len"], 50) for i in range(c["sources"])]
        part = sum(v % c["page"] for v in lens) / len(lens) if c["reserve"] else 0
        # (of each text's holders all but one copy its last rows)
        return {"bytes": int(2 * c["layers"] * token * part * (c["slots"] - c["sources"]))
                + 8 * c["slots"] * c["max_pages"] + lists, "flops": 0}
    if kind == "accept":
        return {"bytes": int(2 * c["layers"] * token * c["slots"] * (c["depth"] - 1) * 0.5) + lists, "flops": 0}
    held = max(1, c["used"] // c["slots"]) * min(c["slots"], c["used"])
    moved = held * (c["pages"] - held) / c["pages"]  # used pages behind the first `held`, of pages anywhere
    return {"bytes": int(2 * c["layers"] * token * c["page"] * moved) + 8 * c["pages"], "flops": 0}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------

def _exact_attend(c, s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    g = c["heads"] // c["kv_heads"]
    first = 0
    for i, (n, r) in enumerate(zip(_lens(c), _rows(c))):
        ids = s["table"][i, :-(-(n + r) // c["page"])].tolist()
        k, v = (torch.cat([s[x][0, p] for p in ids], 1)[:, :n + r].double() for x in ("k", "v"))
        for j in range(r):
            if s["masks"] is None:
                keep = list(range(n + j + 1))
            else:
                word = int(s["masks"][first + j, 0])
                keep = list(range(n)) + [n + t for t in range(r) if word >> t & 1]
            keep = torch.tensor(keep, device=DEV)
            q = s["q"][first + j].double().view(c["kv_heads"], g, c["dim"])
            a = torch.softmax(torch.matmul(q, k[:, keep].transpose(1, 2).contiguous()) / math.sqrt(c["dim"]), -1)
            out[first + j] = torch.matmul(a, v[:, keep]).view(c["heads"], c["dim"])
        first += r
    return out


def _exact_append(c, s):
    pair = torch.arange(c["dim"], device=DEV)
    pair = (pair + c["dim"] // 2) % c["dim"]
    sign = torch.where(pair >= c["dim"] // 2, -1.0, 1.0).double()
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    first = 0
    for i, (n, r) in enumerate(zip(_lens(c), _rows(c))):
        for j in range(first, first + r):
            p = n + (j - first if s["depths"] is None else int(s["depths"][j]))
            co, si = s["cos"][p].double(), s["sin"][p].double()
            q[j] = q[j] * co + sign * q[j][:, pair] * si
            x = s["new_k"][j].double()
            at = n + j - first
            where = int(s["table"][i, at // c["page"]])
            k[0, where, :, at % c["page"]] = x * co + sign * x[:, pair] * si
            v[0, where, :, at % c["page"]] = s["new_v"][j].double()
        first += r
    return q, k, v


def exact(case, seed):
    kind = case["kind"]
    if kind in ("fork", "accept", "compact"):
        return None  # lists, and rows moved as they are
    s = _inputs(case, seed)
    if kind == "attend":
        return _exact_attend(case, s)
    if kind == "append":
        return _exact_append(case, s)
    best = []
    for b in range(case["batch"]):
        cand = []
        for r in range(b * case["beams"], (b + 1) * case["beams"]):
            score = float(s["scores"][r])
            if score == -math.inf:
                continue
            if int(s["finished"][r]):
                cand.append(torch.tensor([score], dtype=torch.float64, device=DEV))
            else:
                cand.append(torch.log_softmax(s["logits"][r].double(), 0).topk(min(case["count"], case["vocab"])).values
                            + score)
        top = torch.cat(cand).sort(descending=True).values[:case["count"]]
        best.append(torch.cat([top, top.new_full((case["count"] - top.shape[0],), -math.inf)]))
    return None, None, torch.stack(best), None, None
