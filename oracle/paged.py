"""The cache in pages and the beam search's selection in 64 bits and plain loops (numpy), written from their
definitions: what the kernels are compared with."""
import math

import numpy as np


def page_of(table, slot, j, pages):
    p = int(table[slot][j]) if 0 <= j < len(table[slot]) else -1
    return p if 0 <= p < pages else -1


def gather(pool, table, slot, n):
    """Rows 0 .. n - 1 of a slot from one layer's pool [pages, kv, page, dim]: [n, kv, dim] in 64 bits."""
    page = pool.shape[2]
    out = np.full((n, pool.shape[1], pool.shape[3]), np.nan)
    for t in range(n):
        p = page_of(table, slot, t // page, pool.shape[0])
        if p >= 0:
            out[t] = pool[p, :, t % page].astype(np.float64)
    return out


def sees(masks, row, j, i):
    """Whether row j (packed row `row`) sees its step's row i."""
    if masks is None:
        return i <= j
    return i < 64 * masks.shape[1] and bool(int(masks[row][i // 64]) >> (i % 64) & 1)


def attention(q, kpool, vpool, table, lens, starts, masks, scale, max_rows=None):
    """(out [rows, heads, dim] in 64 bits with NaN in rows of no slot, and what a tolerance needs: the sums of
    weight * |v|, and the largest of sum |q k| * scale and of |score|, per row and head)."""
    rows, heads, dim = q.shape
    kv, page = kpool.shape[1], kpool.shape[2]
    g = heads // kv
    out = np.full((rows, heads, dim), np.nan)
    mag = np.zeros((rows, heads, dim))
    dot = np.zeros((rows, heads, 1))
    top = np.zeros((rows, heads, 1))
    cap = table.shape[1] * page
    for s in range(table.shape[0]):
        a, b = int(starts[s]), min(int(starts[s + 1]), rows)
        if a < 0 or a >= rows:
            continue
        b = a + min(max(b - a, 0), rows if max_rows is None else max_rows)
        base = min(max(int(lens[s]), 0), cap)
        n = min(base + b - a, cap)
        k, v = gather(kpool, table, s, n), gather(vpool, table, s, n)
        for j in range(b - a):
            seen = [t for t in range(n) if t < base or sees(masks, a + j, j, t - base)]
            if not seen:
                out[a + j] = 0.0
                continue
            for h in range(heads):
                x = q[a + j, h].astype(np.float64)
                kk, vv = k[seen, h // g], v[seen, h // g]
                sc = kk @ x * scale
                w = np.exp(sc - sc.max())
                w /= w.sum()
                out[a + j, h] = w @ vv
                mag[a + j, h] = w @ np.abs(vv)
                dot[a + j, h] = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                top[a + j, h] = np.abs(sc).max()
    return out, mag, dot, top


def turn(x, cos, sin):
    half = x.shape[-1] // 2
    return x * cos + np.concatenate([-x[..., half:], x[..., :half]], -1) * sin


def fork(table, lens, refs, page, parents, keep, reserve):
    """(table, lens, refs, shortage, copies [(source, destination, rows)]) after a fork; the lists as they were where
    pages are missing."""
    table, lens, refs = table.astype(np.int64), lens.astype(np.int64), refs.astype(np.int64)
    slots, wide = table.shape
    pages = len(refs)
    cap = wide * page
    new_refs = refs.copy()
    for row in table:
        for p in row:
            if 0 <= p < pages:
                new_refs[p] -= 1
    rows, new_lens, want = [], [], []
    over = 0
    for i in range(slots):
        p = int(parents[i])
        ok = 0 <= p < slots
        n = min(max(int(lens[p]), 0), cap) if ok else 0
        if keep is not None and keep[i] >= 0:
            n = min(n, int(keep[i]))
        held = -(-n // page)
        total = -(-(n + reserve) // page) if ok else 0
        row = [int(x) if 0 <= x < pages else -1 for x in table[p][:held]] if ok else []
        for x in row:
            if x >= 0:
                new_refs[x] += 1
        rows.append(row)
        new_lens.append(n)
        want.append(max(total - held, 0))
        over += max(total - wide, 0)
    last = [rows[i][-1] if reserve > 0 and new_lens[i] % page else -1 for i in range(slots)]
    copying = []
    for i in range(slots):
        w = last[i]
        sharers = [j for j in range(slots) if w >= 0 and last[j] == w]
        copying.append(w >= 0 and not (new_refs[w] == len(sharers) and sharers[0] == i))
    free = [p for p in range(pages) if new_refs[p] == 0]
    need = sum(want[i] if want[i] <= wide - len(rows[i]) else wide - len(rows[i]) for i in range(slots)) + sum(copying)
    missing = max(need - len(free), 0) + over
    if missing:
        return table, lens, refs, missing, []
    copies = []
    out = np.full((slots, wide), -1, np.int64)
    for i in range(slots):
        row = list(rows[i])
        if copying[i]:
            to = free.pop(0)
            copies.append((row[-1], to, new_lens[i] % page))
            new_refs[row[-1]] -= 1
            new_refs[to] = 1
            row[-1] = to
        for _ in range(want[i]):
            to = free.pop(0)
            new_refs[to] = 1
            row.append(to)
        out[i, :len(row)] = row
    return out, np.array(new_lens), new_refs, 0, copies


def accept_lengths(table, lens, pages, page, path, counts):
    """How many entries of each slot's path hold."""
    out = []
    cap = table.shape[1] * page
    for s in range(len(lens)):
        base, last, d = min(max(int(lens[s]), 0), cap), -1, 0
        while d < int(counts[s]) and (path is None or d < path.shape[1]):
            to = d if path is None else int(path[s][d])
            if to <= last or base + to >= cap or page_of(table, s, (base + to) // page, pages) < 0 or \
                    page_of(table, s, (base + d) // page, pages) < 0:
                break
            last, d = to, d + 1
        out.append(d)
    return out


def accept(pools, table, lens, path, counts):
    """The pools [layers, pages, kv, page, dim] changed in place, and the new lengths."""
    page, pages = pools[0].shape[3], pools[0].shape[1]
    n = accept_lengths(table, lens, pages, page, path, counts)
    new = []
    for s, m in enumerate(n):
        base = min(max(int(lens[s]), 0), table.shape[1] * page)
        for d in range(m):
            to = d if path is None else int(path[s][d])
            for pool in pools:
                pool[:, table[s][(base + d) // page], :, (base + d) % page] = \
                    pool[:, table[s][(base + to) // page], :, (base + to) % page]
        new.append(base + m)
    return np.array(new)


def compact(table, refs):
    """(table, refs, used, moves [(source, destination)])."""
    used = int((refs != 0).sum())
    src = [p for p in range(used, len(refs)) if refs[p] != 0]
    dst = [p for p in range(used) if refs[p] == 0]
    to = {a: b for a, b in zip(src, dst)}
    new = refs.copy()
    for a, b in zip(src, dst):
        new[b], new[a] = refs[a], 0
    return np.vectorize(lambda p: to.get(p, p))(table), new, used, list(zip(src, dst))


def beam(logits, scores, beams, count, finished=None, eos=-1):
    """(tokens, parents, scores in 64 bits, finished) of [searches, count]."""
    rows = len(scores)
    out = []
    for b in range(rows // beams):
        cand = []
        for w in range(beams):
            r = b * beams + w
            score = float(scores[r])
            if not score > -math.inf:
                continue
            if finished is not None and finished[r]:
                cand.append((-score, w, 0, eos))
                continue
            lg = logits[r].astype(np.float64)
            lg = np.where(np.isnan(lg), -np.inf, np.minimum(lg, np.finfo(np.float32).max))
            m = lg.max()
            if m == -np.inf:
                continue
            lse = m + math.log(np.exp(lg - m).sum())
            # (the largest logits alone: the order within a beam is theirs, ties to the lower token)
            for place, i in enumerate(np.argsort(-lg, kind="stable")[:count]):
                if lg[i] > -np.inf:
                    cand.append((-(score + (lg[i] - lse)), w, place, int(i)))
        cand.sort()
        cand = cand[:count]
        row = [(t, b * beams + w, -s, int(bool(finished is not None and finished[b * beams + w]) or t == eos))
               for s, w, _, t in cand]
        out.append(row + [(-1, -1, -math.inf, 0)] * (count - len(row)))
    t = np.array([[c[0] for c in r] for r in out])
    p = np.array([[c[1] for c in r] for r in out])
    s = np.array([[c[2] for c in r] for r in out])
    f = np.array([[c[3] for c in r] for r in out])
    return t, p, s, f
