"""Plain float64 forms of serving by drafted trees over the paged cache: attention of a tree's nodes, sampling, the accepted path, its move in the cache,
the sequences of the next step.  numpy only; loops from the definitions."""
from __future__ import annotations

import numpy as np

from oracle.paged_oracle import e4m3_decode, e4m3_round

TREE_NODES = 256


def ancestors(parents) -> np.ndarray:
    """[nodes, nodes]: whether the row's node is, or descends from, the column's.  A parent that is no earlier node is none."""
    n = len(parents)
    out = np.zeros((n, n), dtype=bool)
    for i in range(n):
        node = i
        while node >= 0:
            out[i, node] = True
            up = int(parents[node])
            node = up if 0 <= up < node else -1
    return out


def tree_attention(q, key_codes, value_codes, key_scales, value_scales, table, lengths, parents, cu_steps, scale: float):
    """As paged_oracle.attention, the new tokens being nodes of trees: outputs float64 [tokens, heads, dim] and their errors' measures."""
    pool, kv_heads, page, dim = key_codes.shape
    tokens, heads, _ = q.shape
    out = np.zeros((tokens, heads, dim))
    note = dict(spread=np.zeros((tokens, heads, dim)), score=np.zeros((tokens, heads, 1)), keys=np.zeros((tokens, heads, 1)), top=np.zeros((tokens, heads, 1)))
    for s, length in enumerate(lengths):
        n = cu_steps[s + 1] - cu_steps[s]
        if n > TREE_NODES:
            continue
        past, family = int(length) - n, ancestors(parents[cu_steps[s]:cu_steps[s + 1]])
        places = [(p, table[s, p // page]) for p in range(max(min(length, table.shape[1] * page), 0))]
        places = np.array([(p, w) for p, w in places if 0 <= w < pool], dtype=np.int64).reshape(-1, 2)
        at, which = places[:, 0], places[:, 1]
        k = e4m3_decode(key_codes[which, :, at % page]) * key_scales[which][:, :, None]
        v = e4m3_decode(value_codes[which, :, :, at % page]) * value_scales[which][:, :, None]
        for i in range(n):
            sees = np.array([p < past or family[i, p - past] for p in at], dtype=bool)
            if not sees.any():
                continue
            for h in range(heads):
                kv, t = h // (heads // kv_heads), (cu_steps[s] + i, h)
                row = q[t].astype(np.float64)
                score = k[sees, kv] @ row * scale
                w = np.exp(score - score.max()) if np.isfinite(score).all() else np.full(score.shape, np.nan)
                with np.errstate(invalid="ignore"):
                    out[t] = w @ v[sees, kv] / w.sum()
                    note["spread"][t] = w @ np.abs(v[sees, kv]) / w.sum()
                    note["score"][t] = (np.abs(k[sees, kv]) @ np.abs(row)).max() * abs(scale)
                    note["keys"][t] = sees.sum()
                    note["top"][t] = np.nanmax(np.abs(v[sees, kv]), initial=0.0) / w.sum()
    return out, note


def sample(x, u: float, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0):
    """The token of a row of logits and how far the nearest border is from what p, min_p or u are compared with: the least distance, over what weights that are rounded
    to 2 ** -44 of the largest can be off by.  n of them with the sum `total`: n * 2 ** -44, and 2 ** -45 of `total` for exponents formed in 64 bits (products of up to 44 * 2 ** -52,
    the series' rest of 7e-15); twice, for both sides of a comparison."""
    x = np.asarray(x, dtype=np.float64)
    there = [i for i in range(len(x)) if x[i] > -np.inf]
    if not there:
        return -1, np.inf
    order = sorted(there, key=lambda i: (-x[i], i))
    if not temperature > 0:
        return order[0], np.inf
    top = x[order[0]]
    w = {i: 1.0 if x[i] == top else float(np.exp((x[i] - top) / temperature)) for i in there}
    near = np.inf
    if top_k > 0:
        order = order[:top_k]
    total, kept = sum(sorted(w[i] for i in order)), []
    off = lambda total: len(there) * 2.0 ** -43 + total * 2.0 ** -44
    before = 0.0
    for rank, i in enumerate(order):
        if rank and top_p < 1 and before >= top_p * total:
            break
        kept.append(i)
        before += w[i]
        if top_p < 1:
            near = min(near, abs(before - top_p * total) / off(total))
    if min_p > 0:
        near = min(near, min(abs(w[i] - min_p) for i in kept) / off(1.0))
        kept = [i for i in kept if w[i] >= min(min_p, 1.0)]
    kept.sort()
    total = sum(sorted(w[i] for i in kept))
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    so_far = 0.0
    for i in kept:
        so_far += w[i]
        near = min(near, abs(so_far - u * total) / off(total))
        if so_far > u * total:
            return i, near
    return kept[-1], near


def accept(parents, drafted, sampled, lengths, cu_steps, most: int):
    kept = np.full((len(lengths), most), -1, dtype=np.int32)
    counts, tokens, news = [], [], []
    for s, length in enumerate(lengths):
        at, n = cu_steps[s], cu_steps[s + 1] - cu_steps[s]
        path = [0] if n > 0 else []
        while path and len(path) < most:
            here = path[-1]
            child = [i for i in range(here + 1, min(n, TREE_NODES)) if parents[at + i] == here and drafted[at + i] == sampled[at + here]]
            if not child:
                break
            path.append(child[0])
        kept[s, :len(path)] = path
        counts.append(len(path))
        tokens.append(sampled[at + path[-1]] if path else -1)
        news.append(max(int(length) - n + len(path), 0))
    return kept, np.array(counts), np.array(tokens), np.array(news)


def compact(key_codes, value_codes, key_scales, value_scales, table, lengths, kept, counts, steps):
    """The four arrays of one layer afterwards: codes as values [pool, kv_heads, page, dim] / [pool, kv_heads, dim, page], scales.  steps: nodes of every sequence."""
    pool, kv_heads, page, dim = key_codes.shape
    out = []
    for codes, scales in ((e4m3_decode(key_codes), key_scales.astype(np.float64)), (e4m3_decode(value_codes).transpose(0, 1, 3, 2), value_scales.astype(np.float64))):
        new, new_scales = codes.copy(), scales.copy()
        for s, n in enumerate(steps):
            if not 0 < n <= TREE_NODES:
                continue
            first, path = int(lengths[s]) - int(n), []
            for node in kept[s, :max(min(counts[s], n, kept.shape[1]), 0)]:
                if node <= (path[-1] if path else -1) or node >= n:
                    break
                path.append(int(node))
            where = lambda p: (table[s, p // page], p % page) if p >= 0 and p // page < table.shape[1] and 0 <= table[s, p // page] < pool else None
            by_page = {}
            for j, node in enumerate(path):
                if where(first + j) is not None:
                    by_page.setdefault((first + j) // page, []).append((first + j, first + node))
            for p, moves in sorted(by_page.items()):
                to = table[s, p]
                if all(a == b for a, b in moves):
                    continue
                moves = [(a, where(b)) for a, b in moves if where(b) is not None]
                if not moves:
                    continue
                held = max(first, p * page) - p * page
                scale = np.max([scales[w[0]] for _, w in moves] + ([scales[to]] if held else []), axis=0)
                if held:
                    new[to, :, :held] = e4m3_round(codes[to, :, :held] * (scales[to] / scale)[:, None, None])
                for a, (which, slot) in moves:
                    new[to, :, a % page] = e4m3_round(codes[which, :, slot] * (scales[which] / scale)[:, None])
                new_scales[to] = scale
        out.append((new, new_scales))
    return out[0][0], out[1][0].transpose(0, 1, 3, 2), out[0][1], out[1][1]


def fork(table, uses, sources, kept, reserve, page: int):
    """New table, uses, missing pages per row and the copies [(from, to)].  Room ends with the table; of it a row lacks what the pool has no page for, and a page kept in part that the
    source has not."""
    seqs, width = table.shape
    pool = len(uses)
    uses = [int(n) for n in uses]
    for p in table.reshape(-1):
        if 0 <= p < pool:
            uses[p] -= 1
    rows = []
    for r, src in enumerate(sources):
        src = int(src) if 0 <= src < seqs else -1
        n = min(max(int(kept[r]), 0), width * page) if src >= 0 else 0
        shared = [int(p) if 0 <= p < pool else -1 for p in table[src, :n // page]] if src >= 0 else []
        for p in shared:
            if p >= 0:
                uses[p] += 1
        begun = None
        if n % page:
            begun = int(table[src, n // page])
            begun = begun if 0 <= begun < pool else -1
        rows.append([shared, begun, -(-min(max(int(reserve[r]), n), width * page) // page)])
    first, stay = {}, {}
    for r, (_, begun, _) in enumerate(rows):
        if begun is not None and begun >= 0:
            first.setdefault(begun, r)
    for p, r in first.items():
        if uses[p] <= 0:
            stay[r] = p
    uses = [max(n, 0) for n in uses]
    for p in stay.values():
        uses[p] = 1
    free = [p for p in range(pool) if uses[p] == 0]
    copies, missing, out = [], [], np.full((len(rows), width), -1, dtype=np.int32)
    for r, (pages, begun, last) in enumerate(rows):
        pages, lacks = list(pages), 0
        copied = None
        if begun is not None:
            if begun < 0 or r in stay:
                pages.append(begun)
                lacks += begun < 0
            else:
                copied = begun
        while len(pages) < last:
            p = free.pop(0) if free else -1
            if p >= 0:
                uses[p] = 1
                if copied is not None:
                    copies.append((copied, p))
            else:
                lacks += 1
            copied = None
            pages.append(p)
        out[r, :len(pages)] = pages
        missing.append(lacks)
    return out, np.array(uses), np.array(missing), copies
