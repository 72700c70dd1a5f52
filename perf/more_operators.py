"""Serving by drafted trees over the paged E4M3 cache: what is measured, and the operators' plain forms.

    tree     attention of the nodes of a drafted tree per sequence: each sees the past, its ancestors and itself      (paged_attention_tree_forward)
    sample   a token per row of logits by temperature, top-k, top-p and min-p from given random numbers               (sample_tokens_forward)
    accept   the path of a drafted tree that the sampled tokens follow                                                (draft_tree_accept_forward)
    compact  the keys and values of that path to the places right behind the past, in every layer's cache             (paged_cache_compact_forward)
    fork     the sequences of the next step out of the present ones: pages shared, copied, taken and freed            (paged_cache_fork_forward)

Sizes: head counts, head widths and the vocabulary of bench.py (48 query and 8 key/value heads of 128, 200064 tokens), and generic ones beside them; trees
of one to 256 nodes, pasts of one position to 131072.  The cache: key pages [pages, kv_heads, page, head_dim], value pages [pages, kv_heads, head_dim, page],
one power-of-two float32 scale per page and key/value head.

With `own` false `run` computes the same in elementary torch operations, attention in float32, the sampler's weights and sums in float64 (a float32 sum over a
vocabulary is coarser than a token's share); `exact` computes all of it in float64, by loops.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn


# ---- the cases ---------------------------------------------------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # one sequence, a tree of eight nodes, 64-wide heads of their own keys: the smallest attention call, latency counts
        dict(name="tree_token", op="tree", seqs=1, nodes=8, even=True, ragged=False, past=700, heads=32, kv_heads=32, dim=64, page=16, dtype="f16"),
        # a serving step: 32 sequences of up to 8192 positions, 26 nodes each
        dict(name="tree_batch", op="tree", seqs=32, nodes=26, even=True, ragged=True, past=8191, heads=48, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # a few sequences with wide trees of different sizes behind long pasts: the largest products
        dict(name="tree_long", op="tree", seqs=5, nodes=200, even=False, ragged=True, past=30000, heads=64, kv_heads=8, dim=128, page=32, dtype="f16"),
        # the token of one sequence: the smallest call over a large vocabulary
        dict(name="sample_token", op="sample", rows=1, vocab=200064, dtype="f32", mixed=False, spread=3.0),
        # every node of 32 trees of 26, each sequence with parameters of its own, some of them greedy
        dict(name="sample_nodes", op="sample", rows=832, vocab=32000, dtype="f16", mixed=True, spread=2.5),
        # a batch over a large vocabulary
        dict(name="sample_wide", op="sample", rows=96, vocab=200064, dtype="bf16", mixed=True, spread=2.0),
        # one tree of 26 nodes
        dict(name="accept_one", op="accept", seqs=1, nodes=26, even=True),
        # 256 trees of up to 200 nodes
        dict(name="accept_batch", op="accept", seqs=256, nodes=200, even=False),
        # one sequence's accepted path, two layers
        dict(name="compact_one", op="compact", seqs=1, nodes=64, even=True, past=900, layers=2, kv_heads=8, dim=128, page=64),
        # 32 sequences, eight layers, paths that cross pages
        dict(name="compact_batch", op="compact", seqs=32, nodes=26, even=False, past=400, layers=8, kv_heads=8, dim=128, page=16),
        # four prompts become 16 beams
        dict(name="fork_beams", op="fork", seqs=4, rows=16, past=1000, room=8, layers=2, kv_heads=8, dim=128, page=16),
        # a serving step of 64 sequences: most go on, some branch, some end, new ones begin
        dict(name="fork_step", op="fork", seqs=64, rows=64, past=4000, room=26, layers=4, kv_heads=8, dim=128, page=64),
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _cost(case: dict) -> float:
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 1e15


def draw(rng) -> dict:
    """One more case of the ranges that the listed ones stand for."""
    largest = {}
    for c in listed():
        largest[c["op"]] = max(largest.get(c["op"], 0.0), _cost(c))
    op = rng.choice(["tree", "tree", "tree", "sample", "sample", "accept", "compact", "fork"])
    while True:
        if op == "sample":
            case = dict(op=op, rows=_spread(rng, 1, 1024), vocab=_spread(rng, 500, 262144), dtype=rng.choice(["bf16", "f16", "f32"]), mixed=rng.random() < 0.7,
                        spread=rng.choice([1.0, 2.0, 3.0, 5.0]))
        elif op == "accept":
            case = dict(op=op, seqs=_spread(rng, 1, 256), nodes=_spread(rng, 1, 256), even=rng.random() < 0.5)
        else:
            kv_heads = rng.choice([1, 2, 4, 8, 8, 32])
            case = dict(op=op, dim=rng.choice([64, 128, 128]), kv_heads=kv_heads, page=rng.choice([16, 32, 64, 128]))
            if op == "tree":
                case.update(heads=rng.choice([1, 2, 4, 5, 6, 8, 8, 16]) * kv_heads, seqs=_spread(rng, 1, 64), nodes=_spread(rng, 1, 256), even=rng.random() < 0.5,
                            ragged=rng.random() < 0.7, past=_spread(rng, 1, 131072) - 1, dtype=rng.choice(["bf16", "f16"]))
                if case["heads"] > 64:
                    continue
            elif op == "compact":
                case.update(seqs=_spread(rng, 1, 64), nodes=_spread(rng, 1, 256), even=rng.random() < 0.5, past=_spread(rng, 1, 2000) - 1, layers=rng.choice([1, 2, 3, 5, 8]))
            else:
                case.update(seqs=_spread(rng, 1, 64), rows=_spread(rng, 1, 96), past=_spread(rng, 1, 4000), room=_spread(rng, 1, 256), layers=rng.choice([1, 2, 3, 4]))
        if _cost(case) <= largest[op]:
            return case


def _rng_of(case: dict):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _nodes(case: dict, rng) -> list[int]:
    return [case["nodes"] if case["even"] else rng.randint(max(1, case["nodes"] // 8), case["nodes"]) for _ in range(case["seqs"])]


def _trees(case: dict):
    """Nodes, pasts and parents (-1 for a root, else an earlier node of the tree) of every sequence, the same for every seed."""
    rng = _rng_of(case)
    nodes = _nodes(case, rng)
    pasts = [rng.randint(0, case["past"]) if case.get("ragged", True) else case["past"] for _ in nodes] if "past" in case else [0] * len(nodes)
    parents = [[-1] + [rng.randint(i // 4, i - 1) for i in range(1, n)] for n in nodes]
    return nodes, pasts, parents


def _path(rng, n: int) -> list[int]:
    """The nodes of an accepted path through a tree of n: rising, the root first."""
    count = min(n, 1 + min(rng.randint(0, 12), rng.randint(0, 12)))
    return [0] + sorted(rng.sample(range(1, n), count - 1))


def _fork_plan(case: dict):
    """What the present rows hold (pages each), and source (-1: none), tokens kept and tokens to have room for of the next ones."""
    rng, page = _rng_of(case), case["page"]
    lengths = [rng.randint(1, case["past"]) for _ in range(case["seqs"])]
    held = [-(-(n + case["room"]) // page) for n in lengths]                   # (room for the last step's tree)
    sources, kept, reserve = [], [], []
    for r in range(case["rows"]):
        kind = rng.random()
        s = rng.randrange(case["seqs"]) if case["rows"] > case["seqs"] or kind < 0.2 else r % case["seqs"]
        n = lengths[s] - (rng.randint(0, min(lengths[s], 3 * page)) if kind > 0.9 else 0)
        if 0.2 <= kind < 0.27:
            s, n = -1, 0                                                      # a row for a new prompt
        sources.append(s)
        kept.append(n)
        reserve.append(n + (rng.randint(1, case["past"]) if s < 0 else case["room"]))
    return held, sources, kept, reserve


def _fork_layout(case: dict):
    """Page counts of the rows, width of the tables, pages of the pool (what the next rows need, and a few more)."""
    held, sources, kept, reserve = _fork_plan(case)
    page = case["page"]
    need = sum(-(-r // page) - k // page for k, r in zip(kept, reserve))
    width = max(held + [-(-r // page) for r in reserve])
    return held, width, sum(held) + need + 5


# ---- what a user's program has before the call ------------------------------------------------------------------------

def _codes(g, *shape) -> torch.Tensor:
    """Codes of values of unit size."""
    codes = torch.empty(*shape, dtype=F8, device=DEV)
    part = max(1, (64 << 20) // max(1, math.prod(shape[1:])))
    for first in range(0, shape[0], part):
        some = codes[first:first + part]
        some.copy_((torch.randn(some.shape, generator=g, device=DEV) * 96.0).clamp_(-448, 448).to(F8))
    return codes


def _pool(g, case: dict, pool: int):
    """Pages and scales; pages of somewhat different size, so of different scales."""
    kv_heads, page, dim = case["kv_heads"], case["page"], case["dim"]
    pages = [_codes(g, pool, kv_heads, page, dim), _codes(g, pool, kv_heads, dim, page)]
    return (*pages, *(torch.pow(2.0, torch.randint(-8, -5, (pool, kv_heads), generator=g, device=DEV).float()).contiguous() for _ in pages))


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _table(g, counts: list[int], width: int, pool: int) -> torch.Tensor:
    """Rows of page numbers in no order, -1 behind a row's last page."""
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = order[at:at + c]
        at += c
    return table


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    host = random.Random(int(seed))
    state = dict(case=case)
    if case["op"] == "sample":
        rows = case["rows"]
        # logits of a language model: a wide bulk, a few tokens ahead of it
        logits = torch.randn(rows, case["vocab"], generator=g, device=DEV) * case["spread"]
        ahead = torch.randint(0, case["vocab"], (rows, 12), generator=g, device=DEV)
        logits.scatter_add_(1, ahead, torch.rand(rows, 12, generator=g, device=DEV) * 4.0 * case["spread"])
        logits[:, torch.randint(0, case["vocab"], (7,), generator=g, device=DEV)] = float("-inf")          # tokens that are not allowed
        state.update(logits=logits.to(DTYPES[case["dtype"]]), uniform=torch.rand(rows, generator=g, device=DEV))
        if case["mixed"]:
            pick = lambda values, dtype: torch.tensor([host.choice(values) for _ in range(rows)], dtype=dtype, device=DEV)
            state.update(temperature=pick([0.0, 0.3, 0.7, 1.0, 1.0, 1.3], torch.float32), top_k=pick([0, 0, 1, 20, 50, 1000], torch.int32),
                         top_p=pick([1.0, 0.5, 0.9, 0.95, 0.99], torch.float32), min_p=pick([0.0, 0.0, 0.02, 0.1], torch.float32))
        else:
            state.update(temperature=0.8, top_k=50, top_p=0.95, min_p=0.0)
        return state
    if case["op"] == "fork":
        held, sources, kept, reserve = _fork_plan(case)
        _, width, pool = _fork_layout(case)
        table = _table(g, held, width, pool)
        uses = torch.zeros(pool, dtype=torch.int32, device=DEV)
        uses[table[table >= 0].long()] = 1
        own_pages = torch.nonzero(uses).view(-1)
        uses[own_pages[torch.randint(0, own_pages.numel(), (3,), generator=g, device=DEV)]] += 1            # pages that a store of prefixes holds too
        state.update(layers=[_pool(g, case, pool) for _ in range(case["layers"])], table=table, uses=uses, sources=_ints(sources), kept=_ints(kept), reserve=_ints(reserve),
                     plan=(held, sources, kept, reserve))
        return state
    nodes, pasts, parents = _trees(case)
    cu = [0]
    for n in nodes:
        cu.append(cu[-1] + n)
    lengths = [p + n for p, n in zip(pasts, nodes)]
    state.update(nodes=nodes, pasts=pasts, cu_host=cu, cu_steps=_ints(cu), lengths=_ints(lengths), parents_host=parents, parents=_ints(sum(parents, [])))
    if case["op"] == "accept":
        # drafted tokens, siblings different; what is sampled at a node is one of its children more often than not
        drafted, sampled = [], []
        for tree in parents:
            tokens = host.sample(range(30000), len(tree))
            children = [[] for _ in tree]
            for i, p in enumerate(tree):
                if p >= 0:
                    children[p].append(i)
            drafted += tokens
            sampled += [tokens[host.choice(c)] if c and host.random() < 0.7 else 30000 + host.randrange(2000) for c in children]
        state.update(drafted=torch.tensor(drafted, device=DEV), sampled=torch.tensor(sampled, device=DEV))
        return state
    page = case["page"]
    counts = [-(-n // page) for n in lengths]
    pool, width = sum(counts) + 3, max(counts)
    state["table"] = _table(g, counts, width, pool)
    if case["op"] == "compact":
        paths = [_path(host, n) for n in nodes]
        most = max(nodes)
        state.update(layers=[_pool(g, case, pool) for _ in range(case["layers"])], paths=paths, kept=_ints([p + [-1] * (most - len(p)) for p in paths]),
                     counts=_ints([len(p) for p in paths]))
        return state
    state.update(cache=_pool(g, case, pool), q=torch.randn(cu[-1], case["heads"] * case["dim"], generator=g, device=DEV).to(DTYPES[case["dtype"]]) * 1.5)
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------

def _held(s: dict, seq: int, length: int, dtype: torch.dtype):
    """Keys and values [kv_heads, length, dim] of one sequence."""
    key_pages, value_pages, key_scales, value_scales = s["cache"]
    ids = s["table"][seq, :-(-length // s["case"]["page"])].long()
    k = key_pages[ids].to(dtype) * key_scales[ids].to(dtype)[:, :, None, None]
    v = value_pages[ids].to(dtype) * value_scales[ids].to(dtype)[:, :, None, None]
    kv_heads, dim = k.size(1), k.size(3)
    k = k.permute(1, 0, 2, 3).reshape(kv_heads, -1, dim)[:, :length].contiguous()
    v = v.permute(1, 0, 3, 2).reshape(kv_heads, -1, dim)[:, :length].contiguous()
    return k, v


def _plain_tree(s: dict) -> torch.Tensor:
    c, q = s["case"], s["q"]
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    group, out = heads // kv_heads, torch.empty_like(q)
    for seq, (n, past) in enumerate(zip(s["nodes"], s["pasts"])):
        at, length = s["cu_host"][seq], past + n
        keys, values = _held(s, seq, length, torch.float32)
        # who descends from whom: (1 + steps to the parent) to a power of at least the depth
        nodes = torch.arange(n, device=DEV)
        sees = ((nodes[None] == nodes[:, None]) | (nodes[None] == s["parents"][at:at + n, None])).float()
        for _ in range(max(1, (n - 1).bit_length())):
            sees = (torch.matmul(sees, sees) > 0).float()
        hidden = torch.cat([torch.zeros(n, past, dtype=torch.bool, device=DEV), sees == 0], 1)
        rows = q[at:at + n].float().view(n, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * n, dim).contiguous()
        got = torch.empty_like(rows)
        together = max(1, (1 << 30) // max(1, group * n * length))            # heads whose scores fit beside one another
        for h in range(0, kv_heads, together):
            scores = torch.matmul(rows[h:h + together], keys[h:h + together].transpose(1, 2).contiguous()) * dim ** -0.5
            scores.view(-1, group, n, length).masked_fill_(hidden, float("-inf"))
            scores = torch.exp(scores - scores.amax(-1, keepdim=True))
            got[h:h + together] = torch.matmul(scores, values[h:h + together]) / scores.sum(-1, keepdim=True)
        out[at:at + n] = got.view(kv_heads, group, n, dim).permute(2, 0, 1, 3).reshape(n, heads * dim).to(q.dtype)
    return out


def _column(v, rows: int, dtype: torch.dtype) -> torch.Tensor:
    """A parameter of every row, [rows, 1]."""
    return (v.to(dtype) if isinstance(v, torch.Tensor) else torch.full((rows,), v, dtype=torch.float32, device=DEV).to(dtype))[:, None]


def _plain_sample(s: dict) -> torch.Tensor:
    rows, vocab = s["logits"].shape
    x = s["logits"].double()
    x = torch.where(x.isnan(), -math.inf, x)
    t, k = _column(s["temperature"], rows, torch.float64), _column(s["top_k"], rows, torch.int64)
    top_p, min_p = _column(s["top_p"], rows, torch.float64), _column(s["min_p"], rows, torch.float64)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)             # equal ones by rising index
    most = x[:, :1]
    w = torch.where(x == most, 1.0, torch.exp((x - most) / torch.where(t > 0, t, 1.0)))
    w = torch.where(x == -math.inf, 0.0, w)
    rank = torch.arange(vocab, device=DEV)[None]
    keep = (rank < torch.where(k > 0, k, vocab)) & (w >= min_p)
    inside = torch.where(rank < torch.where(k > 0, k, vocab), w, 0.0)
    before = torch.cumsum(inside, -1)
    keep &= (top_p >= 1) | (rank == 0) | (before - inside < top_p * before[:, -1:])
    keep &= (t > 0) | (rank == 0)
    shares = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0)).cumsum(-1)
    u = s["uniform"].double().clamp(0, 1 - 2.0 ** -24)[:, None]
    token = (shares <= u * shares[:, -1:]).sum(-1)
    return torch.where(most[:, 0] == -math.inf, -1, token.clamp_max(vocab - 1))


def _plain_accept(s: dict):
    c = s["case"]
    cu = s["cu_steps"].long()
    nodes, most = cu[1:] - cu[:-1], c["nodes"]
    place = torch.arange(most, device=DEV)[None]
    there = place < nodes[:, None]
    at = (cu[:-1, None] + place).clamp_max(s["drafted"].numel() - 1)
    parents, drafted = torch.where(there, s["parents"][at].long(), -2), s["drafted"][at]
    here = torch.zeros_like(nodes)                                            # the path's last node
    kept, going = [here.clone()], torch.ones_like(nodes, dtype=torch.bool)
    token = s["sampled"][cu[:-1]]
    for _ in range(most - 1):
        match = (parents == here[:, None]) & (drafted == token[:, None]) & (place > here[:, None])
        child = torch.where(match, place, most).amin(-1)
        going = going & (child < most)
        here = torch.where(going, child, here)
        token = s["sampled"][cu[:-1] + here]
        kept.append(torch.where(going, child, -1))
    kept = torch.stack(kept, 1).to(torch.int32)
    counts = (kept >= 0).sum(-1).to(torch.int32)
    return kept, counts, token, s["lengths"] - nodes.to(torch.int32) + counts


def _plain_compact(s: dict):
    page = s["case"]["page"]
    cu = s["cu_steps"].long()
    first = s["lengths"].long() - (cu[1:] - cu[:-1])
    most, pool = s["kept"].size(1), s["layers"][0][0].size(0)
    seq = torch.arange(first.numel(), device=DEV)[:, None].expand(-1, most)
    rank = torch.arange(most, device=DEV)[None].expand(first.numel(), -1)
    valid = rank < s["counts"][:, None]
    src, dst = (first[:, None] + s["kept"]).clamp_min(0), first[:, None] + rank
    width = s["table"].size(1)
    src_page = s["table"][seq, (src // page).clamp_max(width - 1)].long()
    dst_page = s["table"][seq, (dst // page).clamp_max(width - 1)].long()
    valid, src_page, dst_page, src, dst = (t.reshape(-1) for t in (valid, src_page, dst_page, src % page, dst % page))
    # (places that are not on a path write to a page of no sequence, one more than the pool has)
    dst_page = torch.where(valid, dst_page, pool)
    src_page = torch.where(valid, src_page, 0)
    begun = s["table"][seq[:, 0], (first // page).clamp_max(width - 1)].long()
    held = torch.zeros(pool + 1, dtype=torch.long, device=DEV)
    held[torch.where(first % page > 0, begun, pool)] = first % page           # slots of a page that keep what they have
    written = torch.zeros(pool + 1, dtype=torch.bool, device=DEV)
    written[dst_page] = True
    written[pool] = False
    held, written = held[:pool], written[:pool]
    for keys, values, key_scales, value_scales in s["layers"]:
        for pages, scales, tokens_last in ((keys, key_scales, False), (values, value_scales, True)):
            kv_heads = scales.size(1)
            from_scale = scales[src_page]
            new = torch.zeros(pool + 1, kv_heads, device=DEV).scatter_reduce(0, dst_page[:, None].expand(-1, kv_heads), torch.where(valid[:, None], from_scale, 0.0), "amax")[:pool]
            new = torch.where((held > 0)[:, None], torch.maximum(new, scales), new)
            new = torch.where(written[:, None], new, scales)
            per_token = pages.transpose(2, 3) if tokens_last else pages       # [pool, kv_heads, page, dim]
            to_scale = torch.cat([new, torch.ones(1, kv_heads, device=DEV)])[dst_page]
            moved = (per_token[src_page, :, src].float() * (from_scale / to_scale)[:, :, None]).to(F8)
            again = (per_token.float() * (scales / new)[:, :, None, None]).to(F8)
            old = (torch.arange(page, device=DEV)[None] < held[:, None]) & written[:, None]
            whole = torch.cat([torch.where(old[:, None, :, None], again.float(), per_token.float()).to(F8), torch.zeros(1, *per_token.shape[1:], device=DEV).to(F8)])
            whole.view(torch.uint8)[dst_page, :, dst] = moved.view(torch.uint8)
            per_token.copy_(whole[:pool])
            scales.copy_(new)
    return [t for layer in s["layers"] for t in layer]


def _plain_fork(s: dict):
    table, page, pool = s["table"].long(), s["case"]["page"], s["uses"].numel()
    rows, width = s["sources"].numel(), s["table"].size(1)
    count = lambda entries: torch.zeros(pool + 1, dtype=torch.long, device=DEV).index_add_(0, torch.where(entries >= 0, entries, pool).reshape(-1), torch.ones(entries.numel(), dtype=torch.long, device=DEV))[:pool]
    source = s["sources"].long()
    kept = torch.where(source >= 0, s["kept"].long(), 0)
    full, some, last = kept // page, kept % page > 0, (torch.maximum(s["reserve"].long(), kept) + page - 1) // page
    place = torch.arange(width, device=DEV)[None]
    theirs = torch.where(source[:, None] >= 0, table[source.clamp_min(0)], -1)
    shared = torch.where(place < full[:, None], theirs, -1)
    uses = s["uses"].long() - count(table) + count(shared)
    # a page that a row goes on to fill: its own if no other row and no other holder has it (of several such rows the first), else copied
    begun = torch.where(some, theirs.gather(1, full.clamp_max(width - 1)[:, None])[:, 0], -1)
    row = torch.arange(rows, device=DEV)
    begun_at = torch.where(begun >= 0, begun, pool)
    first = torch.full((pool + 1,), rows, device=DEV).scatter_reduce(0, begun_at, row, "amin")
    stays = (begun >= 0) & (first[begun_at] == row) & (torch.cat([uses, uses.new_ones(1)])[begun_at] == 0)
    copied = (begun >= 0) & ~stays
    uses = uses + count(torch.where(stays, begun, -1))
    # the free pages, lowest first, to the rows one after the other
    wants = (place >= full[:, None] + some[:, None]) & (place < last[:, None]) | copied[:, None] & (place == full[:, None])
    rank = torch.cumsum(wants.reshape(-1), 0).view(rows, width) - 1
    free = torch.argsort((uses > 0).to(torch.int8), stable=True)
    held = (uses > 0).to(torch.int8).argmax()
    given = wants & (rank < (uses <= 0).sum())
    fresh = torch.where(given, free[rank.clamp(0, pool - 1)], -1)
    uses = uses + count(fresh)
    out = torch.where(wants, fresh, shared)
    out = torch.where((stays[:, None]) & (place == full[:, None]), begun[:, None], out)
    to = torch.where(copied, out.gather(1, full.clamp_max(width - 1)[:, None])[:, 0], -1)
    copied = copied & (to >= 0)
    to, begun = torch.where(copied, to, held), torch.where(copied, begun, held)                           # (rows without a copy: a page onto itself, one that none goes to)
    for layer in s["layers"]:
        for t in layer:
            t = t.view(torch.uint8) if t.dtype == F8 else t
            t[to] = t[begun]
    return [out.to(torch.int32), uses.clamp_min(0).to(torch.int32), (wants & ~given).sum(-1).to(torch.int32)] + [t for layer in s["layers"] for t in layer]


# ---- one pass ---------------------------------------------------------------------------------------------------------

PLAIN = {"tree": _plain_tree, "sample": _plain_sample, "accept": _plain_accept, "compact": _plain_compact, "fork": _plain_fork}


def run(state: dict):
    c = state["case"]
    if not own:
        return PLAIN[c["op"]](state)
    from pocketllm_amd import hip_kernel as ops

    cu_steps = None if c.get("even") else state.get("cu_steps")
    if c["op"] == "tree":
        return ops.paged_attention_tree_forward(state["q"], *state["cache"], state["table"], state["lengths"], state["parents"], cu_steps=cu_steps)
    if c["op"] == "sample":
        return ops.sample_tokens_forward(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state["top_k"], top_p=state["top_p"], min_p=state["min_p"])
    if c["op"] == "accept":
        return ops.draft_tree_accept_forward(state["parents"], state["drafted"], state["sampled"], state["lengths"], cu_steps=cu_steps, most=c["nodes"])
    if c["op"] == "compact":
        steps = c["nodes"] if c["even"] else state["cu_steps"]
        ops.paged_cache_compact_forward(state["layers"], state["table"], state["lengths"], state["kept"], state["counts"], steps)
        return [t for layer in state["layers"] for t in layer]
    made = ops.paged_cache_fork_forward(state["layers"], state["table"], state["uses"], state["sources"], state["kept"], state["reserve"])
    return [*made] + [t for layer in state["layers"] for t in layer]


# ---- what a pass cannot do without ------------------------------------------------------------------------------------

def work(case: dict) -> dict:
    op = case["op"]
    if op == "sample":
        values = case["rows"] * case["vocab"]
        return {"bytes": float(values * (4 if case["dtype"] == "f32" else 2) + 28 * case["rows"]), "flops": 4.0 * values}
    if op == "fork":
        held, sources, kept, reserve = _fork_plan(case)
        page = case["page"]
        taken, copies = set(), 0
        for r, (src, n) in enumerate(zip(sources, kept)):
            if src < 0 or n % page == 0:
                continue
            whole = any(o == src and m // page > n // page for o, m in zip(sources, kept))
            copies += whole or (src, n // page) in taken
            taken.add((src, n // page))
        _, width, pool = _fork_layout(case)
        copied = copies * case["layers"] * case["kv_heads"] * 2 * (2 * page * case["dim"] + 8)
        return {"bytes": float(copied + 4 * sum(held) + 4 * case["rows"] * (width + 4) + 8 * pool), "flops": float(sum(held) + case["rows"] * width)}
    nodes, pasts, parents = _trees(case)
    total = sum(nodes)
    if op == "accept":
        return {"bytes": float(20 * total + case["seqs"] * (4 * case["nodes"] + 20)), "flops": float(total)}
    dim, kv_heads = case["dim"], case["kv_heads"]
    if op == "compact":
        rng = random.Random(0)
        moved = sum(len(_path(rng, n)) for n in nodes)
        return {"bytes": float(case["layers"] * kv_heads * moved * 4 * dim + 4 * case["seqs"] * (case["nodes"] + 3)), "flops": float(case["layers"] * kv_heads * moved * 2 * dim)}
    heads, visible = case["heads"], 0
    for n, past, tree in zip(nodes, pasts, parents):
        depth = []
        for p in tree:
            depth.append(1 if p < 0 else depth[p] + 1)
        visible += n * past + sum(depth)
    return {"bytes": float(2 * (sum(pasts) + total) * kv_heads * dim + 4 * total * heads * dim + 4 * total), "flops": 4.0 * dim * heads * visible}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------

def _e4m3(v: torch.Tensor) -> torch.Tensor:
    """float64 to the nearest E4M3 value, ties to even: steps of 2 ** (e - 3) in [2 ** e, 2 ** (e + 1)), 2 ** -9 below 2 ** -6."""
    _, e = torch.frexp(v.abs().clamp_min(2.0 ** -6))
    step = torch.ldexp(torch.ones_like(v), e - 4)
    return torch.round(v / step) * step


def _exact_tree(s: dict) -> torch.Tensor:
    c = s["case"]
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    q = s["q"].double().view(-1, heads, dim)
    out = torch.empty_like(q)
    for seq, (n, past, tree) in enumerate(zip(s["nodes"], s["pasts"], s["parents_host"])):
        seen = np.zeros((n, past + n), dtype=bool)
        seen[:, :past] = True
        for i in range(n):
            node = i
            while node >= 0:
                seen[i, past + node] = True
                node = tree[node]
        seen = torch.from_numpy(seen).to(DEV)
        keys, values = _held(s, seq, past + n, torch.float64)
        at = s["cu_host"][seq]
        for head in range(heads):
            k, v = keys[head // (heads // kv_heads)].t().contiguous(), values[head // (heads // kv_heads)]
            score = (q[at:at + n, head] @ k / math.sqrt(dim)).masked_fill(~seen, -math.inf)
            out[at:at + n, head] = torch.softmax(score, -1) @ v
    return out.view(s["q"].shape)


def _exact_sample(s: dict) -> torch.Tensor:
    logits, uniform = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy()
    rows, vocab = logits.shape
    of = lambda v: v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(rows, np.float32(v), dtype=np.float64)
    temperature, top_k, top_p, min_p = (of(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    tokens = []
    for r in range(rows):
        x = logits[r]
        allowed = np.flatnonzero(x > -np.inf)
        if allowed.size == 0 or temperature[r] == 0:
            tokens.append(int(np.argmax(x)) if allowed.size else -1)
            continue
        weight = np.exp((x[allowed] - x[allowed].max()) / temperature[r])
        order = np.argsort(-x[allowed], kind="stable")
        if top_k[r] > 0:
            order = order[:int(top_k[r])]
        if top_p[r] < 1:
            sums = np.cumsum(weight[order])
            order = order[:int(np.searchsorted(sums, top_p[r] * sums[-1], side="left")) + 1]
        order = np.sort(order[weight[order] >= min_p[r]])
        sums = np.cumsum(weight[order])
        tokens.append(int(allowed[order[min(int(np.searchsorted(sums, uniform[r] * sums[-1], side="right")), order.size - 1)]]))
    return torch.tensor(tokens, device=DEV)


def _exact_accept(s: dict):
    drafted, sampled, most = s["drafted"].tolist(), s["sampled"].tolist(), s["case"]["nodes"]
    kept, counts, tokens, lengths = [], [], [], []
    for seq, tree in enumerate(s["parents_host"]):
        at, path = s["cu_host"][seq], [0]
        while True:
            follow = [i for i, p in enumerate(tree) if p == path[-1] and drafted[at + i] == sampled[at + path[-1]]]
            if not follow:
                break
            path.append(follow[0])
        kept.append(path + [-1] * (most - len(path)))
        counts.append(len(path))
        tokens.append(sampled[at + path[-1]])
        lengths.append(s["pasts"][seq] + len(path))
    return _ints(kept), _ints(counts), torch.tensor(tokens, device=DEV), _ints(lengths)


def _exact_compact(s: dict):
    page, table = s["case"]["page"], s["table"].tolist()
    out = []
    for keys, values, key_scales, value_scales in s["layers"]:
        done = []
        for pages, scales in ((keys.double(), key_scales.double()), (values.double().transpose(2, 3).contiguous(), value_scales.double())):
            pages_new, scales_new = pages.clone(), scales.clone()
            for seq, path in enumerate(s["paths"]):
                past = s["pasts"][seq]
                for first in range(0, len(path), 1):
                    if first and (past + first) % page:
                        continue                                              # (one pass over the path for every page that it ends in)
                    to = table[seq][(past + first) // page]
                    here = [(past + j, past + path[j]) for j in range(first, len(path)) if (past + j) // page == (past + first) // page]
                    held = here[0][0] % page
                    from_pages = [table[seq][src // page] for _, src in here]
                    scale = scales[torch.tensor(from_pages + [to] * (held > 0), device=DEV)].max(0).values
                    if held:
                        pages_new[to, :, :held] = _e4m3(pages[to, :, :held] * (scales[to] / scale)[:, None, None])
                    for (dst, src), which in zip(here, from_pages):
                        pages_new[to, :, dst % page] = _e4m3(pages[which, :, src % page] * (scales[which] / scale)[:, None])
                    scales_new[to] = scale
            done.append((pages_new, scales_new))
        out += [done[0][0], done[1][0].transpose(2, 3).contiguous(), done[0][1], done[1][1]]
    return out


def _exact_fork(s: dict):
    page, table, uses = s["case"]["page"], s["table"].tolist(), s["uses"].tolist()
    _, sources, kept, reserve = s["plan"]
    width = len(table[0])
    for row in table:
        for p in row:
            if p >= 0:
                uses[p] -= 1
    rows = []
    for src, n in zip(sources, kept):
        row = table[src][:n // page] if src >= 0 else []
        for p in row:
            uses[p] += 1
        rows.append(row)
    copies, taken, unfinished = [], set(), []
    for r, (src, n) in enumerate(zip(sources, kept)):
        unfinished.append(None)
        if src >= 0 and n % page:
            p = table[src][n // page]
            if uses[p] == 0 and p not in taken:
                rows[r].append(p)
            else:
                unfinished[r] = p
            taken.add(p)
    for r, (src, n) in enumerate(zip(sources, kept)):
        if src >= 0 and n % page and unfinished[r] is None:
            uses[rows[r][-1]] += 1
    free, missing = [p for p, n in enumerate(uses) if n <= 0], []
    free.reverse()
    for r, row in enumerate(rows):
        missing.append(0)
        while len(row) < -(-max(reserve[r], kept[r]) // page):
            if free:
                p = free.pop()
                uses[p] = 1
                if unfinished[r] is not None:
                    copies.append((unfinished[r], p))
            else:
                p = -1
                missing[-1] += 1
            unfinished[r] = None
            row.append(p)
        row += [-1] * (width - len(row))
    out = [_ints(rows), _ints([max(n, 0) for n in uses]), _ints(missing)]
    for layer in s["layers"]:
        for t in layer:
            new = t.float()
            for src, dst in copies:
                new[dst] = t[src].float()
            out.append(new)
    return out


EXACT = {"tree": _exact_tree, "sample": _exact_sample, "accept": _exact_accept, "compact": _exact_compact, "fork": _exact_fork}


def exact(case: dict, seed: int):
    return EXACT[case["op"]](prepare(case, seed))
