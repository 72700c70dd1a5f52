"""Serving by drafted trees from step to step, as a server runs it: the nodes' keys and values appended with the phases of their depths, tree attention, logits, a sampled token
at every node, the accepted path, its keys and values moved, the sequences of the next step forked with room for its trees.  Every operator is held to its plain form on
what the ones before it gave; then whole steps from a captured graph."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as P, tree_oracle as T
from paged_cases import DEV, Cache, close
from pocketllm_amd import hip_kernel as K

pytestmark = pytest.mark.gpu
HEADS, KV_HEADS, DIM, ROPE, LAYERS, VOCAB = 4, 2, 64, 32, 2, 500
WIDTH, KV_WIDTH = HEADS * DIM, KV_HEADS * DIM


def ints(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


class Model:
    """Per layer one projection to queries, keys and values; the attention's outputs added up; tokens by the embedding's own rows."""

    def __init__(self, dtype, positions, page):
        g = torch.Generator().manual_seed(0)
        self.embedding = (torch.randn(VOCAB, WIDTH, generator=g) * 0.5).to(dtype).to(DEV)
        self.qkv = [(torch.randn(WIDTH, WIDTH + 2 * KV_WIDTH, generator=g) / 16).to(dtype).to(DEV) for _ in range(LAYERS)]
        self.tables = P.rotary_rows(positions, DIM, ROPE)
        self.cos, self.sin = (torch.from_numpy(t).to(DEV) for t in self.tables)

    def __call__(self, tokens, positions, parents, caches, table, lengths, cu, note=None):
        x = self.embedding[tokens]
        for w, cache in zip(self.qkv, caches):
            q, k, v = (x @ w).split([WIDTH, KV_WIDTH, KV_WIDTH], dim=-1)
            before = [t.clone() for t in cache] if note is not None else None
            turned = K.paged_kv_append_forward(q, k, v, *cache, table, lengths, cu_steps=cu, cos_table=self.cos, sin_table=self.sin, rope_dim=ROPE, positions=positions)
            mixed = K.paged_attention_tree_forward(turned, *cache, table, lengths, parents, cu_steps=cu)
            if note is not None:
                note.append((before, q, k, v, turned, mixed))
            x = x + mixed
        return (x.float() @ self.embedding.float().t()) * 0.5


def host(cache):
    return [t.view(torch.uint8).cpu().numpy() for t in cache[:2]] + [t.cpu().numpy() for t in cache[2:]]


def random_tree(rng, n):
    parents = [-1] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]
    depths = [0] * n
    for i in range(1, n):
        depths[i] = depths[parents[i]] + 1
    return parents, depths


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 64])
def test_steps_of_a_server(page, dtype):
    width = 512 // page
    model, rng = Model(dtype, 600, page), np.random.default_rng(page)
    pool = 3 * width
    shape = [Cache([page] * pool, KV_HEADS, DIM, page, seed=i) for i in range(LAYERS)]
    caches = [list(c.device()[:4]) for c in shape]
    pool = caches[0][0].size(0)
    # three sequences with a past of their own: pages of random content
    held = np.array([130, 17, 64])
    table = torch.full((3, width), -1, dtype=torch.int32, device=DEV)
    uses = torch.zeros(pool, dtype=torch.int32, device=DEV)
    free = [p for p in shape[0].table.reshape(-1).tolist() if 0 <= p < pool]
    at = 0
    for s, n in enumerate(held):
        for p in range(-(-n // page)):
            table[s, p] = free[at]
            uses[free[at]] = 1
            at += 1
    for c in caches:                                                          # numbers everywhere: the layers' unused pages are not the same
        for t in c[:2]:
            t.view(torch.uint8).copy_(torch.where((t.view(torch.uint8) & 0x7f) == 0x7f, 0, t.view(torch.uint8)))
        for t in c[2:]:
            t.copy_(torch.where(t.isnan(), torch.full_like(t, 0.125), t))
    last = rng.integers(0, VOCAB, 3)
    for step in range(5):
        # the next step's rows: sequences branch, end and go on
        sources = [np.arange(len(held)), np.array([0, 1, 2, 0]), np.array([3, 1, 0]), np.array([0, 0, 2]), np.array([2, 1, 0])][step]
        nodes = rng.integers(1, 20, len(sources))
        kept_tokens, last = held[sources], last[sources]
        before = [host(c) for c in caches], table.cpu().numpy(), uses.cpu().numpy()
        table, uses, missing = K.paged_cache_fork_forward([tuple(c) for c in caches], table, uses, ints(sources), ints(kept_tokens), ints(kept_tokens + nodes))
        torch.cuda.synchronize()
        want_table, want_uses, want_missing, copies = T.fork(before[1], before[2], sources, kept_tokens, kept_tokens + nodes, page)
        assert np.array_equal(table.cpu().numpy(), want_table) and np.array_equal(uses.cpu().numpy(), want_uses) and not want_missing.any() and not missing.any()
        for arrays, c in zip(before[0], caches):
            for src, dst in copies:
                for a in arrays:
                    a[dst] = a[src]
            assert all(np.array_equal(a, b) for a, b in zip(arrays, host(c)))
        # trees of drafted tokens
        trees = [random_tree(rng, n) for n in nodes]
        cu = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
        parents, depths = np.array(sum((t[0] for t in trees), []), dtype=np.int32), np.array(sum((t[1] for t in trees), []), dtype=np.int32)
        drafted = rng.integers(0, VOCAB, cu[-1])
        drafted[cu[:-1]] = last
        lengths = kept_tokens + nodes
        positions = np.repeat(kept_tokens, nodes).astype(np.int32) + depths
        note = []
        args = torch.from_numpy(drafted).to(DEV), ints(positions), ints(parents)
        logits = model(*args, caches, table, ints(lengths), ints(cu), note)
        uniform = torch.rand(int(cu[-1]), generator=torch.Generator().manual_seed(step)).to(DEV)
        sampled = K.sample_tokens_forward(logits, uniform, temperature=0.7, top_k=20, top_p=0.95)
        # the drafts are what was sampled, now and then, so that paths are longer than a node
        for i in range(int(cu[-1])):
            s = int(np.searchsorted(cu, i, side="right")) - 1
            if parents[i] >= 0 and rng.random() < 0.7:
                drafted[i] = int(sampled[int(cu[s]) + parents[i]])
        kept, counts, tokens, news = K.draft_tree_accept_forward(ints(parents), torch.from_numpy(drafted).to(DEV), sampled, ints(lengths), cu_steps=ints(cu), most=12)
        torch.cuda.synchronize()
        host_table, turns = table.cpu().numpy(), [t[positions] for t in model.tables]
        for layer, (old, q, k, v, turned, mixed) in enumerate(note):
            old = host(old)
            keys = P.turn(k.double().cpu().numpy().reshape(-1, KV_HEADS, DIM), *turns, ROPE)
            want = P.append(keys, v.double().cpu().numpy().reshape(-1, KV_HEADS, DIM), *old, host_table, lengths, cu)
            now = host(caches[layer])
            for s, n in enumerate(lengths):
                for p in range(int(n)):
                    which, slot = host_table[s, p // page], p % page
                    assert np.array_equal(P.e4m3_decode(now[0][which, :, slot]), want[0][which, :, slot]) and np.array_equal(P.e4m3_decode(now[1][which, :, :, slot]), want[1][which, :, :, slot])
            got = turned.cpu()
            close(mixed, *T.tree_attention(got.double().numpy().reshape(-1, HEADS, DIM), *now, host_table, lengths, parents, cu, DIM ** -0.5), dtype)
        x, u = logits.double().cpu().numpy(), uniform.double().cpu().numpy()
        for i, token in enumerate(sampled.tolist()):
            want, near = T.sample(x[i], u[i], float(np.float32(0.7)), 20, float(np.float32(0.95)))
            assert near <= 1 or token == want
        want = T.accept(parents, drafted, sampled.cpu().numpy(), lengths, cu, 12)
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip((kept, counts, tokens, news), want))
        old = [host(c) for c in caches]
        K.paged_cache_compact_forward([tuple(c) for c in caches], table, ints(lengths), kept, counts, ints(cu))
        torch.cuda.synchronize()
        for arrays, c in zip(old, caches):
            want = T.compact(*arrays, host_table, lengths, kept.cpu().numpy(), counts.cpu().numpy(), nodes)
            now = host(c)
            assert np.array_equal(P.e4m3_decode(now[0]), want[0], equal_nan=True) and np.array_equal(P.e4m3_decode(now[1]), want[1], equal_nan=True)
            assert np.array_equal(now[2], want[2]) and np.array_equal(now[3], want[3])
        held, last = news.cpu().numpy().astype(np.int64), tokens.cpu().numpy()
        assert (counts.cpu().numpy() > 0).all()


def test_a_captured_step_moves_on_by_itself():
    """One graph of a whole step with trees of one shape: what it accepts is the next replay's past.  Every replay against the same step eagerly, on a copy."""
    page, width, n, dtype = 16, 16, 9, torch.bfloat16
    model, rng = Model(dtype, 400, page), np.random.default_rng(3)
    parents, depths = random_tree(rng, n)
    shape = [Cache([200, 230], KV_HEADS, DIM, page, seed=i, width=width) for i in range(LAYERS)]
    caches = [list(c.device()[:4]) for c in shape]
    table, held = shape[0].device()[4], ints([60, 21])
    drafted, uniform = torch.zeros(2 * n, dtype=torch.int64, device=DEV), torch.zeros(2 * n, device=DEV)
    steps, tree = ints(depths * 2), ints(parents * 2)

    def step(caches, held):
        lengths = held + n
        positions = held.repeat_interleave(n, output_size=2 * n) + steps
        logits = model(drafted, positions, tree, caches, table, lengths, None)
        sampled = K.sample_tokens_forward(logits, uniform, temperature=0.9, top_p=0.9)
        kept, counts, tokens, news = K.draft_tree_accept_forward(tree, drafted, sampled, lengths)
        K.paged_cache_compact_forward([tuple(c) for c in caches], table, lengths, kept, counts, n)
        held.copy_(news)
        return sampled, kept, counts, tokens, news

    copies = lambda: ([[t.clone() for t in c] for c in caches], held.clone())
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*copies())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    other, other_held = copies()
    with torch.cuda.graph(graph):
        out = step(caches, held)
    g = torch.Generator().manual_seed(5)
    for _ in range(4):
        drafted.copy_(torch.randint(0, 3, (2 * n,), generator=g))
        uniform.copy_(torch.rand(2 * n, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        want = step(other, other_held)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and torch.equal(held, other_held)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for c, o in zip(caches, other) for a, b in zip(c, o))
