"""Drafted steps as a serving program runs them: the tree's positions, keys and queries rotated as they are written,
attention of the tree, the accepted path kept, over several steps and layers, contiguous and paged. After every step the
cache is, bit for bit, the one that writing the accepted tokens one by one gives; attention is checked against the 64-bit
oracle."""

import math

import numpy as np
import pytest
import torch

from myinfer_amd import attention, kernels
from myinfer_amd.cache import QuantizedKVCache, keep_rows
from myinfer_amd.paged import PagedRadixKVCache
from oracle import attention as OA
from oracle import quantize as OQ
from oracle import tree as OT
from tests.helpers import NP_DTYPE, assert_close, seeded_normal, triple_to_np
from tests.test_gpu_read_keep import bits_of
from tests.test_gpu_tree import make_parents

pytestmark = pytest.mark.gpu
DEV = "cuda"


def longest_path(parents):
    """The deepest node and its ancestors, from the root down."""
    d = OT.depths(parents)
    return OT.path(parents, int(np.argmax(d)))[::-1]


def values(tr, dtype, bits):
    return OQ.dequantize(*triple_to_np(tr), NP_DTYPE[dtype], 64, bits)


@pytest.mark.parametrize("dtype,bits,L,Hq", [(torch.bfloat16, 8, 12, 16), (torch.float16, 4, 40, 32)])
def test_steps_over_contiguous_caches(dtype, bits, L, Hq):
    print(f"draft steps {dtype} bits={bits} L={L}", flush=True)
    layers, Hkv, D, first = 2, 4, 128, 250
    r = kernels.RopeAxes(D, base=1e6)
    drafted = [QuantizedKVCache(64, bits) for _ in range(layers)]
    single = [QuantizedKVCache(64, bits) for _ in range(layers)]
    prompt = torch.arange(first, dtype=torch.int32, device=DEV)[None]
    for i in range(layers):
        k, v = (seeded_normal((1, Hkv, first, D), 10 * i + j, dtype, DEV) for j in range(2))
        drafted[i].update_and_fetch(k, v, rope=r, positions=prompt)
        single[i].update_and_fetch(k, v, rope=r, positions=prompt)
    start = first
    for step in range(3):
        parents = make_parents("random", 1, L, 50 + step)
        tree = kernels.DraftTree(torch.tensor(parents, dtype=torch.int32, device=DEV), starts=start)
        path = longest_path(parents[0])
        for i in range(layers):
            k, v = (seeded_normal((1, Hkv, L, D), 100 * step + 10 * i + j, dtype, DEV) for j in range(2))
            q = seeded_normal((1, Hq, L, D), 100 * step + 10 * i + 2, dtype, DEV)
            keys, vals = drafted[i].update_and_fetch(k, v, rope=r, positions=tree.positions, queries=q)
            out = attention.scaled_dot_product_attention(q, keys, vals, drafted[i], 1 / math.sqrt(D), tree)
            S = start + L
            vis = OT.visible(parents[0], S, S)[None, None]
            ref = OA.exact_attention(q.cpu().double().numpy(), values(keys, dtype, bits), values(vals, dtype, bits),
                                     1 / math.sqrt(D), vis=vis)
            assert_close(out, ref, f"step {step} layer {i}")
            for d, node in enumerate(path):  # one token at a time
                p = torch.tensor([[start + d]], dtype=torch.int32, device=DEV)
                single[i].update_and_fetch(k[:, :, node: node + 1], v[:, :, node: node + 1], rope=r, positions=p)
        start = keep_rows(drafted, start, torch.tensor(path, dtype=torch.int32, device=DEV))
        for a, b in zip(drafted, single):
            assert a.offset == b.offset == start
            for x, y in zip(a.fetch()[0] + a.fetch()[1], b.fetch()[0] + b.fetch()[1]):
                assert torch.equal(bits_of(x), bits_of(y))


def test_steps_over_pages():
    """Three sequences of unequal lengths and trees over a shared pool."""
    B, layers, Hq, Hkv, D, L, dtype, bits = 3, 2, 16, 4, 128, 10, torch.float16, 8
    r = kernels.RopeAxes(D, base=1e6)
    drafted, single = (PagedRadixKVCache(layers, Hkv, D, max_blocks=16, bits=bits, dtype=dtype) for _ in range(2))
    tables = torch.randperm(15, generator=torch.Generator().manual_seed(3))[:15].view(3, 5).to(torch.int32).to(DEV)
    lens = torch.tensor([60, 5, 130], dtype=torch.int32)
    n = int(lens.max())
    pos = torch.arange(n, dtype=torch.int32, device=DEV)[None]
    for layer in range(layers):
        k, v = (seeded_normal((B, Hkv, n, D), 10 * layer + j, dtype, DEV) for j in range(2))
        for p in (drafted, single):
            p.append(layer, k, v, tables, rope=r, positions=pos)
    for step in range(3):
        parents = make_parents("random", B, L, 70 + step)
        for b in range(B):  # unequal trees: the last nodes of some are absent
            for l in range(L - 2 * b, L):
                parents[b][l] = -2
        starts = lens.to(DEV)
        tree = kernels.DraftTree(torch.tensor(parents, dtype=torch.int32, device=DEV), starts=starts)
        paths = [longest_path(p) for p in parents]
        for layer in range(layers):
            k, v = (seeded_normal((B, Hkv, L, D), 100 * step + 10 * layer + j, dtype, DEV) for j in range(2))
            q = seeded_normal((B, Hq, L, D), 100 * step + 10 * layer + 2, dtype, DEV)
            drafted.append(layer, k, v, tables, starts=starts, rope=r, positions=tree.positions, queries=q)
            out = drafted.attention(layer, q, tables, starts + L, 1 / math.sqrt(D), tree=tree)
            for b in range(B):
                S = int(lens[b]) + L
                kt, vt = drafted.gather(layer, tables[b].tolist(), S)
                ref = OA.exact_attention(q[b: b + 1].cpu().double().numpy(), values(kt, dtype, bits), values(vt, dtype, bits),
                                         1 / math.sqrt(D), vis=OT.visible(parents[b], S, S)[None, None])
                assert_close(out[b: b + 1], ref, f"step {step} layer {layer} sequence {b}")
                for d, node in enumerate(paths[b]):
                    at = int(lens[b]) + d
                    single.append(layer, k[b: b + 1, :, node: node + 1], v[b: b + 1, :, node: node + 1], tables[b: b + 1],
                                  row_offset=at, rope=r, positions=torch.tensor([[at]], dtype=torch.int32, device=DEV))
        M = max(len(p) for p in paths)
        rows = torch.tensor([p + [-1] * (M - len(p)) for p in paths], dtype=torch.int32, device=DEV)
        drafted.keep_rows(tables, rows, starts, L)
        lens = lens + torch.tensor([len(p) for p in paths], dtype=torch.int32)
        seq = lens.to(DEV)
        for layer in range(layers):
            a, b = (p.dequantized(layer, tables, seq, max_len=int(lens.max())) for p in (drafted, single))
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
            for s in range(B):
                for x, y in zip(*(p.gather(layer, tables[s].tolist(), int(lens[s])) for p in (drafted, single))):
                    assert all(torch.equal(bits_of(i), bits_of(j)) for i, j in zip(x, y))


@pytest.mark.parametrize("L,S", [(6, 300), (24, 1900)])
def test_captured_steps_over_pages(L, S):
    """A drafted step captured into a graph (the tree, the append with its queries, attention, the kept rows, reading back),
    two of them over their own pools, replayed with new inputs in place, by turns and at once: the eager step's results
    and pools, bit for bit."""
    print(f"captured draft steps L={L} S={S}", flush=True)
    B, Hq, Hkv, D, dtype = 4, 64, 8, 128, torch.bfloat16
    r = kernels.RopeAxes(D, base=1e6)
    width = -(-(S + L) // 64)
    tables = torch.randperm(B * width, generator=torch.Generator().manual_seed(5)).view(B, width).to(torch.int32).to(DEV)
    pools = [PagedRadixKVCache(1, Hkv, D, max_blocks=B * width, dtype=dtype) for _ in range(4)]  # graphs', eager ones
    k, v = (seeded_normal((B, Hkv, S, D), j, dtype, DEV) for j in range(2))
    pos = torch.arange(S, dtype=torch.int32, device=DEV)[None]
    for p in pools:
        p.append(0, k, v, tables, rope=r, positions=pos)

    def inputs(seed):
        g = torch.Generator().manual_seed(seed)
        parents = torch.tensor(make_parents("gaps", B, L, seed), dtype=torch.int32)
        rows = torch.stack([torch.randperm(L, generator=g)[:4].sort()[0] for _ in range(B)]).to(torch.int32)
        starts = torch.randint(1, S + 1, (B,), generator=g, dtype=torch.int32)
        new = [seeded_normal(shape, seed + j, dtype, DEV) for j, shape in
               enumerate([(B, Hkv, L, D), (B, Hkv, L, D), (B, Hq, L, D)])]
        return [parents.to(DEV), rows.to(DEV), starts.to(DEV), *new]

    def step(pool, tree, rows, starts, k, v, q):
        tree.refresh()
        pool.append(0, k, v, tables, starts=starts, rope=r, positions=tree.positions, queries=q)
        out = pool.attention(0, q, tables, starts + L, 1 / math.sqrt(D), max_len=S + L, tree=tree)
        pool.keep_rows(tables, rows, starts, L)
        return [out, q, *pool.dequantized(0, tables, starts + 4, max_len=S + L)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, held = [], []
    for i in range(2):
        x = inputs(600 + i)
        with torch.cuda.stream(side):
            tree = kernels.DraftTree(x[0], starts=x[2])
            step(pools[i], tree, x[1], x[2], *x[3:])  # loads the code
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step(pools[i], tree, x[1], x[2], *x[3:])
        graphs.append(g)
        held.append((x, out, tree))
    torch.cuda.synchronize()
    for i in range(2):  # the eager pools as the graphs' are
        for a, b in zip((*pools[i].k_cache(0), *pools[i].v_cache(0)), (*pools[2 + i].k_cache(0), *pools[2 + i].v_cache(0))):
            bits_of(b).copy_(bits_of(a))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        fresh = [inputs(700 + 10 * rep + i) for i in range(2)]
        for i in range(2):
            for a, b in zip(held[i][0], fresh[i]):
                a.copy_(b)
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i] if rep % 2 else torch.cuda.current_stream()):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            x = fresh[i]
            want = step(pools[2 + i], kernels.DraftTree(x[0], starts=x[2]), x[1], x[2], *x[3:])
            torch.cuda.synchronize()
            assert torch.equal(held[i][1][0], want[0]) and torch.equal(held[i][0][5], want[1]), f"replay {rep}, graph {i}"
            for a, b in zip(held[i][1][2:], want[2:]):
                for s in range(B):
                    n = int(x[2][s]) + 4
                    assert torch.equal(a[s, :, :n], b[s, :, :n])
            for a, b in zip((*pools[i].k_cache(0), *pools[i].v_cache(0)), (*pools[2 + i].k_cache(0), *pools[2 + i].v_cache(0))):
                assert torch.equal(bits_of(a), bits_of(b)), f"replay {rep}, pool {i}"
