"""Attention of trees of drafted tokens against the exact 64-bit oracle (oracle/tree.py's visibility), over
quantized, unquantized and paged caches: every head dim and kernel, chains, stars, random trees, absent nodes,
windows, unequal lengths, views, graphs and streams. The tolerances are those of the other attention tests
(tests/helpers.py)."""

import math

import numpy as np
import pytest
import torch

from myinfer_amd import _lib, attention, kernels
from oracle import attention as OA
from oracle import quantize as OQ
from oracle import tree as OT
from tests.helpers import NP_DTYPE, assert_close, seeded_normal, triple_to_np
from tests.test_gpu_decode import make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_parents(kind, B, L, seed):
    """[B][L] lists: a chain, a star, or random trees; "gaps" has absent nodes among them."""
    rng = np.random.default_rng(seed)
    if kind == "chain":
        return [[l - 1 for l in range(L)] for _ in range(B)]
    if kind == "star":
        return [[-1] * L for _ in range(B)]
    out = []
    for b in range(B):
        row = [int(rng.integers(-1, l)) if l else -1 for l in range(L)]
        if kind == "gaps":
            for l in rng.choice(L, size=max(1, L // 4), replace=False):
                row[int(l)] = -2 if l % 2 else L  # either side of the valid range
        out.append(row)
    return out


def tensor(parents):
    return torch.tensor(parents, dtype=torch.int32, device=DEV)


def vis(parents, lens, S, window=0):
    return np.stack([OT.visible(p, n, S, window) for p, n in zip(parents, lens)])[:, None]


def values_of(tr, dtype, G, bits):
    return OQ.dequantize(*triple_to_np(tr), NP_DTYPE[dtype], G, bits)


def exact(q, k, v, scale, parents, lens, S, window=0):
    return OA.exact_attention(q.detach().cpu().double().numpy(), k, v, scale, vis=vis(parents, lens, S, window),
                              seq_lens=lens)


def check(out, ref, parents, what):
    assert_close(out, ref, what)
    for b, p in enumerate(parents):  # absent rows are exactly 0
        gone = [l for l, d in enumerate(OT.depths(p)) if d < 0]
        assert not out[b, :, gone].any(), what


@pytest.mark.parametrize("kind", ["chain", "star", "random", "gaps"])
@pytest.mark.parametrize("L", [1, 2, 31, 32, 33, 64, 200, 1024])
def test_bits_and_depths(kind, L):
    B = 3
    parents = make_parents(kind, B, L, L)
    starts = torch.tensor([5, 0, 70000], dtype=torch.int32, device=DEV)
    t = kernels.DraftTree(tensor(parents), starts=starts)
    for b, p in enumerate(parents):
        d = OT.depths(p)
        assert t.depths[b].tolist() == d
        assert np.array_equal(t.bits[b].cpu().numpy().view(np.uint32), OT.words(p))
        assert t.positions[0, b].tolist() == [int(starts[b]) + max(x, 0) for x in d]
    one = kernels.DraftTree(tensor(parents[0]), starts=9)  # shared by a batch
    assert torch.equal(one.bits[0], t.bits[0]) and one.positions[0, 0].tolist() == [9 + max(x, 0) for x in OT.depths(parents[0])]


QUANT = [
    # (B, Hq, Hkv, D, G, bits, dtype, L, S, kind, window)
    (1, 8, 8, 128, 64, 8, torch.float16, 1, 1, "star", 0),          # the tree is the whole cache, one node
    (1, 16, 8, 128, 64, 8, torch.float16, 10, 4106, "random", 0),
    (2, 8, 2, 128, 64, 8, torch.bfloat16, 33, 33, "gaps", 0),       # no prefix
    (2, 32, 4, 128, 64, 4, torch.float16, 16, 1000, "random", 0),
    (1, 64, 8, 128, 64, 8, torch.bfloat16, 64, 2111, "gaps", 0),
    (1, 8, 1, 128, 128, 4, torch.bfloat16, 130, 777, "random", 0),
    (1, 32, 4, 128, 32, 8, torch.float16, 31, 513, "random", 0),
    (1, 16, 2, 64, 64, 8, torch.bfloat16, 65, 900, "random", 0),
    (2, 8, 8, 64, 32, 4, torch.float16, 7, 95, "gaps", 0),
    (1, 32, 2, 64, 64, 4, torch.float16, 40, 6000, "random", 0),
    (1, 8, 4, 256, 64, 8, torch.float16, 9, 700, "random", 0),
    (1, 16, 2, 256, 128, 4, torch.bfloat16, 50, 1300, "gaps", 0),
    (1, 8, 2, 256, 64, 8, torch.bfloat16, 100, 260, "random", 0),
    (1, 8, 8, 96, 32, 8, torch.float16, 12, 333, "random", 0),      # narrow rows
    (1, 32, 4, 96, 32, 4, torch.float16, 20, 901, "gaps", 0),
    (1, 4, 4, 32, 32, 8, torch.bfloat16, 5, 77, "random", 0),
    (1, 8, 4, 192, 64, 4, torch.float16, 6, 300, "random", 0),
    (1, 16, 8, 128, 64, 8, torch.float16, 10, 2000, "random", 64),  # windows
    (1, 64, 8, 128, 64, 8, torch.float16, 48, 1500, "random", 100),
    (2, 16, 2, 64, 64, 4, torch.bfloat16, 70, 1100, "gaps", 71),
    (1, 16, 2, 256, 64, 8, torch.bfloat16, 40, 900, "random", 300),
    (1, 8, 1, 128, 64, 8, torch.float16, 300, 5000, "chain", 0),
    (1, 4, 1, 128, 64, 4, torch.bfloat16, 1024, 1500, "random", 0),
]


@pytest.mark.parametrize("B,Hq,Hkv,D,G,bits,dtype,L,S,kind,window", QUANT)
def test_quantized(B, Hq, Hkv, D, G, bits, dtype, L, S, kind, window):
    print(f"tree quantized B={B} Hq={Hq} Hkv={Hkv} D={D} G={G} bits={bits} {dtype} L={L} S={S} {kind} window={window}", flush=True)
    kt, vt = make_cache(B, Hkv, S, D, bits, dtype, 40 + L, group=G)
    q = seeded_normal((B, Hq, L, D), 41 + S, dtype, DEV)
    parents = make_parents(kind, B, L, 42 + D)
    scale = 1.0 / math.sqrt(D)
    out = attention.blocked_quantized_sdpa(q, kt, vt, scale, kernels.DraftTree(tensor(parents)), G, bits, window=window)
    ref = exact(q, values_of(kt, dtype, G, bits), values_of(vt, dtype, G, bits), scale, parents, [S] * B, S, window)
    check(out, ref, parents, f"D={D} L={L}")


@pytest.mark.parametrize("B,Hq,Hkv,D,dtype,L,S,kind,window", [
    (1, 8, 8, 128, torch.float16, 1, 5, "star", 0),
    (4, 32, 8, 64, torch.float16, 31, 2047, "random", 0),
    (2, 16, 8, 128, torch.bfloat16, 3, 700, "gaps", 0),
    (1, 32, 4, 128, torch.bfloat16, 40, 1111, "gaps", 0),
    (1, 8, 2, 256, torch.float16, 17, 400, "gaps", 0),
    (1, 8, 2, 80, torch.bfloat16, 9, 130, "random", 0),
    (1, 8, 2, 160, torch.float16, 20, 300, "random", 0),
    (1, 16, 4, 128, torch.float16, 30, 900, "random", 33),
    (2, 8, 2, 64, torch.bfloat16, 6, 500, "random", 40),
    (1, 8, 2, 256, torch.bfloat16, 30, 700, "random", 200),
])
def test_unquantized(B, Hq, Hkv, D, dtype, L, S, kind, window):
    print(f"tree unquantized B={B} Hq={Hq} Hkv={Hkv} D={D} {dtype} L={L} S={S} {kind} window={window}", flush=True)
    k, v = (seeded_normal((B, Hkv, S, D), 50 + i, dtype, DEV) for i in range(2))
    q = seeded_normal((B, Hq, L, D), 52, dtype, DEV)
    parents = make_parents(kind, B, L, 53)
    scale = 1.0 / math.sqrt(D)
    out = attention.scaled_dot_product_attention(q, k, v, None, scale, kernels.DraftTree(tensor(parents))) if not window \
        else attention.fast_scaled_dot_product_attention(q, k, v, scale, kernels.DraftTree(tensor(parents)), window=window)
    ref = exact(q, k.cpu().double().numpy(), v.cpu().double().numpy(), scale, parents, [S] * B, S, window)
    check(out, ref, parents, f"D={D} L={L}")


@pytest.mark.parametrize("Hq,Hkv,D,G,bits,dtype,L,window", [
    (16, 8, 128, 64, 8, torch.float16, 6, 0),
    (32, 4, 128, 64, 4, torch.bfloat16, 37, 0),
    (8, 2, 64, 32, 8, torch.float16, 20, 0),
    (8, 2, 256, 128, 8, torch.bfloat16, 40, 0),
    (16, 2, 96, 32, 4, torch.float16, 18, 0),
    (32, 4, 128, 128, 8, torch.float16, 37, 80),
])
def test_paged_unequal_lengths(Hq, Hkv, D, G, bits, dtype, L, window):
    """Pages in a shuffled order whose unused rows hold NaN scales; one sequence is its tree alone, one tree
    ends on a page's last row and one on the next page's first."""
    from tests.test_gpu_paged import build

    print(f"tree paged Hq={Hq} Hkv={Hkv} D={D} G={G} bits={bits} {dtype} L={L} window={window}", flush=True)
    lens = [L, 640, 641, 1999]
    B = len(lens)
    _, tables, kp, vp, kc, vc = build(B, Hkv, lens, D, bits, dtype, 60, group=G)
    if dtype == torch.bfloat16:  # the pools' range words, as PagedRadixKVCache registers them
        for tr in (kp, vp):
            kernels.register_range_word(tr[0], torch.zeros(1, dtype=torch.int32, device=DEV))
    q = seeded_normal((B, Hq, L, D), 61, dtype, DEV)
    parents = make_parents("gaps", B, L, 62)
    scale = 1.0 / math.sqrt(D)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    tree = kernels.DraftTree(tensor(parents))
    out = kernels.paged_attention(q, kp, vp, tables, seq, scale, group_size=G, bits=bits, tree=tree, window=window,
                                  max_len=max(lens))
    S = max(lens)
    ref = exact(q, values_of(kc, dtype, G, bits), values_of(vc, dtype, G, bits), scale, parents, lens, S, window)
    check(out, ref, parents, f"D={D}")
    # the contiguous call over the same rows, with lengths
    out2 = kernels.attention(q, kc, vc, scale, seq_lens=seq, group_size=G, bits=bits, tree=tree, window=window)
    check(out2, ref, parents, f"contiguous D={D}")


def test_lengths_below_the_tree():
    """A length the documentation does not allow (fewer rows than nodes) reads nothing outside the cache: the nodes
    past the missing ones see the rows that exist."""
    L, D, lens = 12, 128, [5, 12]
    kt, vt = make_cache(2, 2, 40, D, 8, torch.float16, 70)
    q = seeded_normal((2, 4, L, D), 71, torch.float16, DEV)
    parents = make_parents("chain", 2, L, 0)
    out = kernels.attention(q, kt, vt, 0.1, seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                            tree=kernels.DraftTree(tensor(parents)))
    ref = exact(q, values_of(kt, torch.float16, 64, 8), values_of(vt, torch.float16, 64, 8), 0.1, parents, lens, 40)
    assert_close(out, ref, "short")


@pytest.mark.parametrize("L", [8, 48])
def test_views_strides_and_shared_tree(L):
    """Capacity-padded cache views, queries and an output that are transposed views, one tree for the batch,
    parents as a strided view."""
    B, Hq, Hkv, S, D, dtype = 2, 16, 4, 600, 128, torch.bfloat16
    kt, vt = make_cache(B, Hkv, S, D, 8, dtype, 80, cap=768)
    q = seeded_normal((B, L, Hq, D), 81, dtype, DEV).transpose(1, 2)
    out = torch.full((B, L, Hq, D), float("nan"), dtype=dtype, device=DEV).transpose(1, 2)
    p = make_parents("random", 1, L, 82)
    scale = 0.09
    res = kernels.attention(q, kt, vt, scale, out=out, tree=kernels.DraftTree(tensor(p[0])))
    assert res is out
    ref = exact(q, values_of(kt, dtype, 64, 8), values_of(vt, dtype, 64, 8), scale, p * B, [S] * B, S)
    assert_close(out, ref, "views")
    wide = torch.full((B, 2 * L), -2, dtype=torch.int32, device=DEV)
    wide[:, :L] = tensor(p * B)
    again = kernels.attention(q, kt, vt, scale, tree=kernels.DraftTree(wide[:, :L]))
    assert torch.equal(again, out)


@pytest.mark.parametrize("L,Hq,Hkv", [(6, 8, 8), (40, 32, 4)])
def test_nonfinite_queries_and_hidden_keys(L, Hq, Hkv):
    """NaN in an absent node's query and in the keys hidden from the others stays where it is hidden; a row that
    sees a NaN key is NaN."""
    D, S, dtype = 128, 300, torch.float16
    k, v = (seeded_normal((1, Hkv, S, D), 90 + i, dtype, DEV) for i in range(2))
    q = seeded_normal((1, Hq, L, D), 92, dtype, DEV)
    parents = make_parents("star", 1, L, 0)
    parents[0][2] = -2
    q[:, :, 2] = float("nan")
    k[:, :, S - L + 2] = float("nan")  # the absent node's key, which none sees
    ref = exact(q.nan_to_num(0), k.nan_to_num(0).cpu().double().numpy(), v.cpu().double().numpy(), 0.1, parents, [S], S)
    out = kernels.attention(q, k, v, 0.1, tree=kernels.DraftTree(tensor(parents)))
    check(out, ref, parents, "dense")
    k[:, :, S - 1] = float("inf")  # the last node's own key
    out = kernels.attention(q, k, v, 0.1, tree=kernels.DraftTree(tensor(parents)))
    assert_close(out[:, :, :-1], ref[:, :, :-1], "others")
    assert not torch.isfinite(out[:, :, -1]).any()


def test_large_bf16_values():
    """bf16 values beyond the fp16 range, with the cache's range words, on the kernels that serve many rows."""
    from myinfer_amd.cache import QuantizedKVCache

    L, Hq, Hkv, S, D = 48, 32, 4, 500, 128
    cache = QuantizedKVCache(64, 8)
    k, v = (seeded_normal((1, Hkv, S, D), 95 + i, torch.float32, DEV) for i in range(2))
    cache.update_and_fetch(k.bfloat16(), (v * 3e5).bfloat16())
    kt, vt = cache.fetch()
    q = seeded_normal((1, Hq, L, D), 97, torch.bfloat16, DEV)
    parents = make_parents("random", 1, L, 98)
    out = attention.scaled_dot_product_attention(q, kt, vt, cache, 0.09, kernels.DraftTree(tensor(parents)))
    ref = exact(q, values_of(kt, torch.bfloat16, 64, 8), values_of(vt, torch.bfloat16, 64, 8) / 3e5, 0.09, parents, [S], S)
    assert_close((out.float() / 3e5).bfloat16(), ref, "large values")


@pytest.mark.parametrize("B,Hq,Hkv,L,S", [(1, 16, 8, 8, 6000), (8, 32, 8, 4, 2000), (1, 64, 8, 64, 4096), (8, 32, 8, 40, 900)])
def test_graph_replays(B, Hq, Hkv, L, S):
    """Two graphs captured on one stream, each building its tree and attending, replayed by turns and at once with
    eager work between; new parents and queries are picked up in place."""
    print(f"tree graphs B={B} Hq={Hq} Hkv={Hkv} L={L} S={S}", flush=True)
    D, dtype = 128, torch.bfloat16
    kt, vt = make_cache(B, Hkv, S, D, 8, dtype, 100)
    for tr in (kt, vt):
        kernels.register_range_word(tr[0], torch.zeros(1, dtype=torch.int32, device=DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, ins, outs = [], [], []
    for i in range(2):
        q = seeded_normal((B, Hq, L, D), 101 + i, dtype, DEV)
        par = tensor(make_parents("random", B, L, 103 + i))
        with torch.cuda.stream(side):
            tree = kernels.DraftTree(par)
            kernels.attention(q, kt, vt, 0.09, tree=tree)  # loads the code
            side.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                tree.refresh()
                outs.append(kernels.attention(q, kt, vt, 0.09, tree=tree))
        graphs.append(g)
        ins.append((q, par, tree))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for i in range(2):
            ins[i][0].copy_(seeded_normal((B, Hq, L, D), 110 + 2 * rep + i, dtype, DEV))
            ins[i][1].copy_(tensor(make_parents("gaps", B, L, 120 + 2 * rep + i)))
        torch.cuda.synchronize()
        if rep % 2:
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        else:
            for i in range(2):
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            want = kernels.attention(ins[i][0], kt, vt, 0.09, tree=kernels.DraftTree(ins[i][1].clone()))
            assert torch.equal(outs[i], want), f"replay {rep}, graph {i}"


def test_prepared_call_and_streams():
    B, Hq, Hkv, L, S, D, dtype = 1, 32, 8, 12, 5000, 128, torch.float16
    kt, vt = make_cache(B, Hkv, S, D, 8, dtype, 130)
    qs = [seeded_normal((B, Hq, L, D), 131 + i, dtype, DEV) for i in range(2)]
    tree = kernels.DraftTree(tensor(make_parents("random", B, L, 133)))
    ref = [kernels.attention(q, kt, vt, 0.1, tree=tree) for q in qs]
    call = kernels.prepare_attention(qs[0], kt, vt, 0.1, tree=tree)
    assert torch.equal(call(), ref[0])
    n = _lib.lib().kvq_tree_workspace_size(B, Hq, Hkv, L, D, S, 0)
    mine = kernels.prepare_attention(qs[0], kt, vt, 0.1, tree=tree, workspace=kernels.new_workspace(n, DEV))
    qs[0].copy_(qs[1])
    assert torch.equal(call(), ref[1]) and torch.equal(mine(), ref[1])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            got.append(kernels.attention(qs[1], kt, vt, 0.1, tree=tree))
    torch.cuda.synchronize()
    assert all(torch.equal(g, ref[1]) for g in got)


def test_refusals():
    kt, vt = make_cache(2, 2, 40, 128, 8, torch.float16, 140)
    q = seeded_normal((2, 4, 6, 128), 141, torch.float16, DEV)
    tree = kernels.DraftTree(tensor(make_parents("star", 2, 6, 0)))
    with pytest.raises(ValueError, match="nodes"):
        kernels.attention(q[:, :, :5], kt, vt, 0.1, tree=tree)
    with pytest.raises(ValueError, match="batch"):
        kernels.attention(q[:1], tuple(x[:1] for x in kt), tuple(x[:1] for x in vt), 0.1, tree=tree)
    with pytest.raises(ValueError, match="causal"):
        kernels.attention(q, kt, vt, 0.1, causal=True, tree=tree)
    with pytest.raises(ValueError, match="last rows"):
        kernels.attention(q, tuple(x[:, :, :5] for x in kt), tuple(x[:, :, :5] for x in vt), 0.1, tree=tree)
    with pytest.raises(NotImplementedError, match="window"):
        kernels.attention(q, kt, vt, 0.1, window=5, tree=tree)
    with pytest.raises(ValueError, match="workspace"):
        kernels.prepare_attention(q, kt, vt, 0.1, tree=tree, workspace=torch.zeros(16, dtype=torch.uint8, device=DEV))
    for bad in (torch.zeros(2, 3, 1, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV),
                torch.zeros(2, 0, dtype=torch.int32, device=DEV), torch.zeros(2, 8, dtype=torch.int32, device=DEV)[:, ::2]):
        with pytest.raises(ValueError):
            kernels.DraftTree(bad)
    with pytest.raises(NotImplementedError, match="1024"):
        kernels.DraftTree(torch.zeros(1025, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="starts"):
        kernels.DraftTree(tensor([[-1], [-1]]), starts=torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="int32"):
        kernels.DraftTree(tensor([-1]), starts=2 ** 31)
