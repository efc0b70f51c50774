"""Reading a quantized cache back, and keeping accepted rows.

Tolerance of a value read back: code * scale is exact in fp32, the FMA rounds once to fp32 (2^-24) and the result once to
T (eps/2; 2^-25 where fp16 is subnormal). Kept rows are equal bit for bit."""

import numpy as np
import pytest
import torch

from myinfer_amd import kernels
from myinfer_amd.cache import KVCache, QuantizedKVCache, keep_rows
from myinfer_amd.paged import PAGE_ROWS, PagedRadixKVCache
from oracle import quantize as OQ
from tests.helpers import NP_DTYPE, seeded_normal, triple_to_np
from tests.test_gpu_decode import make_cache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bits_of(x):
    return x.contiguous().view({4: torch.int32, 2: torch.int16}[x.element_size()])


def check_values(got, tr, G, bits, what):
    ref = OQ.dequantize(*triple_to_np(tr), NP_DTYPE[got.dtype], G, bits)
    half = torch.finfo(got.dtype).eps / 2
    bound = np.abs(ref) * (half + 2.0 ** -24 * (1 + half)) + 2.0 ** -25
    err = np.abs(got.cpu().double().numpy() - ref)
    assert (err <= bound).all(), f"{what}: {(err - bound).max()}"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,S,D,G,bits", [
    (1, 1, 1, 64, 64, 8), (2, 3, 37, 128, 64, 8), (1, 8, 1000, 128, 32, 4), (2, 2, 65, 96, 32, 2), (1, 4, 9, 256, 128, 4),
    (1, 2, 130, 32, 32, 8), (1, 8, 40000, 128, 64, 8), (3, 5, 4001, 192, 64, 4),
])
def test_read_back(B, H, S, D, G, bits, dtype):
    print(f"dequantize B={B} H={H} S={S} D={D} G={G} bits={bits} {dtype}", flush=True)
    kt, vt = make_cache(B, H, S, D, bits, dtype, 5, cap=S + 3, group=G)
    k, v = kernels.dequantize_rows(kt, vt, group_size=G, bits=bits)
    if S <= 5000:
        check_values(k, kt, G, bits, "k")
    check_values(v[:, :, -100:], tuple(x[:, :, -100:] for x in vt), G, bits, "v")
    assert torch.equal(kernels.dequantize_rows(vt, group_size=G, bits=bits)[0], v)
    # into views of a wider buffer, nothing beside them
    wide = torch.full((B, S, H, D + 8), 7.0, dtype=dtype, device=DEV)
    out = wide[..., :D].transpose(1, 2)
    kernels.dequantize_rows(kt, group_size=G, bits=bits, out=(out,))
    assert torch.equal(out, k) and bool((wide[..., D:] == 7.0).all())
    flat = kernels.dequantize(*(x[0, 0] for x in kt), group_size=G, bits=bits)
    assert torch.equal(flat, k[0, 0])


def test_large_and_special_groups():
    """Groups of one value, zeros, the largest values of the type; a group with an infinity stores no finite scale, and
    the quantizer gives a NaN element code 0."""
    x = seeded_normal((1, 1, 6, 64), 6, torch.bfloat16, DEV)
    x[0, 0, 0] = 0.0
    x[0, 0, 1] = 3.0
    x[0, 0, 2] *= 1e30
    x[0, 0, 3, 5] = float("inf")
    x[0, 0, 4, 5] = float("nan")
    tr = kernels.quantize(x)
    got = kernels.dequantize(*tr)
    assert bool((got[0, 0, 0] == 0).all()) and bool((got[0, 0, 1] == 3.0).all())
    fine = [0, 1, 2, 4, 5]
    check_values(got[:, :, fine], tuple(t[:, :, fine] if t.dtype != torch.uint32 else
                                        t.view(torch.int32)[:, :, fine].view(torch.uint32) for t in tr), 64, 8, "special")
    assert not torch.isfinite(got[0, 0, 3]).any()


def test_cache_reads_back():
    c = QuantizedKVCache(64, 8)
    k, v = (seeded_normal((2, 3, 300, 128), 7 + i, torch.float16, DEV) for i in range(2))
    c.update_and_fetch(k, v)
    kt, vt = c.fetch()
    rk, rv = c.dequantized()
    check_values(rk, kt, 64, 8, "k")
    check_values(rv, vt, 64, 8, "v")
    part = c.dequantized(250, 299)
    assert torch.equal(part[0], rk[:, :, 250:299]) and torch.equal(part[1], rv[:, :, 250:299])
    assert c.dequantized(5, 5)[0].shape[2] == 0
    plain = c.to_unquantized()
    assert plain.offset == 300 and torch.equal(plain.state[0], rk) and torch.equal(plain.state[1], rv)
    again = plain.to_quantized(64, 8)  # the values of a group quantize to its own codes, or a step beside
    assert torch.allclose(again.dequantized()[0].float(), rk.float(), atol=float(rk.float().abs().max()) / 100)
    with pytest.raises(ValueError, match="cache of 300"):
        c.dequantized(0, 301)
    r = QuantizedKVCache(64, 8)
    r.restore(c.keys, c.values, 300)
    r.update_and_fetch(k[:, :, :5], v[:, :, :5])
    assert torch.equal(bits_of(r.fetch()[0][0][:, :, :300]), bits_of(kt[0])) and r.offset == 305


def _paged(lens, H, D, bits, G, dtype, seed):
    from tests.test_gpu_paged import build

    return build(len(lens), H, lens, D, bits, dtype, seed, group=G)


@pytest.mark.parametrize("H,D,G,bits,dtype", [(2, 128, 64, 8, torch.float16), (3, 64, 32, 4, torch.bfloat16), (1, 256, 128, 8, torch.bfloat16)])
def test_paged_read_back(H, D, G, bits, dtype):
    _, tables, kp, vp, kc, vc = _paged([3, 64, 65, 500], H, D, bits, G, dtype, 9)
    lens = [1, 64, 65, 500]  # the first sequence's last rows are not read
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = kernels.dequantize_rows(kc, vc, group_size=G, bits=bits)
    out = tuple(torch.full((4, H, 500, D), 7.0, dtype=dtype, device=DEV) for _ in range(2))
    kernels.paged_dequantize(kp, vp, tables, seq, group_size=G, bits=bits, out=out)
    fresh = kernels.paged_dequantize(kp, vp, tables, seq, group_size=G, bits=bits, max_len=70)
    for i in range(2):
        for b, n in enumerate(lens):
            assert torch.equal(out[i][b, :, :n], want[i][b, :, :n])
            assert bool((out[i][b, :, n:] == 7.0).all())  # rows behind a sequence stay
            assert torch.equal(fresh[i][b, :, :min(n, 70)], want[i][b, :, :min(n, 70)])
            assert not fresh[i][b, :, n:].any()
    bad = tables.clone()
    bad[:, 1:] = -1  # clamped: read from some page of the pool, never outside it
    kernels.paged_dequantize(kp, vp, bad, seq, group_size=G, bits=bits, max_len=500)
    torch.cuda.synchronize()


def reference_move(x, start, rows, n):
    """x [B, H, cap, W] with row start + i = the old row start + rows[b][i] where rows[b][i] is in [i, n)."""
    y = x.clone()
    for b, list_b in enumerate(rows):
        for i, r in enumerate(list_b):
            if i <= r < n:
                y[b, :, start + i] = x[b, :, start + r]
    return y


@pytest.mark.parametrize("rows,n", [
    ([[0]], 1), ([[3]], 5), ([[0, 1, 2]], 4), ([[1, 3, 4, 9], [0, 2, -1, -1]], 10),
    ([[5, 5, 5], [2, 1, 2]], 6),                  # the same row again; a list that is not ascending
    ([[2, 0, 3], [9, 1, 10 ** 6]], 4),            # entries below their index or past the drafted rows: left as they are
    ([list(range(1, 41))], 41),                   # longer than one round of loads
    ([list(range(3, 300, 2))[:140]], 300),
])
@pytest.mark.parametrize("G,bits,D,dtype", [(64, 8, 128, torch.float16), (32, 4, 96, torch.bfloat16), (64, 2, 64, torch.float16)])
def test_keep_rows(rows, n, G, bits, D, dtype):
    print(f"keep_rows {len(rows[0])} of {n} bits={bits} D={D}", flush=True)
    B, H, start = len(rows), 3, 70
    caches, before = [], []
    for i in range(3):
        c = QuantizedKVCache(G, bits)
        c.update_and_fetch(*(seeded_normal((B, H, start + n, D), 20 + 2 * i + j, dtype, DEV) for j in range(2)))
        caches.append(c)
    plain = KVCache()
    plain.update_and_fetch(*(seeded_normal((B, H, start + n, D), 30 + j, dtype, DEV) for j in range(2)))
    caches.append(plain)
    arrays = [t for c in caches for t in ((*c.keys, *c.values) if c is not plain else (c.keys, c.values))]
    before = [bits_of(t).clone() for t in arrays]
    idx = torch.tensor(rows, dtype=torch.int32, device=DEV)
    assert keep_rows(caches, start, idx) == start + len(rows[0])
    for t, old in zip(arrays, before):
        assert torch.equal(bits_of(t), reference_move(old, start, rows, n))
    assert all(c.offset == start + len(rows[0]) for c in caches)


def test_keep_rows_of_many_layers_and_shared_list():
    """More arrays than a launch takes, of more shapes than it holds, one list for the batch."""
    B, start, n, rows = 2, 10, 9, [1, 4, 8]
    arrays = []
    for i in range(40):
        c = QuantizedKVCache(64, 8 if i % 3 else 4)
        c.reserve(seeded_normal((B, 2, 1, 128), i, torch.float16, DEV), 256 * (1 + i % 5))
        c.update_and_fetch(*(seeded_normal((B, 2, start + n, 128), 40 + 2 * i + j, torch.float16, DEV) for j in range(2)))
        arrays += [*c.keys, *c.values]
    before = [bits_of(t).clone() for t in arrays]
    kernels.keep_rows(arrays, torch.tensor(rows, dtype=torch.int32, device=DEV), start, n)
    for t, old in zip(arrays, before):
        assert torch.equal(bits_of(t), reference_move(old, start, [rows] * B, n))


def test_shared_memory_refused():
    """The same cache twice, and tensors broadcast along an axis, before anything moves; an axis of one row may have any stride."""
    c = QuantizedKVCache(64, 8)
    c.update_and_fetch(*(seeded_normal((2, 2, 20, 128), 70 + j, torch.float16, DEV) for j in range(2)))
    before = [bits_of(t).clone() for t in (*c.keys, *c.values)]
    rows = torch.tensor([1, 3], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="twice"):
        keep_rows([c, c], 10, rows)
    assert c.offset == 20 and all(torch.equal(bits_of(t), b) for t, b in zip((*c.keys, *c.values), before))
    one = seeded_normal((1, 1, 3, 128), 72, torch.float16, DEV)
    for shape in ((2, 1, 3, 128), (1, 2, 3, 128)):
        with pytest.raises(ValueError, match="broadcast"):
            kernels.keep_rows([one.expand(shape)], rows[:1], 0, 3)
        with pytest.raises(ValueError, match="share"):
            kernels.rope_axes(one.expand(shape), kernels.RopeAxes(128), torch.zeros(1, 3, dtype=torch.int32, device=DEV))
        with pytest.raises(ValueError, match="share"):
            k = tuple(x[: shape[0], : shape[1], :3] for x in c.keys)
            kernels.dequantize_rows(k, k, group_size=64, bits=8, out=(one.expand(shape), one.expand(shape)))
    pos = torch.arange(3, dtype=torch.int32, device=DEV).view(1, 3)
    strange = one.clone().as_strided((1, 1, 3, 128), (0, 0, 128, 1))
    assert torch.equal(kernels.rope_axes(strange, kernels.RopeAxes(128), pos),
                       kernels.rope_axes(one.clone(), kernels.RopeAxes(128), pos))


def test_nothing_kept():
    c = QuantizedKVCache(64, 8)
    c.update_and_fetch(*(seeded_normal((1, 2, 20, 128), 50 + j, torch.float16, DEV) for j in range(2)))
    before = [bits_of(t).clone() for t in (*c.keys, *c.values)]
    assert keep_rows([c], 12, torch.zeros(1, 0, dtype=torch.int32, device=DEV)) == 12 and c.offset == 12
    assert all(torch.equal(bits_of(t), b) for t, b in zip((*c.keys, *c.values), before))


def test_paged_keep_rows():
    """Drafted rows that cross a page's end, shuffled pages, unequal starts and counts; pages outside the pool are left."""
    H, D, dtype = 2, 128, torch.float16
    pool = PagedRadixKVCache(3, H, D, max_blocks=12, bits=8, group_size=64, dtype=dtype)
    tables = torch.tensor([[7, 2], [0, 11], [5, -1]], dtype=torch.int32, device=DEV)
    for layer in range(3):
        pool.append(layer, *(seeded_normal((3, H, 100, D), 60 + 2 * layer + j, dtype, DEV) for j in range(2)), tables)
    starts, rows, n = [61, 3, 60], [[1, 3, 4, 9], [0, 2, -1, -1], [2, 3, 5, 6]], 12
    layers = [pool.k_cache(l) for l in range(3)] + [pool.v_cache(l) for l in range(3)]
    before = [[bits_of(x).clone() for x in tr] for tr in layers]
    pool.keep_rows(tables, torch.tensor(rows, dtype=torch.int32, device=DEV), torch.tensor(starts, dtype=torch.int32, device=DEV), n)
    for tr, old in zip(layers, before):
        for x, o in zip(tr, old):
            want = o.clone()
            for b in range(3):
                for i, r in enumerate(rows[b]):
                    src, dst = starts[b] + r, starts[b] + i
                    pages = [int(tables[b, s // PAGE_ROWS]) for s in (src, dst)]
                    if i <= r < n and min(pages) >= 0:
                        want[pages[1], :, dst % PAGE_ROWS] = o[pages[0], :, src % PAGE_ROWS]
            assert torch.equal(bits_of(x), want)


def test_graph_replays():
    """A read and a move captured into a graph, replayed with new rows and new contents in between."""
    c = QuantizedKVCache(64, 8)
    c.reserve(seeded_normal((1, 4, 1, 128), 0, torch.float16, DEV), 256)
    c.update_and_fetch(*(seeded_normal((1, 4, 200, 128), 70 + j, torch.float16, DEV) for j in range(2)))
    rows = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV)
    out = tuple(torch.empty(1, 4, 50, 128, dtype=torch.float16, device=DEV) for _ in range(2))
    view = lambda tr: tuple(x[:, :, 150:200] for x in tr)  # noqa: E731
    arrays = [*c.keys, *c.values]

    def step():
        kernels.keep_rows(arrays, rows, 150, 50)
        kernels.dequantize_rows(view(c.keys), view(c.values), out=out)

    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step()
    for rep in range(4):
        c.trim(50)
        c.update_and_fetch(*(seeded_normal((1, 4, 50, 128), 80 + 2 * rep + j, torch.float16, DEV) for j in range(2)))
        new = [rep, rep + 2, 10 + rep, 40 + rep]
        rows.copy_(torch.tensor(new, dtype=torch.int32))
        want = [reference_move(x, 0, [new], 50) for x in c.dequantized(150, 200)]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    c = QuantizedKVCache(64, 8)
    c.update_and_fetch(*(seeded_normal((2, 2, 20, 128), 90 + j, torch.float16, DEV) for j in range(2)))
    ok = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    for rows, start in [(ok.long(), 10), (ok.cpu(), 10), (ok[:1], 10), (ok, 18), (ok, 21), (ok.T, 10), (ok[:, ::2], 10)]:
        with pytest.raises(ValueError):
            keep_rows([c], start, rows)
        assert c.offset == 20
    with pytest.raises(ValueError, match="same shapes"):
        kernels.dequantize_rows(c.keys, tuple(x[:, :, :5] for x in c.values))
    with pytest.raises(ValueError, match="one width"):
        kernels.dequantize_rows(c.keys, bits=4)
    with pytest.raises(ValueError, match="out must be"):
        kernels.dequantize_rows(c.keys, out=(torch.empty(2, 2, 20, 128, device=DEV),))
    with pytest.raises(ValueError, match="leading dims"):
        kernels.dequantize(c.keys[0], c.keys[1][:, :, :5], c.keys[2][:, :, :5])
    pool = PagedRadixKVCache(1, 2, 128, max_blocks=4)
    t = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="seq_lens"):
        pool.dequantized(0, t, torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="cannot hold"):
        pool.dequantized(0, t, torch.zeros(2, dtype=torch.int32, device=DEV), max_len=129)
    with pytest.raises(ValueError, match="starts"):
        pool.keep_rows(t, ok, torch.zeros(3, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="kept"):
        pool.keep_rows(t, ok, torch.zeros(2, dtype=torch.int32, device=DEV), n=2)


def test_restored_twice_raises_the_registered_word():
    """Appends after a second restore of the same buffers raise the range word that is registered then, by either
    append, and the earlier one is left alone."""
    from myinfer_amd.cache import QuantizedKVCache

    r = kernels.RopeAxes(128)
    k, v = (seeded_normal((1, 2, 8, 128), 700 + i, torch.bfloat16, DEV) for i in range(2))
    pos = torch.zeros(1, 8, dtype=torch.int32, device=DEV)
    for rope in (None, r):
        kw = {} if rope is None else dict(rope=rope, positions=pos)
        c = QuantizedKVCache(64, 8)
        c.reserve(k, 256)
        keys, values = c.keys, c.values
        c.restore(keys, values, 0)
        c.update_and_fetch(k, v, **kw)
        first = c.range_exp
        c.restore(keys, values, 8)
        c.update_and_fetch(k, v * 1e6, **kw)
        assert c.range_exponents()[1] > 0 and first.tolist() == [0, 0]


def test_rows_that_do_not_exist():
    """Reading and keeping of nothing: no rows, no arrays' change."""
    from myinfer_amd.cache import QuantizedKVCache, keep_rows as keep_cached

    c = QuantizedKVCache(64, 8)
    k = seeded_normal((1, 2, 8, 128), 710, torch.float16, DEV)
    c.update_and_fetch(k, k)
    before = [bits_of(x).clone() for x in (*c.keys, *c.values)]
    assert c.dequantized(3, 3)[0].shape == (1, 2, 0, 128)
    assert keep_cached([c], 8, torch.zeros(1, 0, dtype=torch.int32, device=DEV)) == 8
    assert keep_cached([c], 5, torch.zeros(0, dtype=torch.int32, device=DEV)) == 5
    assert all(torch.equal(bits_of(x), y) for x, y in zip((*c.keys, *c.values), before))
    plain = QuantizedKVCache(64, 8).to_unquantized()
    assert plain.keys is None and plain.offset == 0
