"""The native host path of a drafted step (csrc/host): it serves the calls that programs make, with the results of the
Python path bit for bit, hands back what it does not take, and does not try a failed launch again."""

import copy
import ctypes
import pickle
import subprocess

import pytest
import torch

from myinfer_amd import _lib, attention, kernels
from myinfer_amd.cache import KVCache, QuantizedKVCache, keep_rows
from tests.helpers import seeded_normal
from tests.test_gpu_decode import make_cache
from tests.test_gpu_read_keep import bits_of
from tests.test_gpu_tree import make_parents

pytestmark = pytest.mark.gpu
DEV = "cuda"


def python_path(monkeypatch, fn):
    """fn() with the native path switched off."""
    with monkeypatch.context() as m:
        m.setattr(kernels, "_native", lambda t: (None, 0))
        return fn()


def native_path(monkeypatch, fn):
    """fn() where only the native path can serve it: the library's calls from Python raise."""
    def refuse(*a, **k):
        raise AssertionError("the Python path was taken")

    with monkeypatch.context() as m:
        m.setattr(_lib, "rows", refuse)
        m.setattr(_lib, "qtensor", refuse)
        return fn()


def same(a, b):
    return all(torch.equal(bits_of(x), bits_of(y)) for x, y in zip(a, b))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("form", ["quant", "lens", "dense", "paged", "shared"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_tree_attention(monkeypatch, form, dtype):
    B, Hq, Hkv, D, L, S = 2, 32, 4, 128, 20, 900
    parents = ints(make_parents("gaps", B, L, 500))
    if form == "shared":
        parents = parents[0].contiguous()
    q = seeded_normal((B, Hq, L, D), 501, dtype, DEV)
    if form == "dense":
        k, v = (seeded_normal((B, Hkv, S, D), 502 + i, dtype, DEV) for i in range(2))
    elif form == "paged":
        from tests.test_gpu_paged import build

        _, table, k, v, _, _ = build(B, Hkv, [S, 300], D, 8, dtype, 503)
        lens = ints([S, 300])
    else:
        c = QuantizedKVCache(64, 8)
        k, v = c.update_and_fetch(*(seeded_normal((B, Hkv, S, D), 504 + i, dtype, DEV) for i in range(2)))

    def run():
        tree = kernels.DraftTree(parents)
        if form == "paged":
            return kernels.paged_attention(q, k, v, table, lens, 0.09, tree=tree, max_len=S)
        if form == "dense":
            return attention.fast_scaled_dot_product_attention(q, k, v, 0.09, tree, window=400)
        return attention.blocked_quantized_sdpa(q, k, v, 0.09, tree, window=0, seq_lens=ints([S, 70]) if form == "lens" else None)

    out = native_path(monkeypatch, run)
    assert torch.equal(out, python_path(monkeypatch, run))
    assert out.shape == q.shape and torch.isfinite(out).all()


@pytest.mark.parametrize("starts", [None, 7, "tensor"])
@pytest.mark.parametrize("shared", [False, True])
def test_draft_tree(monkeypatch, starts, shared):
    B, L = (1, 33) if shared else (3, 33)
    parents = ints(make_parents("gaps", B, L, 510))
    parents = parents[0] if shared else parents
    st = ints([5, 70000, 0][:B]) if starts == "tensor" else starts
    t = native_path(monkeypatch, lambda: kernels.DraftTree(parents, starts=st))
    u = python_path(monkeypatch, lambda: kernels.DraftTree(parents, starts=st))
    assert torch.equal(t.bits, u.bits) and torch.equal(t.depths, u.depths)
    assert (t.positions is None) == (starts is None) == (u.positions is None)
    if starts is not None:
        assert torch.equal(t.positions, u.positions) and t.positions.shape == (1, B, L)
    parents.fill_(-1)  # refreshed over the same buffers
    t.refresh()
    assert not t.depths.any() and t.bits.data_ptr() == t.desc.bits


@pytest.mark.parametrize("queries", [True, False])
@pytest.mark.parametrize("pos3d", [True, False])
def test_append_read_and_rotate(monkeypatch, queries, pos3d):
    B, Hq, Hkv, D, L, dtype = 2, 8, 4, 128, 19, torch.bfloat16
    r = kernels.RopeAxes(D, (16, 24, 24), base=1e6)
    assert pickle.loads(pickle.dumps(r)) == copy.deepcopy(r) == r
    k, v = (seeded_normal((B, Hkv, L, D), 520 + i, dtype, DEV) for i in range(2))
    pos = torch.randint(0, 5000, (3, B, L) if pos3d else (3, L), dtype=torch.int32, device=DEV)

    def step():
        c = QuantizedKVCache(64, 8)
        c.update_and_fetch(*(seeded_normal((B, Hkv, 30, D), 522 + i, dtype, DEV) for i in range(2)))
        q = seeded_normal((B, Hq, L, D), 524, dtype, DEV)
        c.update_and_fetch(k, v, rope=r, positions=pos, queries=q if queries else None)
        return [*c.fetch()[0], *c.fetch()[1], q, *c.dequantized(), *c.dequantized(29, 48), *c.dequantized(48, 48)]

    def rotated():
        return [kernels.rope_axes(seeded_normal((B, Hq, L, D), 525, dtype, DEV), r, pos)]

    assert same(step(), python_path(monkeypatch, step))
    assert same(native_path(monkeypatch, rotated), python_path(monkeypatch, rotated))


def test_reads_back(monkeypatch):
    from tests.test_gpu_paged import build

    _, table, kp, vp, kc, vc = build(2, 3, [200, 131], 128, 4, torch.float16, 530)
    lens = ints([200, 131])
    rows = native_path(monkeypatch, lambda: kernels.dequantize_rows(kc, vc, bits=4))
    assert same(rows, python_path(monkeypatch, lambda: kernels.dequantize_rows(kc, vc, bits=4)))

    def paged():
        out = tuple(torch.full((2, 3, 210, 128), 7.0, dtype=torch.float16, device=DEV) for _ in range(2))
        got = kernels.paged_dequantize(kp, vp, table, lens, bits=4, out=out)
        assert got[0] is out[0] and got[1] is out[1]
        return got

    got = native_path(monkeypatch, paged)
    assert same(got, python_path(monkeypatch, paged)) and bool((got[0][1, :, 131:] == 7).all())
    assert torch.equal(got[0][0, :, :200], rows[0][0])


@pytest.mark.parametrize("mixed", [False, True])
def test_keeps_rows(monkeypatch, mixed):
    def caches():
        out = []
        for i in range(4):
            c = KVCache() if mixed and i % 2 else QuantizedKVCache(64, 8)
            c.update_and_fetch(*(seeded_normal((2, 4, 40, 128), 540 + 2 * i + j, torch.float16, DEV) for j in range(2)))
            out.append(c)
        return out

    rows = ints([[0, 3, 7], [1, 2, -1]])

    def run():
        cs = caches()
        assert keep_rows(cs, 30, rows) == 33 and all(c.offset == 33 for c in cs)
        return [x for c in cs for a in (c.keys, c.values) for x in ((a,) if torch.is_tensor(a) else a)]

    with monkeypatch.context() as m:
        m.setattr(kernels, "keep_rows", None)  # the native path alone
        got = run()
    assert same(got, python_path(monkeypatch, run))


def test_keeps_paged_rows(monkeypatch):
    from tests.test_gpu_paged import build

    _, table, kp, vp, _, _ = build(2, 4, [200, 131], 128, 8, torch.float16, 550)

    def run():  # over a copy of the pools, whose unused rows hold anything
        k, v = (tuple(x.clone() for x in tr) for tr in (kp, vp))
        kernels.paged_keep_rows([(k, v)], table, ints([[1, 5], [2, -1]]), starts=ints([120, 63]))
        return [x.nan_to_num(3) if x.is_floating_point() else x for x in (*k, *v)]

    with monkeypatch.context() as m:
        m.setattr(kernels, "_row_arrays", None)
        got = run()
    assert same(got, python_path(monkeypatch, run))
    assert not same(got, [x.nan_to_num(3) if x.is_floating_point() else x for x in (*kp, *vp)])


@pytest.mark.parametrize("starts,queries", [(True, True), (False, False)])
def test_paged_append(monkeypatch, starts, queries):
    from myinfer_amd.paged import PagedRadixKVCache

    r = kernels.RopeAxes(128, (16, 24, 24))
    k, v = (seeded_normal((2, 4, 9, 128), 580 + i, torch.bfloat16, DEV) for i in range(2))
    pos = torch.randint(0, 500, (3, 2, 9), dtype=torch.int32, device=DEV)

    def run():
        pool = PagedRadixKVCache(1, 4, 128, 8, dtype=torch.bfloat16, device=DEV)
        q = seeded_normal((2, 8, 9, 128), 582, torch.bfloat16, DEV)
        table = ints([[5, 2], [0, 7]])
        for step in range(2):  # (the second with the first's descriptors)
            pool.append(0, k, v, table, starts=ints([60, 3 + step]) if starts else None, row_offset=0 if starts else 50, rope=r,
                        positions=pos, queries=q if queries else None)
        return [*pool.k_cache(0), *pool.v_cache(0), q]

    got = run()
    assert same(got, python_path(monkeypatch, run))
    assert got[1].any()


def test_tables_that_are_views():
    """The first pages of a wider table, whose other entries name pages of somebody else: rows past the view are
    dropped, and nothing there is read."""
    from tests.test_gpu_paged import build

    lens = [130, 70]
    _, table, kp, vp, kc, vc = build(2, 4, lens, 128, 8, torch.float16, 555, npages=20)
    P = table.shape[1]
    mine = set(int(x) for b, n in enumerate(lens) for x in table[b, : -(-n // 64)])
    others = [p for p in range(20) if p not in mine]
    wide = torch.full((2, 8), others[0], dtype=torch.int32, device=DEV)
    wide[:, 2:2 + P] = table
    view = wide[:, 2:2 + P]
    before = [bits_of(x)[others] for x in (*kp, *vp)]
    q = seeded_normal((2, 8, 5, 128), 556, torch.float16, DEV)
    tree = kernels.DraftTree(ints(make_parents("random", 2, 5, 557)))
    seq = ints(lens)
    assert torch.equal(kernels.paged_attention(q, kp, vp, view, seq, 0.1, tree=tree),
                       kernels.paged_attention(q, kp, vp, table, seq, 0.1, tree=tree))
    with pytest.raises(ValueError):  # rows that the view does not hold
        kernels.paged_attention(q, kp, vp, view, seq, 0.1, tree=tree, max_len=64 * P + 1)
    with pytest.raises(ValueError):
        kernels.paged_dequantize(kp, vp, view, seq, max_len=64 * P + 1)
    got = kernels.paged_dequantize(kp, vp, view, seq)
    assert got[0].shape[2] == 64 * P and torch.equal(got[0][0, :, :130], kernels.dequantize_rows(kc, vc)[0][0, :, :130])
    # rows kept, and appended, across the end of the view
    kernels.paged_keep_rows([(kp, vp)], view, ints([1, 3]), starts=ints([64 * P - 1, 64 * P - 2]))
    k = seeded_normal((2, 4, 4, 128), 558, torch.float16, DEV)
    kernels.paged_rope_axes_append(k, kp, k, vp, view, kernels.RopeAxes(128), ints([[0, 1, 2, 3]]), starts=ints([64 * P - 2] * 2))
    assert all(torch.equal(bits_of(x)[others], y) for x, y in zip((*kp, *vp), before))


def test_handed_back():
    """Forms that the Python path serves (or refuses) as before: rows to copy, triples as lists, K alone."""
    kt, vt = make_cache(1, 4, 300, 128, 8, torch.float16, 560)
    q = seeded_normal((1, 8, 6, 128), 561, torch.float16, DEV)
    tree = kernels.DraftTree(ints(make_parents("random", 1, 6, 562)))
    ref = kernels.attention(q, kt, vt, 0.1, tree=tree)
    odd = torch.empty(1, 8, 6, 132, dtype=torch.float16, device=DEV)[..., :128].copy_(q)
    assert torch.equal(kernels.attention(odd, kt, vt, 0.1, tree=tree), ref)
    assert torch.equal(attention.blocked_quantized_sdpa(q, list(kt), list(vt), 0.1, tree), ref)
    out = torch.empty_like(q)
    assert kernels.attention(q, kt, vt, 0.1, tree=tree, out=out) is out and torch.equal(out, ref)
    k1 = kernels.dequantize_rows(kt)
    assert len(k1) == 1 and torch.equal(k1[0], kernels.dequantize_rows(kt, vt)[0])
    for bad, err in [(dict(window=3), NotImplementedError), (dict(bits=4), ValueError), (dict(causal=True), ValueError),
                     (dict(seq_lens=torch.tensor([300], device=DEV)), ValueError), (dict(group_size=32), ValueError)]:
        with pytest.raises(err):
            kernels.attention(q, kt, vt, 0.1, tree=tree, **bad)
    for scale in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            kernels.attention(q, kt, vt, scale, tree=tree)
    for pos in (ints([[0] * 6]).long(), ints([[0] * 5]), ints([[0] * 6] * 2)):
        with pytest.raises(ValueError, match="positions"):
            kernels.rope_axes(q, kernels.RopeAxes(128), pos)
    with pytest.raises(ValueError):
        kernels.dequantize_rows(kt, vt, out=(torch.empty_like(q), torch.empty_like(q)))


STUBS = """
extern "C" {
int calls = 0;
int fails() { ++calls; return -4; }
unsigned long bytes() { return 256; }
int no() { return 0; }
}
"""


def test_a_failed_launch_raises_once(tmp_path):
    (tmp_path / "stubs.cpp").write_text(STUBS)
    subprocess.run(["g++", "-shared", "-fPIC", str(tmp_path / "stubs.cpp"), "-o", str(tmp_path / "stubs.so")], check=True)
    lib = ctypes.CDLL(str(tmp_path / "stubs.so"))
    at = {n: ctypes.cast(getattr(lib, n), ctypes.c_void_p).value for n in ("fails", "bytes", "no")}
    kt, vt = make_cache(1, 4, 300, 128, 8, torch.float16, 570)
    q = seeded_normal((1, 8, 6, 128), 571, torch.float16, DEV)
    parents = ints(make_parents("random", 1, 6, 572))
    tree = kernels.DraftTree(parents)
    kernels.attention(q, kt, vt, 0.1, tree=tree)
    pos = ints([[0] * 6])
    calls = [lambda: kernels.DraftTree(parents), lambda: kernels.attention(q, kt, vt, 0.1, tree=tree),
             lambda: kernels.rope_axes(q, kernels.RopeAxes(128), pos), lambda: kernels.dequantize_rows(kt, vt),
             lambda: kernels.keep_rows([*kt, *vt], ints([1, 2]), 10, 5)]
    try:
        _lib.host().bind_draft(*(at["bytes"] if "workspace" in n else at["no"] if "reads" in n else at["fails"]
                                 for n in _lib.DRAFT_SYMBOLS))
        for i, call in enumerate(calls):
            with pytest.raises(RuntimeError, match="status -4"):
                call()
            assert ctypes.c_int.in_dll(lib, "calls").value == i + 1
    finally:
        _lib._host = None
        _lib.host()
    assert torch.isfinite(kernels.attention(q, kt, vt, 0.1, tree=tree)).all()
