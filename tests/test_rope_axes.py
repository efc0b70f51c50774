"""Rotation over several axes, reading caches back and keeping rows without a GPU: the oracle's pair assignment and
rotation, and what the entry points refuse (no call here reaches a launch)."""

import ctypes
import math

import numpy as np
import pytest
import torch

from myinfer_amd import _lib, cache, kernels
from oracle import axes as OX
from oracle import rope as OR
from tests.test_abi import _fake_q, _fake_rows
from tests.test_abi_attention import _expect
from tests.test_tree import _pool

byref = ctypes.byref


def test_oracle_pair_axes():
    assert OX.pair_axes((2, 3, 1), False) == [0, 0, 1, 1, 1, 2]
    assert OX.pair_axes((2, 3, 1), True) == [0, 1, 2, 0, 1, 1]
    assert OX.pair_axes((4,), True) == [0, 0, 0, 0]
    _, f = OX.freqs(8, (2, 2), 16.0, False, False)
    assert np.allclose(f, [1, 1 / 2, 1 / 4, 1 / 8])
    _, f = OX.freqs(8, (2, 2), 16.0, True, True)  # every axis: 1, 1/4
    assert np.allclose(f, [1, 1, 1 / 4, 1 / 4])


@pytest.mark.parametrize("traditional", [False, True])
def test_oracle_rotation(traditional):
    # unit vectors: pair i = (cos t, sin t)
    D, sections = 16, (3, 5)
    pos = np.array([[[2, 7]], [[5, 11]]])
    ax, f = OX.freqs(D, sections, 100.0, False, False)
    for i in range(8):
        d0, d1 = (2 * i, 2 * i + 1) if traditional else (i, i + 8)
        x = np.zeros((1, 1, 2, D))
        x[..., d0] = 1.0
        y, size = OX.rotate(x, pos, D, sections, traditional, base=100.0)
        for l in range(2):
            t = pos[ax[i], 0, l] * f[i]
            assert math.isclose(y[0, 0, l, d0], math.cos(t), abs_tol=1e-14)
            assert math.isclose(y[0, 0, l, d1], math.sin(t), abs_tol=1e-14)
        assert (size[..., d0] == 1).all() and (size[..., d1] == 1).all()
    # equal positions on every axis are one axis; one axis is the one-axis restatement at small angles
    x = np.random.default_rng(0).standard_normal((2, 3, 5, D))
    p = np.arange(5)[None, None].repeat(2, 1)
    one, _ = OX.rotate(x, p, D, (8,), traditional)
    two, _ = OX.rotate(x, p.repeat(2, 0), D, sections, traditional)
    assert np.array_equal(one, two)
    assert np.abs(one - OR.rope_f32(x, D, traditional, 10000.0, 1.0, 0)).max() < 1e-5
    # rotations compose, and dims past the rotated ones stay
    twice, _ = OX.rotate(OX.rotate(x, p, 8, (4,), traditional)[0], 2 * p, 8, (4,), traditional)
    assert np.allclose(twice, OX.rotate(x, 3 * p, 8, (4,), traditional)[0], atol=1e-12)
    assert np.array_equal(twice[..., 8:], x[..., 8:])


def test_rope_axes_descriptor():
    r = kernels.RopeAxes(128, (16, 24, 24))
    d = r.params()
    assert (d.dims, d.axes, list(d.sections)) == (128, 3, [16, 24, 24, 0]) and r.axes == 3
    assert kernels.RopeAxes(64).sections == (32,)
    assert kernels.RopeAxes(64) == kernels.RopeAxes(64, (32,))
    for bad in ((16, 24), (0, 64), (16, 24, 24, 0), (32, -8, 40), (8, 8, 8, 8, 32)):
        with pytest.raises(ValueError, match="sections|axes"):
            kernels.RopeAxes(128, bad)


def _axes(**kw):
    a = dict(dims=128, traditional=0, axes=2, sections=(40, 24, 0, 0), interleaved=0, restart=0, base=1e4, scale=1.0,
             positions=1 << 28, sa=8, sb=4, sl=1)
    a.update(kw)
    return _lib.Axes(a["dims"], a["traditional"], a["axes"], (ctypes.c_int * 4)(*a["sections"]), a["interleaved"],
                     a["restart"], a["base"], a["scale"], a["positions"], a["sa"], a["sb"], a["sl"])


BAD_AXES = [
    (_axes(dims=24), _lib.ERR_UNSUPPORTED, "dims"),
    (_axes(dims=256, sections=(64, 64, 0, 0)), _lib.ERR_UNSUPPORTED, "dims"),
    (_axes(dims=0), _lib.ERR_UNSUPPORTED, "dims"),
    (_axes(axes=0), _lib.ERR_UNSUPPORTED, "axes"),
    (_axes(axes=5), _lib.ERR_UNSUPPORTED, "axes"),
    (_axes(sections=(64, 0, 0, 0)), _lib.ERR_INVALID, "section"),
    (_axes(sections=(40, 23, 0, 0)), _lib.ERR_INVALID, "pairs"),
    (_axes(base=0.0), _lib.ERR_INVALID, "base"),
    (_axes(base=float("inf")), _lib.ERR_INVALID, "base"),
    (_axes(scale=float("nan")), _lib.ERR_INVALID, "scale"),
    (_axes(positions=None), _lib.ERR_INVALID, "positions"),
    (_axes(positions=(1 << 28) + 2), _lib.ERR_INVALID, "4-byte"),
    (_axes(sl=-1), _lib.ERR_INVALID, "strides"),
]


@pytest.mark.parametrize("bad,code,needle", BAD_AXES)
def test_rope_axes_refuses(bad, code, needle):
    lib, r, q = _lib.lib(), _fake_rows(), _fake_q()
    _expect(lib.kvq_rope_axes(byref(r), byref(bad), 1, 1, 1, 128, 0, None), code, needle)
    _expect(lib.kvq_rope_axes_append(byref(r), byref(q), None, None, None, 0, byref(bad), 0, None, 0, None, 0, 1, 1, 1, 128, 8,
                                     64, 0, None), code, needle)


def test_rope_axes_append_refuses():
    lib, r, q, good = _lib.lib(), _fake_rows(), _fake_q(), _axes()

    def call(k=r, kd=q, v=None, vd=None, qs=None, Hq=0, rope=good, pages=0, table=None, stride=0, starts=None, row=0, B=1, H=1,
             L=1, D=128, bits=8, G=64, dtype=0):
        p = [None if x is None else byref(x) for x in (k, kd, v, vd, qs)]
        return lib.kvq_rope_axes_append(*p, Hq, None if rope is None else byref(rope), pages, table, stride, starts, row, B, H, L,
                                        D, bits, G, dtype, None)

    _expect(call(rope=None), _lib.ERR_INVALID, "rope")
    _expect(call(k=None), _lib.ERR_INVALID, "k_src")
    _expect(call(v=r), _lib.ERR_INVALID, "both")
    _expect(call(bits=3), _lib.ERR_UNSUPPORTED, "bits")
    _expect(call(G=48), _lib.ERR_UNSUPPORTED, "group_size")
    _expect(call(row=-1), _lib.ERR_INVALID, "row_offset")
    _expect(call(starts=1 << 20), _lib.ERR_INVALID, "block table")
    _expect(call(qs=_fake_rows(ptr=(1 << 20) + 2), Hq=8), _lib.ERR_INVALID, "queries")
    _expect(call(qs=r, Hq=-1), _lib.ERR_INVALID, "Hq")
    _expect(call(kd=_pool(), pages=0, table=1 << 20, stride=4), _lib.ERR_INVALID, "num_pages")
    _expect(call(kd=_pool(), pages=4, table=1 << 20, stride=1, row=64), _lib.ERR_INVALID, "cannot hold")
    assert call(L=0) == _lib.OK and call(B=0, qs=r, Hq=4) == _lib.OK and _lib.last_error() == ""


def test_dequantize_refuses():
    lib, r, q = _lib.lib(), _fake_rows(), _fake_q()

    def call(k=q, kd=r, v=None, vd=None, row=0, B=1, H=1, L=1, D=128, bits=8, G=64, dtype=0):
        p = [None if x is None else byref(x) for x in (k, kd, v, vd)]
        return lib.kvq_dequantize(*p, row, B, H, L, D, bits, G, dtype, None)

    _expect(call(k=None), _lib.ERR_INVALID, "k_src")
    _expect(call(kd=None), _lib.ERR_INVALID, "k_dst")
    _expect(call(v=q), _lib.ERR_INVALID, "both")
    _expect(call(bits=5), _lib.ERR_UNSUPPORTED, "bits")
    _expect(call(G=16), _lib.ERR_UNSUPPORTED, "group_size")
    _expect(call(D=96), _lib.ERR_INVALID, "multiple")
    _expect(call(row=-1), _lib.ERR_INVALID, "row_offset")
    _expect(call(kd=_fake_rows(ptr=16 * 1024 + 8)), _lib.ERR_INVALID, "16-byte")
    odd = _fake_q()
    odd.codes += 4
    _expect(call(k=odd), _lib.ERR_INVALID, "8-byte")
    assert call(L=0) == _lib.OK

    def paged(k=_pool(), table=1 << 20, stride=2, lens=1 << 21, L=128, pages=4):
        return lib.kvq_paged_dequantize(byref(k), byref(r), None, None, pages, table, stride, lens, 1, 8, L, 128, 8, 64, 0, None)

    _expect(paged(table=None), _lib.ERR_INVALID, "block_table")
    _expect(paged(L=129), _lib.ERR_INVALID, "cannot hold")
    _expect(paged(lens=None), _lib.ERR_INVALID, "seq_lens")
    _expect(paged(pages=0), _lib.ERR_INVALID, "num_pages")
    assert paged(L=0) == _lib.OK


def test_keep_rows_refuses():
    lib = _lib.lib()
    good = dict(data=1 << 20, stride_b=4096, stride_h=1024, stride_l=128, row_bytes=128)

    def call(arrays=None, n_arrays=1, pages=0, table=None, stride=0, rows=1 << 22, rows_sb=4, starts=None, start=0, n=8, M=4, B=1,
             H=2, **kw):
        a = dict(good, **kw)
        arr = (_lib.RowArray * 1)(_lib.RowArray(*(a[k] for k in ("data", "stride_b", "stride_h", "stride_l", "row_bytes"))))
        return lib.kvq_keep_rows(None if arrays == "null" else arr, n_arrays, pages, table, stride, rows, rows_sb, starts, start,
                                 n, M, B, H, None)

    for kw, code, needle in [
        (dict(M=9), _lib.ERR_INVALID, "kept"),
        (dict(n=-1), _lib.ERR_INVALID, "negative"),
        (dict(B=70000), _lib.ERR_UNSUPPORTED, "65535"),
        (dict(arrays="null"), _lib.ERR_INVALID, "arrays"),
        (dict(rows=None), _lib.ERR_INVALID, "rows"),
        (dict(rows=(1 << 22) + 2), _lib.ERR_INVALID, "4-byte"),
        (dict(rows_sb=-1), _lib.ERR_INVALID, "batch stride"),
        (dict(start=-1), _lib.ERR_INVALID, "start"),
        (dict(starts=1 << 21), _lib.ERR_INVALID, "block table"),
        (dict(table=1 << 21, stride=0, pages=4), _lib.ERR_INVALID, "table_stride"),
        (dict(data=None), _lib.ERR_INVALID, "NULL"),
        (dict(data=(1 << 20) + 1), _lib.ERR_INVALID, "odd"),
        (dict(stride_l=126), _lib.ERR_INVALID, "rows of"),
        (dict(stride_l=0), _lib.ERR_INVALID, "zero stride"),
        (dict(row_bytes=127), _lib.ERR_INVALID, "odd"),
    ]:
        _expect(call(**kw), code, needle)
    assert call(M=0) == _lib.OK and call(n_arrays=0) == _lib.OK and call(H=0) == _lib.OK


def test_refuses_rows_that_share_their_memory():
    # what is written in place, or out, has an address of its own for every row: of a broadcast tensor, or an array named
    # twice, the result would depend on the order of the workgroups
    lib = _lib.lib()
    pos = 1 << 22

    def rows(**kw):
        r = _fake_rows()
        for name, x in kw.items():
            setattr(r, name, x)
        return r

    axes = kernels.RopeAxes(128).params()
    axes.positions = pos
    for name in ("stride_b", "stride_h", "stride_l"):
        x = rows(**{name: 0})
        _expect(lib.kvq_rope_axes(byref(x), byref(axes), 3, 4, 5, 128, 0, None), _lib.ERR_INVALID, "x")
        _expect(lib.kvq_rope_axes_append(byref(rows()), byref(_fake_q()), None, None, byref(x), 4, byref(axes), 0, None, 0, None,
                                         0, 3, 4, 5, 128, 8, 64, 0, None), _lib.ERR_INVALID, "queries")
        _expect(lib.kvq_dequantize(byref(_fake_q()), byref(rows()), byref(_fake_q()), byref(x), 0, 3, 4, 5, 128, 8, 64, 0, None),
                _lib.ERR_INVALID, "v_dst")
        _expect(lib.kvq_paged_dequantize(byref(_pool()), byref(x), None, None, 4, 1 << 20, 2, 1 << 21, 3, 4, 5, 128, 8, 64, 0,
                                         None), _lib.ERR_INVALID, "k_dst")

    def keep(n, data, table=None, B=2, H=2, M=4, **kw):
        a = dict(stride_b=4096, stride_h=1024, stride_l=128, row_bytes=128)
        a.update(kw)
        arr = (_lib.RowArray * n)(*(_lib.RowArray(data(i), *a.values()) for i in range(n)))
        return lib.kvq_keep_rows(arr, n, 4 if table else 0, table, 4 if table else 0, 1 << 22, 4, None, 0, 8, M, B, H, None)

    for n in (2, 6, 192, 200, 3000):  # the twin of the first array comes last
        for table in (None, 1 << 23):
            _expect(keep(n, lambda i: (1 << 24) + (i % (n - 1)) * 8192, table), _lib.ERR_INVALID, "twice")
    _expect(keep(1, lambda i: 1 << 24, stride_b=0), _lib.ERR_INVALID, "broadcast")
    _expect(keep(1, lambda i: 1 << 24, stride_h=0), _lib.ERR_INVALID, "broadcast")
    _expect(keep(1, lambda i: 1 << 24, 1 << 23, stride_b=0, B=1), _lib.ERR_INVALID, "broadcast")  # (all pages one)
    # arrays of their own are nothing to refuse
    assert keep(3000, lambda i: (1 << 24) + i * 8192, M=0) == _lib.OK


def test_python_refusals_on_the_host():
    x = torch.zeros(1, 2, 3, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        kernels.rope_axes(x, kernels.RopeAxes(64), torch.zeros(1, 1, 3, dtype=torch.int32))
    c = cache.KVCache()
    rows = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="no caches"):
        cache.keep_rows([], 0, rows)
    with pytest.raises(ValueError, match="hold rows"):
        cache.keep_rows([c], 0, rows)
    c.update_and_fetch(x, x)
    with pytest.raises(ValueError, match="cannot be kept"):
        cache.keep_rows([c], 1, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="int32 tensor"):
        cache.keep_rows([c], 1, [0])
    with pytest.raises(ValueError, match="GPU"):
        cache.keep_rows([c], 1, rows)
    r = cache.RotatingKVCache(4)
    r.update_and_fetch(x, x)
    with pytest.raises(ValueError, match="RotatingKVCache"):
        cache.keep_rows([r], 0, rows)
    q = cache.QuantizedKVCache(64, 8)
    with pytest.raises(ValueError, match="positions"):
        q.update_and_fetch(x, x, rope=kernels.RopeAxes(64))
    with pytest.raises(ValueError, match="RopeAxes"):
        q.update_and_fetch(x, x, queries=x)
    with pytest.raises(ValueError, match="cache of 0"):
        q.dequantized()
    assert q.to_unquantized().empty() and q.offset == 0


def test_restore_refuses():
    q = cache.QuantizedKVCache(64, 8)
    codes = torch.zeros(1, 2, 8, 32, dtype=torch.int32).view(torch.uint32)
    sb = torch.zeros(1, 2, 8, 2, dtype=torch.float16)
    ok = (codes, sb, sb)
    for k, v, rows in [((codes, sb), ok, 4), (ok, (codes, sb[:, :, :4], sb), 4), (ok, ok, 9), (ok, ok, -1),
                       ((codes[..., :16], sb, sb), ok, 4), (ok, (codes, sb.bfloat16(), sb.bfloat16()), 4),
                       ((codes.view(torch.int32), sb, sb), ok, 4)]:
        with pytest.raises(ValueError):
            q.restore(k, v, rows)
    assert q.empty()
    q.restore(ok, ok, 4)
    assert q.offset == 4 and q.range_exp.tolist() == [0, 0] and kernels.range_word(q.keys[0]) is not None
