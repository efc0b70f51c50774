"""Trees of drafted tokens without a GPU: the oracle's visibility against hand-written trees, and what the
entry points refuse (no call here reaches a launch)."""

import ctypes

import numpy as np
import pytest
import torch

from myinfer_amd import _lib, kernels
from oracle import tree as OT
from tests.test_abi import _fake_q, _fake_rows
from tests.test_abi_attention import WS, _expect

byref = ctypes.byref


def test_oracle_hand_tree():
    #        0
    #      1   2        3 (a second root)
    #     4 5   6 (absent), 7 under the absent one
    parents = [-1, 0, 0, -1, 1, 1, -2, 6]
    assert OT.depths(parents) == [0, 1, 1, 0, 2, 2, -1, -1]
    assert [OT.path(parents, l) for l in (0, 3, 5, 7)] == [[0], [3], [5, 1, 0], None]
    v = OT.visible(parents, 10, 12)  # two keys before the tree, two rows past the sequence
    assert v.astype(int).tolist() == [
        [1, 1, 1, 0, 0, 0, 0, 0, 0, 0, 0, 0],
        [1, 1, 1, 1, 0, 0, 0, 0, 0, 0, 0, 0],
        [1, 1, 1, 0, 1, 0, 0, 0, 0, 0, 0, 0],
        [1, 1, 0, 0, 0, 1, 0, 0, 0, 0, 0, 0],
        [1, 1, 1, 1, 0, 0, 1, 0, 0, 0, 0, 0],
        [1, 1, 1, 1, 0, 0, 0, 1, 0, 0, 0, 0],
        [0] * 12,
        [0] * 12,
    ]
    assert OT.words(parents)[:, 0].tolist() == [1, 3, 5, 8, 19, 35, 0, 0]
    # a parent that does not come before its child makes the node absent
    assert OT.depths([0, -1, 5]) == [-1, 0, -1]


def test_oracle_window_and_chain():
    # a chain is a causal mask, and with a window a causal sliding window
    from oracle.attention import key_mask

    L, S = 7, 40
    chain = [-1] + list(range(L - 1))
    for window in (0, 7, 11):
        assert np.array_equal(OT.visible(chain, S, S, window), key_mask(L, S, S, True, window))
    # siblings of one depth share their window
    v = OT.visible([-1, -1, 1], 20, 20, 5)
    assert v[0].nonzero()[0].tolist() == [13, 14, 15, 16, 17]
    assert v[1].nonzero()[0].tolist() == [13, 14, 15, 16, 18]
    assert v[2].nonzero()[0].tolist() == [14, 15, 16, 18, 19]


def _tree(**kw):
    a = dict(bits=1 << 26, depths=1 << 27, bits_stride_b=0, depths_stride_b=0)
    a.update(kw)
    return _lib.Tree(a["bits"], a["depths"], a["bits_stride_b"], a["depths_stride_b"])


def _call(form="quant", **kw):
    lib = _lib.lib()
    a = dict(q=_fake_rows(), k=_fake_q(), v=_fake_q(ptr=1 << 24), seq=None, out=_fake_rows(ptr=1 << 23), B=1, Hq=8, Hkv=1,
             L=4, D=128, S=256, bits=8, group=64, dtype=0, scale=0.1, tree=_tree(), window=0, ws=WS, wsb=1 << 40, stream=None,
             pages=16, table=1 << 25, table_stride=4)
    if form == "dense":
        a.update(k=_fake_rows(ptr=1 << 21), v=_fake_rows(ptr=1 << 22))
    a.update(kw)
    tree = None if a["tree"] is None else byref(a["tree"])
    tail = (a["dtype"], a["scale"], tree, a["window"], a["ws"], a["wsb"], a["stream"])
    sizes = (a["B"], a["Hq"], a["Hkv"], a["L"], a["D"], a["S"])
    if form == "dense":
        return lib.kvq_tree_attn_dense(byref(a["q"]), byref(a["k"]), byref(a["v"]), a["seq"], byref(a["out"]), *sizes, *tail)
    if form == "paged":
        return lib.kvq_paged_tree_attn(byref(a["q"]), byref(a["k"]), byref(a["v"]), a["pages"], a["table"],
                                       a["table_stride"], a["seq"], byref(a["out"]), *sizes, a["bits"], a["group"], *tail)
    return lib.kvq_tree_attn(byref(a["q"]), byref(a["k"]), byref(a["v"]), a["seq"], byref(a["out"]), *sizes, a["bits"],
                             a["group"], *tail)


@pytest.mark.parametrize("form", ["quant", "dense", "paged"])
@pytest.mark.parametrize("kw,code,needle", [
    (dict(tree=None), _lib.ERR_INVALID, "tree"),
    (dict(tree=_tree(bits=None)), _lib.ERR_INVALID, "tree->bits"),
    (dict(tree=_tree(depths=None)), _lib.ERR_INVALID, "tree->depths"),
    (dict(tree=_tree(bits=(1 << 26) + 2)), _lib.ERR_INVALID, "4-byte"),
    (dict(tree=_tree(bits_stride_b=-1)), _lib.ERR_INVALID, "strides"),
    (dict(window=3), _lib.ERR_UNSUPPORTED, "window"),
    (dict(window=-1), _lib.ERR_INVALID, "window"),
    (dict(L=1025, S=2048, table_stride=64), _lib.ERR_UNSUPPORTED, "1024"),
    (dict(D=100), _lib.ERR_UNSUPPORTED, "multiples of 8"),
    (dict(Hq=7, Hkv=2), _lib.ERR_INVALID, "multiple"),
    (dict(scale=float("nan")), _lib.ERR_INVALID, "scale"),
    (dict(scale=0.0), _lib.ERR_INVALID, "positive scale"),
    (dict(scale=-0.1), _lib.ERR_INVALID, "positive scale"),
    (dict(ws=None), _lib.ERR_WORKSPACE, "workspace"),
    (dict(ws=WS + 64), _lib.ERR_WORKSPACE, "aligned"),
    (dict(out=_fake_rows(ptr=(1 << 23) + 2)), _lib.ERR_INVALID, "out"),
])
def test_tree_attention_refuses(form, kw, code, needle):
    if form == "paged":
        kw = {"k": _pool(), "v": _pool(), "seq": 1 << 28, **kw}
        if kw.get("D") == 100 or kw.get("Hq") == 7:
            kw.pop("k"), kw.pop("v")
    _expect(_call(form, **kw), code, needle)


def _pool(D=128, bits=8):
    w = D * bits // 32
    return _lib.QTensor(1 << 20, 1 << 21, 1 << 22, 8 * 64 * w, 64 * w, w, 8 * 64 * 2, 64 * 2, 2)


def test_paged_tree_needs_lengths():
    _expect(_call("paged", k=_pool(), v=_pool()), _lib.ERR_INVALID, "seq_lens")


def test_tree_workspace_covers_both_kernels():
    lib = _lib.lib()
    for D in (64, 96, 128, 256):
        for L in (1, 16, 64, 200):
            n = lib.kvq_tree_workspace_size(2, 32, 8, L, D, 5000, 0)
            assert n >= lib.kvq_decode_workspace_size(2, 32, 8, L, D, 5000, 0) > 0
    assert lib.kvq_tree_workspace_size(2, 30, 8, 4, 128, 5000, 0) == 0
    assert lib.kvq_tree_workspace_size(2, 32, 8, 0, 128, 5000, 0) == 0
    # few rows stay on the decode kernel, tens and hundreds take kernels of their own
    assert lib.kvq_tree_kernel(1, 8, 8, 8, 128, 5000, 8, 64, 0) == _lib.TREE_DECODE
    assert lib.kvq_tree_kernel(1, 64, 8, 8, 128, 32768, 8, 64, 0) == _lib.TREE_ROWS
    assert lib.kvq_tree_kernel(1, 64, 8, 64, 128, 32768, 8, 64, 0) == _lib.TREE_PREFILL
    assert lib.kvq_tree_kernel(1, 64, 8, 64, 256, 32768, 16, 64, 0) == _lib.TREE_DECODE  # (one kernel at 256 dims unquantized)
    assert lib.kvq_tree_kernel(1, 30, 8, 64, 128, 32768, 8, 64, 0) == _lib.TREE_DECODE  # (no such call)
    for group in (0, 1, 8, -64):  # no such groups: any answer, but an answer
        assert lib.kvq_tree_kernel(1, 64, 8, 64, 256, 32768, 8, group, 0) in (0, 1, 2)
    for D in (96, 256):  # two kernels
        assert lib.kvq_tree_kernel(1, 64, 8, 64, D, 4096, 8, 64 if D > 96 else 32, 0) == _lib.TREE_PREFILL
        assert lib.kvq_tree_kernel(1, 64, 8, 2, D, 300, 8, 64 if D > 96 else 32, 0) == _lib.TREE_DECODE


def test_draft_tree_refuses():
    lib = _lib.lib()
    ok = (1 << 20, 8, 2, 8, 1 << 21, 1 << 22, None, 0, None, None)

    def call(**kw):
        names = ("parents", "stride", "B", "L", "bits", "depths", "starts", "start", "positions", "stream")
        a = dict(zip(names, ok))
        a.update(kw)
        return lib.kvq_draft_tree(*(a[n] for n in names))

    for kw, code, needle in [
        (dict(parents=None), _lib.ERR_INVALID, "parents"),
        (dict(bits=None), _lib.ERR_INVALID, "bits"),
        (dict(depths=None), _lib.ERR_INVALID, "depths"),
        (dict(L=1025), _lib.ERR_UNSUPPORTED, "1024"),
        (dict(B=70000), _lib.ERR_UNSUPPORTED, "65535"),
        (dict(L=-1), _lib.ERR_INVALID, "negative"),
        (dict(stride=-1), _lib.ERR_INVALID, "stride"),
        (dict(positions=(1 << 23) + 2), _lib.ERR_INVALID, "4-byte"),
    ]:
        _expect(call(**kw), code, needle)
    assert call(B=0) == _lib.OK and call(L=0) == _lib.OK  # nothing to do, no launch
    with pytest.raises(ValueError, match="GPU"):
        kernels.DraftTree(torch.tensor([-1, 0], dtype=torch.int32))
