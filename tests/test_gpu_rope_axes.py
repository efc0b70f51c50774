"""Rotation at positions of several axes against the exact 64-bit oracle, and fused with the quantize-append.

Tolerance of a rotated element: cos and sin are off by at most 2^-23 (fp32 rounding and the series' remainder), the two
products and the sum round to fp32 (3 more of 2^-24 of |x| + |y|): under d = 2^-22 (|x| + |y|) in all; then one
rounding to T, at most eps/2 of the result (2^-25 where fp16 is subnormal). Far positions add the angle's own rounding in
double: |angle| 2^-51."""

import numpy as np
import pytest
import torch

from myinfer_amd import kernels
from myinfer_amd.cache import QuantizedKVCache
from oracle import axes as OX
from tests.helpers import seeded_normal, to_np_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def positions(A, B, L, seed, high=40000):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, high, (A, B, L), generator=g, dtype=torch.int32)


def check(got, x, pos, r, what):
    if pos.dim() == 2:
        pos = pos[:, None].expand(-1, x.shape[0], -1)
    ref, size = OX.rotate(x.double().numpy(), pos.numpy(), r.dims, r.sections, r.traditional, r.base, r.scale, r.interleaved,
                          r.restart)
    far = np.abs(pos.numpy().astype(np.float64)).max() * abs(r.scale) * 2.0 ** -51
    d = (2.0 ** -22 + far) * size
    half = torch.finfo(x.dtype).eps / 2
    bound = half * (np.abs(ref) + d) + d + 2.0 ** -25
    g = got.cpu().double().numpy()
    assert np.array_equal(to_np_bits(got)[..., r.dims:], to_np_bits(x)[..., r.dims:]), f"{what}: dims past the rotated ones"
    err = np.abs(g - ref)
    assert (err <= bound).all(), f"{what}: {err.max()} at {np.unravel_index(np.argmax(err - bound), err.shape)}"


ROPES = [
    kernels.RopeAxes(128, (16, 24, 24), base=1e6),
    kernels.RopeAxes(128, (16, 24, 24), base=1e6, interleaved=True),
    kernels.RopeAxes(128, (24, 20, 20), traditional=True, interleaved=True),
    kernels.RopeAxes(64, (16, 16), restart=True),
    kernels.RopeAxes(96, (7, 5, 35, 1), interleaved=True, restart=True, scale=0.25),
    kernels.RopeAxes(16, (8,), traditional=True),
    kernels.RopeAxes(128),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("r", ROPES)
def test_rotation(r, dtype):
    print(f"rope_axes {r} {dtype}", flush=True)
    for B, H, L in [(1, 1, 1), (2, 5, 37), (1, 33, 3)]:
        x = seeded_normal((B, H, L, 128), 7 + H, dtype)
        x[0, 0, 0] *= 30.0
        pos = positions(r.axes, B, L, H)
        y = x.to(DEV)
        assert kernels.rope_axes(y, r, pos.to(DEV)) is y
        check(y, x, pos, r, f"{B} {H} {L}")


@pytest.mark.parametrize("D,dims", [(64, 64), (256, 256), (96, 48), (80, 32), (192, 192)])
def test_head_dims_and_many_rows(D, dims):
    r = kernels.RopeAxes(dims, (dims // 4, dims // 4))
    x = seeded_normal((2, 40, 333, D), D, torch.bfloat16)
    pos = positions(2, 2, 333, D)
    y = x.to(DEV)
    kernels.rope_axes(y, r, pos.to(DEV))
    check(y, x, pos, r, f"D={D}")


def test_views_and_broadcast_positions():
    """Queries as [B, L, H, D] projections seen [B, H, L, D], rows of a wider buffer, one position list for the batch,
    positions as strided views."""
    r = kernels.RopeAxes(64, (10, 12, 10))
    B, H, L = 3, 4, 50
    base = seeded_normal((B, L, H, 3 * 64), 11, torch.float16)
    x = base[..., 64:128].transpose(1, 2)
    dev = base.to(DEV)
    y = dev[..., 64:128].transpose(1, 2)
    wide = positions(6, 1, 2 * L, 12)[:, 0].to(DEV)
    kernels.rope_axes(y, r, wide[::2, ::2])
    check(y, x, wide[::2, ::2].cpu(), r, "views")
    assert torch.equal(dev[..., :64].cpu(), base[..., :64]) and torch.equal(dev[..., 128:].cpu(), base[..., 128:])


@pytest.mark.parametrize("high", [2 ** 20, 2 ** 31 - 1])
def test_far_and_negative_positions(high):
    r = kernels.RopeAxes(128, (32, 32), base=1e4)
    x = seeded_normal((1, 2, 300, 128), 13, torch.float16)
    pos = positions(2, 1, 300, 14, high)
    pos[:, :, ::3] *= -1
    pos[0, 0, 5], pos[1, 0, 6] = -2 ** 31, 2 ** 31 - 1
    y = x.to(DEV)
    kernels.rope_axes(y, r, pos.to(DEV))
    check(y, x, pos, r, "far")


@pytest.mark.parametrize("traditional", [False, True])
def test_one_axis_agrees_with_rope(traditional):
    """Consecutive positions on one axis are Rope's rows: equal at near positions but for an ulp now and then (its
    angles are rounded to fp32)."""
    x = seeded_normal((1, 8, 64, 128), 15, torch.bfloat16, DEV)
    a = kernels.rope(x.clone(), kernels.Rope(128, traditional), offset=9)
    b = kernels.rope_axes(x.clone(), kernels.RopeAxes(128, traditional=traditional),
                          torch.arange(9, 73, dtype=torch.int32, device=DEV)[None])
    assert float((a != b).float().mean()) <= 2e-3
    assert torch.allclose(a.float(), b.float(), rtol=2.0 ** -7, atol=2.0 ** -12)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,H,Hq,L,D,G,bits,r", [
    (1, 8, 64, 16, 128, 64, 8, kernels.RopeAxes(128)),
    (2, 3, 6, 45, 128, 64, 4, kernels.RopeAxes(128, (16, 24, 24), interleaved=True)),
    (1, 2, 0, 9, 128, 128, 2, kernels.RopeAxes(64, (16, 16), traditional=True)),
    (1, 5, 5, 7, 96, 32, 8, kernels.RopeAxes(96, (20, 28))),
    (2, 8, 16, 1100, 128, 64, 8, kernels.RopeAxes(128, (16, 24, 24))),   # 32 elements a thread
    (1, 4, 4, 2500, 256, 128, 4, kernels.RopeAxes(128, (32, 32), restart=True)),
    (1, 4, 4, 2100, 256, 32, 8, kernels.RopeAxes(256, (64, 64), traditional=True)),
])
def test_fused_append(B, H, Hq, L, D, G, bits, r, dtype):
    """The cache holds exactly what quantizing the rotated keys stores, the queries what rope_axes makes of them, and
    nothing else is written."""
    print(f"rope_axes_append B={B} H={H} Hq={Hq} L={L} D={D} G={G} bits={bits} {dtype}", flush=True)
    k, v = (seeded_normal((B, H, L, D), 20 + i, dtype, DEV) for i in range(2))
    q = seeded_normal((B, Hq, L, D), 22, dtype, DEV) if Hq else None
    pos = positions(r.axes, B, L, 23).to(DEV)
    k_was = k.clone()
    row = 5

    def empty():
        codes = torch.full((B, H, L + 9, D * bits // 32), -1, dtype=torch.int32, device=DEV).view(torch.uint32)
        sc = torch.full((B, H, L + 9, D // G), float("nan"), dtype=dtype, device=DEV)
        return codes, sc, sc.clone()

    want = [empty(), empty()]
    kernels.quantize_append(kernels.rope_axes(k.clone(), r, pos), want[0], v, want[1], row_offset=row, group_size=G, bits=bits)
    got = [empty(), empty()]
    words = torch.zeros(2, dtype=torch.int32, device=DEV)
    for i in range(2):
        kernels.register_range_word(got[i][0], words[i: i + 1])
    q2 = None if q is None else q.clone()
    kernels.prepare_axes_append(*got, rope=r, group_size=G, bits=bits)(k, v, pos, row, q2)
    for a, b in zip(got[0] + got[1], want[0] + want[1]):
        kind = torch.int32 if a.dtype == torch.uint32 else torch.int16
        assert torch.equal(a.view(kind), b.view(kind))
    assert torch.equal(k, k_was)
    if q is not None:
        assert torch.equal(q2, kernels.rope_axes(q.clone(), r, pos))
    # keys alone
    alone = empty()
    kernels.prepare_axes_append(alone, rope=r, group_size=G, bits=bits)(k, None, pos, row)
    for a, b in zip(alone, want[0]):
        kind = torch.int32 if a.dtype == torch.uint32 else torch.int16
        assert torch.equal(a.view(kind), b.view(kind))


def test_range_word_is_raised():
    c = QuantizedKVCache(64, 8)
    k = seeded_normal((1, 2, 4, 128), 30, torch.float32, DEV)
    c.update_and_fetch((k * 1e6).bfloat16(), k.bfloat16(), rope=kernels.RopeAxes(128),
                       positions=torch.zeros(1, 4, dtype=torch.int32, device=DEV))
    assert c.range_exponents()[0] >= 6 and c.range_exponents()[1] == 0


def test_cache_update_grows_and_pieces_agree():
    r = kernels.RopeAxes(64, (16, 16))
    B, H, L, D = 2, 3, 300, 64
    k, v = (seeded_normal((B, H, L, D), 31 + i, torch.float16, DEV) for i in range(2))
    q = seeded_normal((B, 6, L, D), 33, torch.float16, DEV)
    pos = positions(2, B, L, 34).to(DEV)
    one, many = QuantizedKVCache(64, 4), QuantizedKVCache(64, 4)
    q1, q2 = q.clone(), q.clone()
    one.update_and_fetch(k, v, rope=r, positions=pos, queries=q1)
    for a, b in [(0, 1), (1, 7), (7, 200), (200, 300)]:
        many.update_and_fetch(k[:, :, a:b], v[:, :, a:b], rope=r, positions=pos[:, :, a:b], queries=q2[:, :, a:b])
    assert torch.equal(q1, q2) and one.offset == many.offset == L
    for x, y in zip(one.fetch()[0] + one.fetch()[1], many.fetch()[0] + many.fetch()[1]):
        kind = torch.int32 if x.dtype == torch.uint32 else torch.int16
        assert torch.equal(x.contiguous().view(kind), y.contiguous().view(kind))


def test_paged_append():
    """Rows at per-sequence starts through shuffled pages equal the contiguous append; rows past the table, or on a page
    marked -1, are dropped."""
    B, H, Hq, L, D, bits, dtype = 3, 2, 4, 20, 128, 8, torch.bfloat16
    r = kernels.RopeAxes(128, (16, 24, 24))
    k, v = (seeded_normal((B, H, L, D), 40 + i, dtype, DEV) for i in range(2))
    q = seeded_normal((B, Hq, L, D), 42, dtype, DEV)
    pos = positions(3, B, L, 43).to(DEV)
    starts = torch.tensor([60, 0, 120], dtype=torch.int32, device=DEV)
    table = torch.tensor([[3, 1], [5, -1], [0, 2]], dtype=torch.int32, device=DEV)

    def pool():
        codes = torch.full((7, H, 64, D * bits // 32), -1, dtype=torch.int32, device=DEV).view(torch.uint32)
        sc = torch.full((7, H, 64, 2), float("nan"), dtype=dtype, device=DEV)
        return codes, sc, sc.clone()

    kp, vp = pool(), pool()
    q2 = q.clone()
    kernels.paged_rope_axes_append(k, kp, v, vp, table, r, pos, starts=starts, queries=q2)
    assert torch.equal(q2, kernels.rope_axes(q.clone(), r, pos))
    want_k, want_v = pool(), pool()
    kernels.paged_quantize_append(kernels.rope_axes(k.clone(), r, pos), want_k, v, want_v, table, starts=starts)
    for a, b in zip(kp + vp, want_k + want_v):
        kind = torch.int32 if a.dtype == torch.uint32 else torch.int16
        assert torch.equal(a.view(kind), b.view(kind))
    assert torch.isnan(kp[1][4]).all() and torch.isnan(kp[1][6]).all()


def test_refusals():
    x = seeded_normal((1, 2, 3, 64), 50, torch.float16, DEV)
    r = kernels.RopeAxes(64, (16, 16))
    ok = torch.zeros(2, 1, 3, dtype=torch.int32, device=DEV)
    for bad in (ok.long(), ok.cpu(), ok[:1], ok[:, :, :2], ok[0], ok.float()):
        with pytest.raises(ValueError, match="positions"):
            kernels.rope_axes(x, r, bad)
    with pytest.raises(ValueError, match="16-byte"):
        kernels.rope_axes(seeded_normal((1, 2, 3, 68), 51, torch.float16, DEV)[..., 2:66], r, ok)
    with pytest.raises(NotImplementedError, match="dims"):
        kernels.rope_axes(x, kernels.RopeAxes(128, (32, 32)), ok)
    c = QuantizedKVCache(64, 8)
    with pytest.raises(ValueError, match="queries"):
        c.update_and_fetch(x, x, rope=r, positions=ok, queries=x[:, :, :2])
    assert c.offset == 0
    with pytest.raises(ValueError, match="values"):
        c.update_and_fetch(x, x[:, :1], rope=r, positions=ok)
