"""The kernel of a tree's tens of query rows against the exact 64-bit oracle: every head dim, group, width and type
it serves, with one split, few (merged by the last to finish) and many, ragged rows and keys, windows, unequal
lengths, unaligned outputs and bf16 caches with and without range words. Operands are fp16 (bf16 over an unquantized
bf16 cache) as in the prefill kernel, and the tolerances are those of the other attention tests (tests/helpers.py)."""

import math

import pytest
import torch

from myinfer_amd import _lib, kernels
from tests.helpers import assert_close, seeded_normal
from tests.test_gpu_decode import make_cache
from tests.test_gpu_tree import check, exact, make_parents, tensor, values_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


def on_rows_kernel(B, Hq, Hkv, D, G, L, S, window=0, bits=8):
    return _lib.lib().kvq_tree_kernel(B, Hq, Hkv, L, D, S, bits, G, window) == _lib.TREE_ROWS


CASES = [
    # (B, Hq, Hkv, D, G, bits, dtype, L, S, kind, window)
    (1, 64, 4, 128, 64, 8, torch.float16, 21, 2049, "random", 0),    # 336 rows, 16 splits
    (2, 64, 8, 128, 64, 8, torch.bfloat16, 33, 577, "gaps", 0),      # few splits, merged by the last
    (8, 64, 8, 128, 64, 4, torch.float16, 30, 130, "random", 0),     # one split
    (2, 32, 4, 128, 64, 4, torch.bfloat16, 30, 1409, "gaps", 0),
    (1, 64, 8, 128, 32, 8, torch.float16, 17, 1100, "random", 0),    # four groups a row
    (2, 64, 4, 128, 32, 4, torch.bfloat16, 13, 1023, "gaps", 0),
    (1, 32, 4, 128, 128, 8, torch.float16, 64, 3500, "star", 0),     # one group a row
    (1, 32, 4, 128, 128, 4, torch.bfloat16, 59, 3500, "random", 0),
    (4, 64, 8, 64, 64, 8, torch.float16, 33, 1201, "chain", 0),
    (2, 64, 8, 64, 64, 4, torch.bfloat16, 40, 2100, "gaps", 0),
    (2, 64, 8, 64, 32, 8, torch.bfloat16, 24, 1601, "random", 0),
    (4, 64, 8, 64, 32, 4, torch.float16, 29, 900, "gaps", 0),
    (4, 64, 8, 128, 64, 8, torch.float16, 64, 600, "random", 80),    # windows: the first keys hidden from all
    (4, 64, 8, 128, 64, 4, torch.bfloat16, 40, 700, "gaps", 200),
    (4, 64, 8, 128, 64, 8, torch.float16, 33, 33, "random", 0),      # no prefix
]


@pytest.mark.parametrize("B,Hq,Hkv,D,G,bits,dtype,L,S,kind,window", CASES)
def test_quantized(B, Hq, Hkv, D, G, bits, dtype, L, S, kind, window):
    print(f"tree rows B={B} Hq={Hq} Hkv={Hkv} D={D} G={G} bits={bits} {dtype} L={L} S={S} {kind} window={window}", flush=True)
    assert on_rows_kernel(B, Hq, Hkv, D, G, L, S, window, bits)
    kt, vt = make_cache(B, Hkv, S, D, bits, dtype, 340 + L, group=G)
    q = seeded_normal((B, Hq, L, D), 341 + S, dtype, DEV)
    parents = make_parents(kind, B, L, 342 + D)
    scale = 1.0 / math.sqrt(D)
    tree = kernels.DraftTree(tensor(parents))
    out = kernels.attention(q, kt, vt, scale, group_size=G, bits=bits, tree=tree, window=window)
    ref = exact(q, values_of(kt, dtype, G, bits), values_of(vt, dtype, G, bits), scale, parents, [S] * B, S, window)
    check(out, ref, parents, f"D={D} L={L}")
    for _ in range(3):  # the splits' counters are left as they were found
        assert torch.equal(kernels.attention(q, kt, vt, scale, group_size=G, bits=bits, tree=tree, window=window), out)


@pytest.mark.parametrize("B,Hq,Hkv,D,dtype,L,S,kind,window", [
    (1, 64, 4, 128, torch.float16, 20, 2047, "random", 0),
    (2, 64, 8, 128, torch.bfloat16, 40, 650, "gaps", 0),
    (4, 64, 16, 128, torch.bfloat16, 30, 150, "random", 0),
    (4, 64, 8, 64, torch.float16, 40, 2000, "gaps", 0),
    (2, 64, 8, 64, torch.bfloat16, 40, 4100, "random", 0),
    (4, 64, 8, 128, torch.float16, 30, 700, "random", 200),
])
def test_unquantized(B, Hq, Hkv, D, dtype, L, S, kind, window):
    print(f"tree rows unquantized B={B} Hq={Hq} Hkv={Hkv} D={D} {dtype} L={L} S={S} {kind} window={window}", flush=True)
    assert on_rows_kernel(B, Hq, Hkv, D, 64, L, S, window, 16)
    k, v = (seeded_normal((B, Hkv, S, D), 350 + i, dtype, DEV) for i in range(2))
    q = seeded_normal((B, Hq, L, D), 352, dtype, DEV)
    parents = make_parents(kind, B, L, 353)
    scale = 1.0 / math.sqrt(D)
    out = kernels.attention(q, k, v, scale, tree=kernels.DraftTree(tensor(parents)), window=window)
    ref = exact(q, k.cpu().double().numpy(), v.cpu().double().numpy(), scale, parents, [S] * B, S, window)
    check(out, ref, parents, f"D={D} L={L}")


@pytest.mark.parametrize("B,Hq,Hkv,D,G,bits,dtype,L,S,kind,window", [
    (1, 64, 8, 128, 64, 8, torch.bfloat16, 64, 3001, "gaps", 0),
    (1, 64, 8, 128, 64, 4, torch.float16, 70, 2700, "random", 0),
    (1, 64, 8, 128, 32, 8, torch.float16, 64, 3001, "random", 0),
    (1, 64, 8, 128, 128, 4, torch.bfloat16, 64, 3001, "chain", 0),
    (2, 64, 8, 64, 64, 4, torch.float16, 80, 2111, "gaps", 0),
    (2, 64, 8, 64, 32, 8, torch.bfloat16, 80, 2111, "random", 0),
    (2, 64, 8, 128, 64, 8, torch.float16, 100, 1500, "random", 1300),
    (2, 64, 8, 128, 64, 16, torch.bfloat16, 64, 1500, "gaps", 0),
    (4, 64, 8, 64, 64, 16, torch.float16, 100, 1450, "random", 0),
    (1, 32, 4, 256, 64, 8, torch.float16, 30, 2100, "gaps", 0),      # the head_dim-256 kernel
    (2, 32, 4, 256, 128, 4, torch.bfloat16, 33, 1500, "random", 0),
    (2, 32, 4, 256, 64, 8, torch.bfloat16, 40, 1501, "gaps", 900),
    (1, 64, 8, 96, 32, 8, torch.bfloat16, 20, 1900, "gaps", 0),      # the 96-wide one
    (2, 32, 4, 96, 32, 4, torch.float16, 45, 1500, "random", 1100),
])
def test_past_the_rows_kernel(B, Hq, Hkv, D, G, bits, dtype, L, S, kind, window):
    """Sizes whose estimate is lowest for the prefill kernels."""
    print(f"tree prefill B={B} Hq={Hq} Hkv={Hkv} D={D} G={G} bits={bits} {dtype} L={L} S={S} {kind} window={window}", flush=True)
    assert _lib.lib().kvq_tree_kernel(B, Hq, Hkv, L, D, S, bits, G, window) == _lib.TREE_PREFILL
    q = seeded_normal((B, Hq, L, D), 331 + S, dtype, DEV)
    parents = make_parents(kind, B, L, 332 + D)
    scale = 1.0 / math.sqrt(D)
    tree = kernels.DraftTree(tensor(parents))
    if bits == 16:
        k, v = (seeded_normal((B, Hkv, S, D), 333 + i, dtype, DEV) for i in range(2))
        out = kernels.attention(q, k, v, scale, tree=tree, window=window)
        kd, vd = k.cpu().double().numpy(), v.cpu().double().numpy()
    else:
        kt, vt = make_cache(B, Hkv, S, D, bits, dtype, 335 + L, group=G)
        out = kernels.attention(q, kt, vt, scale, group_size=G, bits=bits, tree=tree, window=window)
        kd, vd = values_of(kt, dtype, G, bits), values_of(vt, dtype, G, bits)
    check(out, exact(q, kd, vd, scale, parents, [S] * B, S, window), parents, f"D={D} L={L}")


@pytest.mark.parametrize("Hq,Hkv,D,G,bits,dtype,L,window", [
    (64, 8, 128, 64, 8, torch.float16, 20, 0),
    (32, 4, 128, 64, 4, torch.bfloat16, 37, 0),
    (64, 8, 128, 32, 4, torch.float16, 18, 0),
    (64, 8, 64, 64, 8, torch.bfloat16, 40, 0),
    (64, 8, 64, 32, 4, torch.float16, 33, 0),
    (64, 8, 128, 128, 8, torch.float16, 37, 500),
    (64, 8, 128, 64, 8, torch.bfloat16, 70, 0),    # the prefill kernel
    (64, 8, 64, 64, 4, torch.float16, 111, 0),
    (32, 4, 256, 128, 8, torch.bfloat16, 33, 0),
    (32, 4, 96, 32, 4, torch.bfloat16, 40, 0),
])
def test_paged_unequal_lengths(Hq, Hkv, D, G, bits, dtype, L, window):
    """Pages in a shuffled order whose unused rows hold NaN scales; one sequence is its tree alone, one tree ends on
    a page's last row and one on the next page's first. The call with lengths over contiguous rows is the same."""
    from tests.test_gpu_paged import build

    print(f"tree rows paged Hq={Hq} Hkv={Hkv} D={D} G={G} bits={bits} {dtype} L={L} window={window}", flush=True)
    lens = [L, 640, 641, 1999]
    B, S = len(lens), max(lens)
    assert on_rows_kernel(B, Hq, Hkv, D, G, L, S, window, bits) == (L < 70 and D in (64, 128))
    assert _lib.lib().kvq_tree_kernel(B, Hq, Hkv, L, D, S, bits, G, window) != _lib.TREE_DECODE
    _, tables, kp, vp, kc, vc = build(B, Hkv, lens, D, bits, dtype, 360, group=G)
    if dtype == torch.bfloat16:
        for tr in (kp, vp):
            kernels.register_range_word(tr[0], torch.zeros(1, dtype=torch.int32, device=DEV))
    q = seeded_normal((B, Hq, L, D), 361, dtype, DEV)
    parents = make_parents("gaps", B, L, 362)
    scale = 1.0 / math.sqrt(D)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    tree = kernels.DraftTree(tensor(parents))
    out = kernels.paged_attention(q, kp, vp, tables, seq, scale, group_size=G, bits=bits, tree=tree, window=window, max_len=S)
    ref = exact(q, values_of(kc, dtype, G, bits), values_of(vc, dtype, G, bits), scale, parents, lens, S, window)
    check(out, ref, parents, f"D={D}")
    assert torch.equal(kernels.attention(q, kc, vc, scale, seq_lens=seq, group_size=G, bits=bits, tree=tree, window=window), out)


def test_lengths_below_the_tree():
    L, S, D, lens = 30, 1200, 128, [3, 0, 30, 1200]
    kt, vt = make_cache(4, 4, S, D, 8, torch.float16, 370)
    q = seeded_normal((4, 64, L, D), 371, torch.float16, DEV)
    parents = make_parents("chain", 4, L, 0)
    assert on_rows_kernel(4, 64, 4, D, 64, L, S)
    out = kernels.attention(q, kt, vt, 0.1, seq_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                            tree=kernels.DraftTree(tensor(parents)))
    ref = exact(q, values_of(kt, torch.float16, 64, 8), values_of(vt, torch.float16, 64, 8), 0.1, parents, lens, S)
    assert_close(out, ref, "short")


@pytest.mark.parametrize("pad,off", [(4, 0), (0, 4), (12, 4)])
def test_views_and_unaligned_outputs(pad, off):
    """Output rows that are 8-byte aligned only, capacity-padded caches, transposed queries, a shared tree; and the same
    rows where the sizes ask for the prefill kernel, which cannot store them."""
    for B, Hq, Hkv, L, S in [(2, 64, 8, 20, 1000), (2, 16, 1, 48, 1500), (1, 64, 8, 64, 5000)]:
        D, dtype = 128, torch.float16
        kt, vt = make_cache(B, Hkv, S, D, 8, dtype, 380, cap=S + 100)
        q = seeded_normal((B, L, Hq, D), 381, dtype, DEV).transpose(1, 2)
        buf = torch.full((B * L * Hq * (D + pad) + off,), float("nan"), dtype=dtype, device=DEV)
        out = buf[off:].view(B, L, Hq, D + pad)[..., :D].transpose(1, 2)
        assert on_rows_kernel(B, Hq, Hkv, D, 64, L, S) == (S < 5000)
        p = make_parents("random", 1, L, 382)
        kernels.attention(q, kt, vt, 0.09, out=out, tree=kernels.DraftTree(tensor(p[0])))
        ref = exact(q, values_of(kt, dtype, 64, 8), values_of(vt, dtype, 64, 8), 0.09, p * B, [S] * B, S)
        assert_close(out, ref, "unaligned")
        n = torch.isnan(buf).sum().item()
        assert n == off + B * L * Hq * pad  # nothing beside the rows is written


def test_bf16_cache_with_and_without_range_words():
    """A bf16 cache beyond the fp16 range: the rows kernel finds its operands' exponents itself, with or without range
    words, from the tiles' scales and biases."""
    from tests.test_gpu_paged import build

    Hq, Hkv, D, L, lens = 64, 8, 128, 20, [1000, 333]
    S, B = 1000, 2
    assert on_rows_kernel(B, Hq, Hkv, D, 64, L, S)
    _, tables, kp, vp, kc, vc = build(B, Hkv, lens, D, 8, torch.bfloat16, 390)
    for tr in (vp, vc):
        tr[1].mul_(2.0 ** 17), tr[2].mul_(2.0 ** 17)
    q = seeded_normal((B, Hq, L, D), 391, torch.bfloat16, DEV)
    parents = make_parents("random", B, L, 392)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    tree = kernels.DraftTree(tensor(parents))
    ref = exact(q, values_of(kc, torch.bfloat16, 64, 8), values_of(vc, torch.bfloat16, 64, 8) / 2.0 ** 17, 0.09, parents, lens, S)
    out = kernels.attention(q, kc, vc, 0.09, seq_lens=seq, tree=tree)
    assert_close(out / 2.0 ** 17, ref, "contiguous")
    out = kernels.paged_attention(q, kp, vp, tables, seq, 0.09, tree=tree, max_len=S)
    assert_close(out / 2.0 ** 17, ref, "pages")


def test_nonfinite_values_stay_hidden():
    """NaN and infinities in keys that a row does not see, and in absent nodes' queries, stay where they are."""
    Hq, Hkv, D, L, S = 64, 8, 128, 40, 1100
    assert on_rows_kernel(1, Hq, Hkv, D, 64, L, S)
    dtype = torch.float16
    k, v = (seeded_normal((1, Hkv, S, D), 400 + i, dtype, DEV) for i in range(2))
    q = seeded_normal((1, Hq, L, D), 402, dtype, DEV)
    parents = make_parents("star", 1, L, 0)
    parents[0][2] = -2
    q[:, :, 2] = float("nan")
    k[:, :, S - L + 2] = float("nan")
    k[:, :, S - 1] = float("inf")
    ref = exact(q.nan_to_num(0), k.nan_to_num(0, 0, 0).cpu().double().numpy(), v.cpu().double().numpy(), 0.1, parents, [S], S)
    out = kernels.attention(q, k, v, 0.1, tree=kernels.DraftTree(tensor(parents)))
    assert_close(out[:, :, :-1], ref[:, :, :-1], "others")
    assert not out[:, :, 2].any() and not torch.isfinite(out[:, :, -1]).any()


@pytest.mark.parametrize("G,bits,D", [(64, 8, 128), (32, 4, 128), (128, 8, 128), (32, 8, 64), (64, 4, 64)])
def test_bf16_ranges_by_tile(G, bits, D):
    """K and V rows of a bf16 cache whose magnitudes grow and shrink by powers of two from tile to tile, up to 2^40 (K
    2^20): every power of two is exact. With V's, queries of zero weigh all keys alike; with K's, queries of 2^-19 keep the
    scores of the usual size, so that the operands' rounding moves them as little as in the other tests."""
    Hq, Hkv, L, S, B = 64, 8, 30, 2000 if 16 * G // D > 8 else 1500, 2
    assert on_rows_kernel(B, Hq, Hkv, D, G, L, S, 0, bits)
    kt, vt = make_cache(B, Hkv, S, D, bits, torch.bfloat16, 420, group=G)
    p2 = torch.ones(S, dtype=torch.float32)
    for at, n, e in [(64, 40, 20), (333, 5, 40), (700, 1, 17), (1201, 64, 33)]:
        p2[at:at + n] = 2.0 ** e
    p2 = p2.to(DEV)[None, None, :, None]
    big = [tuple([c, (s.float() * m).bfloat16(), (b.float() * m).bfloat16()]) for (c, s, b), m in ((kt, p2), (vt, p2))]
    q = torch.zeros(B, Hq, L, D, dtype=torch.bfloat16, device=DEV)  # no weight depends on the large keys
    parents = make_parents("random", B, L, 421)
    tree = kernels.DraftTree(tensor(parents))
    out = kernels.attention(q, big[0], big[1], 0.1, group_size=G, bits=bits, tree=tree)
    top = 2.0 ** 40
    ref = exact(q, values_of(big[0], torch.bfloat16, G, bits) / top, values_of(big[1], torch.bfloat16, G, bits) / top, 0.1, parents,
                [S] * B, S)
    scale = abs(ref).max()
    assert_close((out.float() / (top * scale)).bfloat16(), ref / scale, "V by tile")
    # large keys, queries so small that the scores are of the usual size
    p2 = torch.ones(S, dtype=torch.float32)
    for at, n, e in [(64, 40, 20), (333, 5, 18), (700, 1, 17), (1201, 64, 19)]:
        p2[at:at + n] = 2.0 ** e
    p2 = p2.to(DEV)[None, None, :, None]
    kbig = (kt[0], (kt[1].float() * p2).bfloat16(), (kt[2].float() * p2).bfloat16())
    q = seeded_normal((B, Hq, L, D), 422, torch.bfloat16, DEV) * 2.0 ** -19
    out = kernels.attention(q, kbig, vt, 0.1, group_size=G, bits=bits, tree=tree)
    ref = exact(q, values_of(kbig, torch.bfloat16, G, bits), values_of(vt, torch.bfloat16, G, bits), 0.1, parents, [S] * B, S)
    assert_close(out, ref, "K by tile")


@pytest.mark.parametrize("amp", [0.0, 1e-4, 60.0])
def test_score_range(amp):
    """Queries of zero, of subnormal products and of scores far apart: one key's weight is 1, the running maximum
    moves by hundreds. fp16 keys' rounding moves a score of size s by 2^-11 s / sqrt(3) at most a key element, so the
    large scores are compared over keys whose codes are exact."""
    Hq, Hkv, D, L, S, dtype = 64, 8, 128, 20, 2000, torch.float16
    assert on_rows_kernel(1, Hq, Hkv, D, 64, L, S)
    codes = torch.randint(0, 256, (1, Hkv, S, D), generator=torch.Generator().manual_seed(410), dtype=torch.uint8).to(DEV)
    kt = (codes.view(torch.uint32), torch.full((1, Hkv, S, 2), 2.0 ** -7, dtype=dtype, device=DEV),
          torch.full((1, Hkv, S, 2), -1.0, dtype=dtype, device=DEV))
    _, vt = make_cache(1, Hkv, S, D, 8, dtype, 411)
    q = seeded_normal((1, Hq, L, D), 412, dtype, DEV) * amp
    parents = make_parents("random", 1, L, 413)
    out = kernels.attention(q, kt, vt, 0.09, tree=kernels.DraftTree(tensor(parents)))
    ref = exact(q, values_of(kt, dtype, 64, 8), values_of(vt, dtype, 64, 8), 0.09, parents, [S], S)
    assert_close(out, ref, f"amp {amp}")
