"""A drafted step over caches whose heads, sequences and pages lie gigabytes apart: every offset that passes 32 bits.

The same numbers in a compact layout go through the same kernels in the same order, so all results are equal bit for bit."""

import pytest
import torch

from myinfer_amd import _lib, attention, kernels
from tests.helpers import seeded_normal
from tests.test_gpu_decode import make_cache
from tests.test_gpu_tree import make_parents, tensor

pytestmark = pytest.mark.gpu
DEV = "cuda"
STEP = 2 ** 31 + 4096  # bytes between heads (contiguous) or pages


class Far:
    """Copies of small tensors in one large buffer, STEP bytes between the entries of an axis."""

    def __init__(self, entries):
        self.buf = torch.empty(entries * STEP, dtype=torch.uint8, device=DEV)
        self.at = 0

    def put(self, x, paged=False):
        n, m = x.shape[:2]
        raw = x.view(torch.int32) if x.dtype == torch.uint32 else x
        size = raw.element_size()
        near = raw[0].numel() if paged else raw[0, 0].numel()
        step = STEP // size
        strides = (step, raw.stride(1)) if paged else (m * step, step)
        last = (n - 1) * strides[0] + (m - 1) * strides[1]
        flat = self.buf.view(raw.dtype)
        assert raw.is_contiguous() and self.at % 4096 == 0 and self.at + near * size <= STEP
        assert (last * size + self.at + near * size) <= self.buf.numel() and last * size >= 2 ** 32
        out = flat.as_strided(raw.shape, (*strides, raw.stride(2), 1), self.at // size)
        out.copy_(raw)
        self.at += -(-near * size // 4096) * 4096
        return out.view(torch.uint32) if x.dtype == torch.uint32 else out


def bits_of(x):
    return x.contiguous().view({4: torch.int32, 2: torch.int16}[x.element_size()])


def same(a, b):
    return all(torch.equal(bits_of(x), bits_of(y)) for x, y in zip(a, b))


@pytest.mark.parametrize("bits,D,Hq,on", [(8, 128, 32, {0, 1, 2}), (4, 64, 32, {0, 1, 2}), (8, 256, 4, {0, 2})])
def test_contiguous(bits, D, Hq, on):
    B, H, cap, rows = 2, 2, 8200, 8192
    far = Far(B * H)
    near = [tuple(x.contiguous() for x in tr) for tr in make_cache(B, H, cap, D, bits, torch.float16, 3)]
    away = [tuple(far.put(x) for x in tr) for tr in near]
    axes = kernels.RopeAxes(D, sections=(D // 8, D // 4, D // 8))
    kernels_seen = set()
    for L in (3, 8, 60, 120):
        print(f"far contiguous bits={bits} D={D} L={L}", flush=True)
        parents = tensor(make_parents("gaps", B, L, L))
        tree = kernels.DraftTree(parents, starts=rows - L)
        positions = tree.positions.expand(3, B, L).contiguous()
        k, v = (seeded_normal((B, H, L, D), 10 + i, torch.float16, DEV) for i in range(2))
        q = seeded_normal((B, Hq, L, D), 12, torch.float16, DEV)
        q2 = q.clone()
        for (kt, vt), qq in ((near, q), (away, q2)):
            kernels.prepare_axes_append(kt, vt, rope=axes, group_size=64, bits=bits)(k, v, positions, rows - L, qq)
        assert same(near[0] + near[1] + (q,), away[0] + away[1] + (q2,))
        got = []
        for kt, vt in (near, away):
            views = [tuple(x[:, :, :rows] for x in tr) for tr in (kt, vt)]
            got.append((attention.blocked_quantized_sdpa(q, *views, 0.1, tree, 64, bits),
                        *kernels.dequantize_rows(*views, group_size=64, bits=bits)))
        assert same(*got)
        kernels_seen.add(_lib.lib().kvq_tree_kernel(B, Hq, H, L, D, rows, bits, 64, 0))
        kept = tensor([list(range(1, L))] * B)
        for kt, vt in (near, away):
            kernels.keep_rows([*kt, *vt], kept, rows - L, L)
        assert same(near[0] + near[1], away[0] + away[1])
    assert kernels_seen == on  # (each kernel has been seen)


@pytest.mark.parametrize("Hq,L", [(2, 3), (32, 60), (32, 120)])  # on the decode, the rows and the prefill kernel
def test_unquantized_and_queries(Hq, L):
    """K, V and the rows read back with far heads, and queries rotated there."""
    print(f"far unquantized Hq={Hq} L={L}", flush=True)
    B, H, S, D = 2, 2, 8192, 64
    far = Far(B * H)
    k, v = (seeded_normal((B, H, S, D), 20 + i, torch.bfloat16, DEV) for i in range(2))
    q = seeded_normal((B, Hq, L, D), 22, torch.bfloat16, DEV)
    tree = kernels.DraftTree(tensor(make_parents("random", B, L, 23)), starts=0)
    fk, fv, fq = far.put(k), far.put(v), far.put(q) if Hq == H else q.clone()
    axes = kernels.RopeAxes(D)
    kernels.rope_axes(fq, axes, tree.positions)
    kernels.rope_axes(q, axes, tree.positions)
    assert same((q,), (fq,))
    assert same((attention.fast_scaled_dot_product_attention(q, k, v, 0.125, tree),),
                (attention.fast_scaled_dot_product_attention(fq, fk, fv, 0.125, tree),))
    kt, vt = make_cache(B, H, S, D, 8, torch.bfloat16, 24)
    got = kernels.dequantize_rows(kt, vt, group_size=64, bits=8, out=(fk, fv))
    assert same(got, kernels.dequantize_rows(kt, vt, group_size=64, bits=8))


@pytest.mark.parametrize("bits,Hq,L", [(8, 2, 20), (4, 32, 60)])  # on the decode and the rows kernel
def test_pages(bits, Hq, L):
    print(f"far pages bits={bits} Hq={Hq} L={L}", flush=True)
    B, H, D, pages = 2, 2, 128, 4
    far = Far(pages)
    near = [tuple(x.contiguous() for x in tr) for tr in make_cache(pages, H, 64, D, bits, torch.float16, 31)]
    away = [tuple(far.put(x, paged=True) for x in tr) for tr in near]
    table, lens = tensor([[3, 0], [1, 2]]), tensor([100, 128])
    starts = lens - L
    axes = kernels.RopeAxes(D)
    tree = kernels.DraftTree(tensor(make_parents("random", B, L, 32)), starts=starts)
    k, v = (seeded_normal((B, H, L, D), 33 + i, torch.float16, DEV) for i in range(2))
    q = seeded_normal((B, Hq, L, D), 35, torch.float16, DEV)
    got = []
    for kt, vt in (near, away):
        qq = q.clone()
        kernels.prepare_axes_append(kt, vt, rope=axes, group_size=64, bits=bits).paged(k, v, tree.positions, table, starts, 0, qq)
        out = kernels.paged_attention(qq, kt, vt, table, lens, 0.1, group_size=64, bits=bits, tree=tree)
        back = [torch.zeros(B, H, 128, D, dtype=torch.float16, device=DEV) for _ in range(2)]
        kernels.paged_dequantize(kt, vt, table, lens, group_size=64, bits=bits, out=tuple(back))
        kernels.paged_keep_rows([(kt, vt)], table, tensor([[1, 4, 9], [0, 2, -1]]), starts=starts, n=L)
        got.append((qq, out, *back, *kt, *vt))
    assert same(*got)
