"""Seeded random trees over random caches against the exact 64-bit oracle: head dims, groups, widths, types, forms,
windows, lengths, absent nodes, capacity-padded views and strided queries drawn together."""

import math
import random

import pytest
import torch

from myinfer_amd import _lib, kernels
from tests.helpers import seeded_normal
from tests.test_gpu_decode import make_cache
from tests.test_gpu_tree import check, exact, make_parents, tensor, values_of

pytestmark = pytest.mark.gpu
DEV = "cuda"
SHAPES = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 64), (256, 128), (96, 32), (32, 32), (192, 64)]


def draw(seed):
    r = random.Random(seed)
    D, G = r.choice(SHAPES)
    form = r.choice(["quant", "quant", "paged", "dense"]) if D in (64, 96, 128, 256) else "quant"
    many = seed % 2 == 1  # rows and keys enough for the kernels of tens and hundreds of rows
    Hkv = 8 if many else r.choice([1, 2, 4, 8])
    L = max(1, int(round(math.exp(r.uniform(math.log(12) if many else 0, math.log(130))))))
    S = L + int(round(math.exp(r.uniform(math.log(400) if many else 0, math.log(2500)))))
    B = r.choice([1, 2, 3])
    rep = 8 if many else r.choice([1, 2, 4, 8])
    while B * Hkv * rep * L * S * D > (4e10 if many else 4e9):
        L, S = max(1, 2 * L // 3), S if many else L + (S - L) // 2 + 1
    return dict(D=D, G=G if form != "dense" else 64, form=form, Hkv=Hkv, Hq=Hkv * rep, L=L, S=S, B=B,
                bits=16 if form == "dense" else r.choice([4, 8]), dtype=r.choice([torch.float16, torch.bfloat16]),
                window=r.choice([0, 0, 0, L, L + 37, 500 + L]), kind=r.choice(["random", "gaps", "gaps", "chain", "star"]),
                lens=r.random() < 0.4 or form == "paged", cap=r.choice([0, 0, 33]), seed=seed, rng=r)


@pytest.mark.parametrize("seed", range(40))
def test_random_trees(seed):
    c = draw(seed)
    B, Hq, Hkv, D, G, bits, dtype, L, S = (c[n] for n in ("B", "Hq", "Hkv", "D", "G", "bits", "dtype", "L", "S"))
    kernel = _lib.lib().kvq_tree_kernel(B, Hq, Hkv, L, D, S, bits, G, c["window"])
    print({k: v for k, v in c.items() if k != "rng"}, "kernel", kernel, flush=True)
    lens = [S if b == 0 else c["rng"].randint(L, S) for b in range(B)] if c["lens"] else [S] * B
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = seeded_normal((B, L, Hq, D), 8000 + seed, dtype, DEV).transpose(1, 2)
    parents = make_parents(c["kind"], B, L, 8100 + seed)
    tree = kernels.DraftTree(tensor(parents))
    scale = 1.0 / math.sqrt(D)
    kw = dict(tree=tree, window=c["window"])
    if c["form"] == "dense":
        k, v = (seeded_normal((B, Hkv, S + c["cap"], D), 8200 + 2 * seed + i, dtype, DEV)[:, :, :S] for i in range(2))
        out = kernels.attention(q, k, v, scale, seq_lens=seq if c["lens"] else None, **kw)
        kd, vd = k.cpu().double().numpy(), v.cpu().double().numpy()
    elif c["form"] == "quant":
        kt, vt = make_cache(B, Hkv, S, D, bits, dtype, 8300 + seed, cap=S + c["cap"], group=G)
        out = kernels.attention(q, kt, vt, scale, seq_lens=seq if c["lens"] else None, group_size=G, bits=bits, **kw)
        kd, vd = values_of(kt, dtype, G, bits), values_of(vt, dtype, G, bits)
    else:
        from tests.test_gpu_paged import build

        lens = [max(n, 3) for n in lens]  # (its pages are written in two pieces of at least a row)
        S = max(lens)
        seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
        _, tables, kp, vp, kc, vc = build(B, Hkv, lens, D, bits, dtype, 8400 + seed, group=G)
        if c["cap"] and dtype == torch.bfloat16:  # with and without the pools' range words
            for tr in (kp, vp):
                kernels.register_range_word(tr[0], torch.zeros(1, dtype=torch.int32, device=DEV))
        out = kernels.paged_attention(q, kp, vp, tables, seq, scale, group_size=G, bits=bits, max_len=S, **kw)
        kd, vd = values_of(kc, dtype, G, bits), values_of(vc, dtype, G, bits)
    check(out, exact(q, kd, vd, scale, parents, lens, S, c["window"]), parents, f"seed {seed}")
