"""Calls of the operators around a speculative decoding step over a cache, as cases with inputs from a seed,
their work, a plain form in elementary torch operations and a 64-bit reference.

Kinds of case (``kind``):
  rope    query rows rotated at positions of one or several axes (time, height, width).
  write   an attention layer's step up to its attention: queries and keys rotated at given positions, keys
          and values quantized into the cache; the new rows are read back as the values the cache now holds.
  tree    attention of the nodes of a tree of drafted tokens: each sees the cached prefix, its ancestors and
          itself. Over a quantized cache, an unquantized one ("dense") or pages ("paged", sequences of
          unequal lengths and trees of unequal sizes, padded with absent nodes).
  keep    the drafted rows that were accepted move up behind the prefix, the others are dropped, in the
          caches of several layers ("paged" or not).
  read    cached rows read back as values, from a quantized cache or through block tables ("paged").

``run`` computes the plain form, or where ``own`` is set makes the framework's calls on the same state.
"""

import math

import torch

own = False

_DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
_PAGE = 64  # rows of a page


def _rope_case(name, B, H, D, L, dims, sections, dtype, traditional=False, interleaved=False, restart=False):
    return dict(name=name, kind="rope", B=B, Hq=H, D=D, L=L, dims=dims, sections=sections, dtype=dtype,
                traditional=traditional, interleaved=interleaved, restart=restart)


def _write_case(name, B, Hq, Hkv, D, L, S, bits, G, sections, dtype):
    return dict(name=name, kind="write", B=B, Hq=Hq, Hkv=Hkv, D=D, L=L, S=S, bits=bits, G=G, dims=D,
                sections=sections, dtype=dtype, traditional=False, interleaved=False, restart=False)


def _tree_case(name, form, B, Hq, Hkv, D, L, S, bits, G, dtype, window=0):
    return dict(name=name, kind="tree", form=form, B=B, Hq=Hq, Hkv=Hkv, D=D, L=L, S=S, bits=bits, G=G, dtype=dtype,
                window=window)


def _keep_case(name, form, layers, B, Hkv, D, L, M, S, bits, G, dtype):
    return dict(name=name, kind="keep", form=form, layers=layers, B=B, Hkv=Hkv, D=D, L=L, M=M, S=S, bits=bits, G=G,
                dtype=dtype)


def _read_case(name, form, B, Hkv, D, S, bits, G, dtype):
    return dict(name=name, kind="read", form=form, B=B, Hkv=Hkv, D=D, S=S, bits=bits, G=G, dtype=dtype)


def listed():
    return [
        # the queries of one token of a small model that reads images: launch and latency
        _rope_case("rope-token", 1, 16, 128, 1, 128, "16,24,24", "fp16"),
        # the queries of a 4096-token piece of a video prompt
        _rope_case("rope-video", 1, 32, 128, 4096, 128, "16,24,24", "bf16"),
        # sixteen drafted tokens of a large model written at their tree positions after 32K tokens
        _write_case("write-tree", 1, 64, 8, 128, 16, 32784, 8, 64, "64", "bf16"),
        # a 2048-token piece of a video prompt written to the cache
        _write_case("write-video", 1, 32, 4, 128, 2048, 8192, 8, 64, "16,24,24", "fp16"),
        # a small tree over a 4096-token cache of a small model
        _tree_case("tree-small", "quant", 1, 16, 8, 128, 10, 4106, 8, 64, "fp16"),
        # 64 drafted tokens of a large model over 32K tokens
        _tree_case("tree-32k", "quant", 1, 64, 8, 128, 64, 32832, 8, 64, "bf16"),
        # eight users of unequal lengths up to 8K tokens, 16 drafted tokens each, over 4-bit pages
        _tree_case("tree-users", "paged", 8, 32, 8, 128, 16, 8192, 4, 64, "bf16"),
        # a tree of 31 over plain caches of heads of 64, four users
        _tree_case("tree-dense-d64", "dense", 4, 32, 8, 64, 31, 2047, 16, 64, "fp16"),
        # six of 26 drafted tokens accepted, all 32 layers of a model
        _keep_case("keep-model", "quant", 32, 1, 8, 128, 26, 6, 4096, 8, 64, "bf16"),
        # up to five of 16 drafted tokens of each of eight users, pages of four layers
        _keep_case("keep-users", "paged", 4, 8, 8, 128, 16, 5, 2048, 8, 64, "fp16"),
        # a 32K-token cache of a large model handed on unquantized
        _read_case("read-32k", "quant", 1, 8, 128, 32768, 8, 64, "bf16"),
        # four users' 4-bit pages, unequal lengths up to 1999 rows
        _read_case("read-users", "paged", 4, 8, 128, 1999, 4, 64, "fp16"),
    ]


def _pick(rng, lo, hi):
    """A size from lo to hi, even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


# (query heads, KV heads)
_HEADS = ((16, 8), (64, 8), (32, 4), (32, 16), (32, 8), (32, 32), (16, 16), (8, 1))
_MAX_FLOPS = 4.4e10
_MAX_BYTES = 2.0e8


def _sections(rng, dims):
    """Pairs of each axis: one axis, or two to four with at least one pair each."""
    n, pairs = rng.choice((1, 1, 2, 3, 3, 4)), dims // 2
    cuts = sorted(rng.sample(range(1, pairs), n - 1))
    return ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))


def draw(rng):
    while True:
        kind = rng.choice(("rope", "write", "tree", "tree", "keep", "read"))
        Hq, Hkv = rng.choice(_HEADS)
        D, dtype = rng.choice((64, 128, 128, 256, 96)), rng.choice(("fp16", "bf16"))
        G = 32 if D == 96 else rng.choice((64, 64, 128)) if D > 64 else 64
        bits = rng.choice((8, 8, 4))
        if kind in ("rope", "write"):
            dims = rng.choice((D, D, D // 2 // 16 * 16))
            case = dict(kind=kind, B=rng.choice((1, 1, 2, 4)), Hq=Hq, D=D, L=_pick(rng, 1, 4096), dims=dims,
                        sections=_sections(rng, dims), dtype=dtype, traditional=rng.random() < 0.25,
                        interleaved=rng.random() < 0.3, restart=rng.random() < 0.3)
            if kind == "write":
                case.update(Hkv=Hkv, S=case["L"] + _pick(rng, 1, 8192), bits=bits, G=G)
        elif kind == "tree":
            form = rng.choice(("quant", "quant", "paged", "dense"))
            L = _pick(rng, 1, 128)
            case = dict(kind=kind, form=form, B=rng.choice((1, 1, 2, 4)) if form != "paged" else rng.randint(2, 8), Hq=Hq,
                        Hkv=Hkv, D=D, L=L, S=L + _pick(rng, 1, 32768), bits=16 if form == "dense" else bits,
                        G=64 if form == "dense" else G, dtype=dtype, window=rng.choice((0, 0, 0, 512, 1024)))
        elif kind == "keep":
            L = _pick(rng, 1, 128)
            case = dict(kind=kind, form=rng.choice(("quant", "paged")), layers=rng.randint(1, 32), B=rng.choice((1, 2, 8)),
                        Hkv=Hkv, D=D, L=L, M=rng.randint(1, min(L, 16)), S=L + _pick(rng, 1, 1024), bits=bits, G=G,
                        dtype=dtype)
        else:
            case = dict(kind=kind, form=rng.choice(("quant", "paged")), B=rng.choice((1, 1, 2, 4)), Hkv=Hkv, D=D,
                        S=_pick(rng, 1, 32768), bits=bits, G=G, dtype=dtype)
        w = work(case)
        # (a score is 4 D flops: small heads have more of them)
        if w["flops"] <= min(_MAX_FLOPS, 5e8 * D) and w["bytes"] <= _MAX_BYTES and _cache_bytes(case) <= 2e9:
            return case


def _cache_bytes(case):
    if "S" not in case:
        return 0
    return case.get("layers", 1) * case["B"] * case["Hkv"] * case["S"] * 4 * case["D"]


# ---- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, B, H, n, D, dt):
    """K or V rows as projections give them: normal, each dim at a scale of its own within a factor of
    two or so."""
    dims = torch.exp(0.3 * torch.randn(1, 1, 1, D, generator=g, device="cuda"))
    return (torch.randn(B, H, n, D, generator=g, device="cuda") * dims).to(dt)


def _affine(x, bits, G):
    """(codes, scales, biases) of MLX's affine quantizer, in the 32 bits it is defined in; codes as floats."""
    n = float(2 ** bits - 1)
    y = x.float().reshape(*x.shape[:-1], -1, G)
    lo, hi = y.amin(-1, keepdim=True), y.amax(-1, keepdim=True)
    low = lo.abs() > hi.abs()
    s = torch.clamp((hi - lo) / n, min=1e-7)
    s = torch.where(low, s, -s)
    edge = torch.where(low, lo, hi)
    q0 = torch.round(edge / s)
    s = torch.where(q0 != 0, edge / torch.where(q0 != 0, q0, torch.ones_like(q0)), s)
    b = torch.where(q0 != 0, edge, torch.zeros_like(edge))
    codes = torch.clamp(torch.round((y - b) / s), 0, n)
    return codes.reshape(x.shape), s.to(x.dtype)[..., 0], b.to(x.dtype)[..., 0]


def _pack(codes, bits):
    per = 32 // bits
    c = codes.to(torch.int64).view(*codes.shape[:-1], -1, per)
    w = (c << (torch.arange(per, device=codes.device) * bits)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32).view(torch.uint32)


def _unpack(words, bits):
    per = 32 // bits
    w = words.view(torch.int32).unsqueeze(-1)
    c = (w >> (torch.arange(per, device=words.device, dtype=torch.int32) * bits)) & (2 ** bits - 1)
    return c.reshape(*words.shape[:-1], -1)


def _triple(x, bits, G):
    codes, s, b = _affine(x, bits, G)
    return _pack(codes, bits), s.contiguous(), b.contiguous()


def _empty_triple(B, H, n, D, bits, G, dt):
    s = torch.zeros(B, H, n, D // G, dtype=dt, device="cuda")
    return torch.zeros(B, H, n, D * bits // 32, dtype=torch.int32, device="cuda").view(torch.uint32), s, s.clone()


def _sizes(case):
    return [int(n) for n in case["sections"].split(",")]


def _positions(g, case):
    """int32 [axes, B, L]. One axis: a tree's or a prompt's own, some way into a long text. Several: rows of
    frames of some height and width, as a video prompt has them."""
    A, B, L = len(_sizes(case)), case["B"], case["L"]
    start = torch.randint(0, 32768, (B, 1), generator=g, device="cuda")
    i = torch.arange(L, device="cuda")[None]
    if A == 1:
        pos = (start + i // 2)[None]
    else:
        wide = torch.randint(8, 33, (B, 1), generator=g, device="cuda")
        high = torch.randint(8, 33, (B, 1), generator=g, device="cuda")
        pos = torch.stack([start + i // (wide * high), start + i // wide % high, start + i % wide, start + i][:A])
    return pos.to(torch.int32)


def _parents(g, B, L, deep=12):
    """int32 [B, L]: the parent of each drafted token, -1 for those that follow the prefix. Wide near the
    root, a few tokens deep."""
    draws = torch.rand(B, L, generator=g, device="cuda").cpu().tolist()
    out = []
    for row in draws:
        depth, par = [], []
        for l, u in enumerate(row):
            p = int(u * u * (l + 1)) - 1  # (u^2: earlier tokens have more children)
            if p >= 0 and depth[p] >= deep:
                p = -1
            par.append(p)
            depth.append(0 if p < 0 else depth[p] + 1)
        out.append(par)
    return torch.tensor(out, dtype=torch.int32)


def _pages(g, case, lens):
    """A block table over shuffled pages, for sequences of at most S rows."""
    n = -(-case["S"] // _PAGE)
    return torch.randperm(case["B"] * n, generator=g, device="cuda").view(case["B"], n).to(torch.int32)


def _paged(x, table):
    """The rows x [B, H, n, W] in pages [num_pages, H, 64, W] by the block table."""
    B, H, n, W = x.shape
    P = table.shape[1]
    y = x.view(torch.int32) if x.dtype == torch.uint32 else x
    full = torch.zeros(B, H, P * _PAGE, W, dtype=y.dtype, device=x.device)
    full[:, :, :n] = y
    pool = torch.empty(B * P, H, _PAGE, W, dtype=y.dtype, device=x.device)
    pool[table.long().view(-1)] = full.view(B, H, P, _PAGE, W).transpose(1, 2).reshape(B * P, H, _PAGE, W)
    return pool.view(torch.uint32) if x.dtype == torch.uint32 else pool


def _unpaged(pool, table):
    """The pages of each sequence as contiguous rows [B, H, pages * 64, W]."""
    y = pool.view(torch.int32) if pool.dtype == torch.uint32 else pool
    B, P = table.shape
    y = y[table.long()].transpose(1, 2).reshape(B, y.shape[1], P * _PAGE, y.shape[3])
    return y.view(torch.uint32) if pool.dtype == torch.uint32 else y


def prepare(case, seed):
    g, dt, kind = _gen(seed), _DT[case["dtype"]], case["kind"]
    B, D = case["B"], case["D"]
    st = {"case": case}
    if kind in ("rope", "write"):
        st["q"] = torch.randn(B, case["Hq"], case["L"], D, generator=g, device="cuda").to(dt)
        st["pos"] = _positions(g, case)
    if kind == "write":
        st["k"], st["v"] = (_rows(g, B, case["Hkv"], case["L"], D, dt) for _ in range(2))
        cap = -(-case["S"] // 256) * 256
        st["keys"], st["values"] = (_empty_triple(B, case["Hkv"], cap, D, case["bits"], case["G"], dt) for _ in range(2))
    if kind in ("rope", "write"):
        return st
    Hkv, S, bits, G, form = (case[n] for n in ("Hkv", "S", "bits", "G", "form"))
    if kind == "tree":
        L = case["L"]
        st["q"] = torch.randn(B, case["Hq"], L, D, generator=g, device="cuda").to(dt)
        parents = _parents(g, B, L)
        if form == "paged":  # unequal trees: the nodes past a sequence's own are absent
            own_nodes = torch.randint((L + 1) // 2, L + 1, (B,), generator=g, device="cuda").cpu()
            parents[torch.arange(L)[None] >= own_nodes[:, None]] = -2
        st["parents"] = parents.cuda()
        k, v = (_rows(g, B, Hkv, S, D, dt) for _ in range(2))
        st["lens"] = torch.full((B,), S, dtype=torch.int32, device="cuda")
        if form == "paged":
            st["lens"] = torch.randint(max(L, S // 2), S + 1, (B,), generator=g, device="cuda").to(torch.int32)
        st["keys"], st["values"] = (k, v) if form == "dense" else (_triple(x, bits, G) for x in (k, v))
    elif kind == "keep":
        # one buffer for all layers, each cache a view of it; the drafted rows are the last L of S
        N, L, M = case["layers"], case["L"], case["M"]
        st["layers"] = [[_rows_as_words(g, (N, B, Hkv, S, D * bits // 32))] +
                        [torch.randn(N, B, Hkv, S, D // G, generator=g, device="cuda").to(dt) for _ in range(2)]
                        for _ in range(2)]
        rows = torch.rand(B, L, generator=g, device="cuda").argsort(-1)[:, :M].sort(-1)[0].to(torch.int32)
        st["starts"] = torch.full((B,), S - L, dtype=torch.int32, device="cuda")
        if form == "paged":  # unequal lengths, and fewer rows accepted for some
            st["starts"] = torch.randint(0, S - L + 1, (B,), generator=g, device="cuda").to(torch.int32)
            count = torch.randint(1, M + 1, (B, 1), generator=g, device="cuda")
            rows = torch.where(torch.arange(M, device="cuda")[None] < count, rows, -1)
        else:
            rows = rows[:1].expand(B, M)
        st["rows"] = rows.to(torch.int32).contiguous()
    else:
        st["keys"], st["values"] = (_triple(_rows(g, B, Hkv, S, D, dt), bits, G) for _ in range(2))
        st["lens"] = torch.full((B,), S, dtype=torch.int32, device="cuda")
        if form == "paged":
            st["lens"] = torch.randint((S + 1) // 2, S + 1, (B,), generator=g, device="cuda").to(torch.int32)
            st["out"] = tuple(torch.zeros(B, Hkv, S, D, dtype=dt, device="cuda") for _ in range(2))
    if form == "paged":
        st["table"] = _pages(g, case, None)
        if kind == "keep":
            st["layers"] = [[torch.stack([_paged(y, st["table"]).view(torch.int32) if y.dtype == torch.uint32 else
                                          _paged(y, st["table"]) for y in x]) for x in tr] for tr in st["layers"]]
            for tr in st["layers"]:
                tr[0] = tr[0].view(torch.uint32)
        else:
            st["keys"], st["values"] = (tuple(_paged(x, st["table"]) for x in st[n]) for n in ("keys", "values"))
    return st


def _rows_as_words(g, shape):
    return torch.randint(-2 ** 31, 2 ** 31, shape, generator=g, device="cuda", dtype=torch.int64).to(torch.int32).view(torch.uint32)


# ---- the plain forms

def _pair_axes(case):
    """Axis and frequency index of each pair, and the pairs that a frequency index counts to."""
    sizes, pairs = _sizes(case), case["dims"] // 2
    if case["interleaved"]:
        left, axes, a = list(sizes), [], 0
        while len(axes) < pairs:  # dealt to the axes in turn, until each has its pairs
            if left[a]:
                left[a] -= 1
                axes.append(a)
            a = (a + 1) % len(sizes)
    else:
        axes = [a for a, n in enumerate(sizes) for _ in range(n)]
    if case["restart"]:  # each axis counts its own pairs
        index = [axes[:i].count(a) for i, a in enumerate(axes)]
        per = [sizes[a] for a in axes]
    else:
        index, per = list(range(pairs)), [pairs] * pairs
    return axes, [i / n for i, n in zip(index, per)]


_BASE = 1000000.0


def _plain_rotated(x, pos, case):
    """x with its first dims rotated: angles in 64 bits, the rotation in 32, rounded once."""
    axes, fraction = _pair_axes(case)
    freq = _BASE ** -torch.tensor(fraction, dtype=torch.float64, device=x.device)
    angle = pos.double()[torch.tensor(axes, device=x.device)].permute(1, 2, 0) * freq  # [B, L, pairs]
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    n = case["dims"]
    y = x.float()
    if case["traditional"]:
        a, b = y[..., 0:n:2], y[..., 1:n:2]
        r = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    else:
        a, b = y[..., : n // 2], y[..., n // 2: n]
        r = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    return torch.cat([r, y[..., n:]], dim=-1).to(x.dtype)


def _plain_values(tr, bits, G):
    codes, s, b = tr
    c = _unpack(codes, bits).float().view(*s.shape, G)
    return (c * s.float().unsqueeze(-1) + b.float().unsqueeze(-1)).flatten(-2)


def _plain_ancestors(parents):
    """bool [B, L, L]: node j is l or an ancestor of l; no column for an absent node, nor its row."""
    B, L = parents.shape
    p = parents.long()
    here = p >= -1
    seen = torch.eye(L, dtype=torch.bool, device=p.device)[None] & here[:, None]
    up = torch.zeros(B, L + 1, L, dtype=torch.bool, device=p.device)
    while True:  # one generation more each time
        up[:, :L] = seen
        more = (seen | up.gather(1, torch.where(p >= 0, p, L)[:, :, None].expand(B, L, L))) & here[:, :, None]
        if torch.equal(more, seen):
            return seen
        seen = more


def _plain_tree(q, keys, values, parents, lens, scale, window):
    """q [B, Hq, L, D]; keys and values float32 [B, Hkv, S, D]; sequence b has lens[b] rows, its tree last."""
    B, Hq, L, D = q.shape
    Hkv, S = keys.shape[1:3]
    seen = _plain_ancestors(parents)
    depth = seen.sum(-1) - 1  # -1 for an absent node
    first = (lens.long() - L)[:, None]  # the first row of the tree
    t = torch.arange(S, device=q.device)[None]
    node = t - first  # [B, S]
    prefix = (t < first)[:, None] & (depth >= 0)[:, :, None]
    if window:
        prefix = prefix & (t[:, None] > (first + depth)[:, :, None] - window)
    inside = ((node >= 0) & (node < L))[:, None] & seen.gather(2, node.clamp(0, L - 1)[:, None].expand(B, L, S))
    visible = (prefix | inside)[:, None, None]  # [B, 1, 1, L, S]
    qs = q.float().view(B, Hkv, Hq // Hkv * L, D)
    scores = torch.matmul(qs, keys.transpose(-1, -2)).view(B, Hkv, Hq // Hkv, L, S) * scale
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > -math.inf, top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    return torch.matmul(p.view(B, Hkv, -1, S), values).view(B, Hq, L, D).to(q.dtype)


def _scale(case):
    return 1.0 / math.sqrt(case["D"])


def _plain_write(st):
    case = st["case"]
    L, S, bits, G = (case[n] for n in ("L", "S", "bits", "G"))
    st["q"].copy_(_plain_rotated(st["q"], st["pos"], case))
    new = []
    for rows, tr in ((_plain_rotated(st["k"], st["pos"], case), st["keys"]), (st["v"], st["values"])):
        codes, s, b = _triple(rows, bits, G)
        tr[0].view(torch.int32)[:, :, S - L: S] = codes.view(torch.int32)
        tr[1][:, :, S - L: S] = s
        tr[2][:, :, S - L: S] = b
        new.append(_plain_values([x[:, :, S - L: S].contiguous() for x in tr], bits, G).to(rows.dtype))
    return {"q": st["q"], "keys": new[0], "values": new[1]}


def _words(x):
    return x.view(torch.int32) if x.dtype == torch.uint32 else x


def _kept(st):
    """The rows that the move may have written: [layers, B, H, M, W] of every array."""
    case, out = st["case"], []
    for x in st["layers"][0] + st["layers"][1]:
        x = _words(x)
        if case["form"] == "paged":
            b, i = torch.arange(case["B"], device="cuda")[:, None], torch.arange(case["M"], device="cuda")[None]
            at = (st["starts"].long()[:, None] + i)
            out.append(x[:, st["table"].long()[b, at // _PAGE], :, at % _PAGE])
        else:
            out.append(x[:, :, :, case["S"] - case["L"]: case["S"] - case["L"] + case["M"]])
    return out


def _plain_keep(st):
    case, M = st["case"], st["case"]["M"]
    rows, starts = st["rows"].long(), st["starts"].long()[:, None]
    on = rows >= 0
    i = torch.arange(M, device="cuda")[None]
    src, dst = starts + torch.where(on, rows, i), starts + i  # [B, M]; a row not named stays
    b = torch.arange(case["B"], device="cuda")[:, None]
    for x in st["layers"][0] + st["layers"][1]:
        x = _words(x)
        if case["form"] == "paged":
            t = st["table"].long()
            x[:, t[b, dst // _PAGE], :, dst % _PAGE] = x[:, t[b, src // _PAGE], :, src % _PAGE]
        else:
            x[:, b, :, dst] = x[:, b, :, src]
    return _kept(st)


def _plain_read(st):
    case = st["case"]
    bits, G, dt = case["bits"], case["G"], _DT[case["dtype"]]
    if case["form"] != "paged":
        return [_plain_values(st[n], bits, G).to(dt) for n in ("keys", "values")]
    S = case["S"]
    live = (torch.arange(S, device="cuda")[None] < st["lens"][:, None])[:, None, :, None]
    for out, n in zip(st["out"], ("keys", "values")):
        x = _plain_values([_unpaged(y, st["table"])[:, :, :S].contiguous() for y in st[n]], bits, G).to(dt)
        out.copy_(torch.where(live, x, out))
    return list(st["out"])


def _plain_tree_call(st):
    case = st["case"]
    keys, values = st["keys"], st["values"]
    if case["form"] == "dense":
        keys, values = keys.float(), values.float()
    else:
        if case["form"] == "paged":
            keys, values = ([_unpaged(x, st["table"]) for x in tr] for tr in (keys, values))
        keys, values = (_plain_values(tr, case["bits"], case["G"]) for tr in (keys, values))
    return _plain_tree(st["q"], keys, values, st["parents"], st["lens"], _scale(case), case["window"])


# ---- the framework's calls

def _own_rope(st):
    from myinfer_amd import kernels

    case = st["case"]
    return kernels.RopeAxes(case["dims"], tuple(_sizes(case)), traditional=case["traditional"], base=_BASE,
                            interleaved=case["interleaved"], restart=case["restart"])


def _own_cache(st, keys, values, rows):
    """A cache over buffers the program has, as it restores a saved one."""
    from myinfer_amd.cache import QuantizedKVCache

    cache = QuantizedKVCache(group_size=st["case"]["G"], bits=st["case"]["bits"])
    cache.restore(keys, values, rows)
    return cache


def _own(st):
    from myinfer_amd import attention, cache, kernels

    case = st["case"]
    kind, L, S = case["kind"], case.get("L"), case.get("S")
    if kind == "rope":
        if "rope" not in st:
            st["rope"] = _own_rope(st)
        return kernels.rope_axes(st["q"], st["rope"], st["pos"])
    if kind == "write":
        if "rope" not in st:
            st["rope"] = _own_rope(st)
            st["cache"] = _own_cache(st, st["keys"], st["values"], S - L)
        c = st["cache"]
        c.update_and_fetch(st["k"], st["v"], rope=st["rope"], positions=st["pos"], queries=st["q"])
        keys, values = c.dequantized(S - L, S)
        c.trim(L)
        return {"q": st["q"], "keys": keys, "values": values}
    if kind == "tree":
        tree = kernels.DraftTree(st["parents"])
        if case["form"] == "paged":
            return kernels.paged_attention(st["q"], st["keys"], st["values"], st["table"], st["lens"], _scale(case),
                                           window=case["window"], group_size=case["G"], bits=case["bits"], max_len=S,
                                           tree=tree)
        if case["form"] == "dense":
            return attention.fast_scaled_dot_product_attention(st["q"], st["keys"], st["values"], _scale(case), tree,
                                                               window=case["window"])
        if "cache" not in st:
            st["cache"] = _own_cache(st, st["keys"], st["values"], S)
        keys, values = st["cache"].fetch()
        return attention.blocked_quantized_sdpa(st["q"], keys, values, _scale(case), tree, case["G"], case["bits"],
                                                window=case["window"])
    if kind == "keep":
        k, v = st["layers"]
        if case["form"] == "paged":
            if "pools" not in st:
                st["pools"] = [(tuple(x[i] for x in k), tuple(x[i] for x in v)) for i in range(case["layers"])]
            kernels.paged_keep_rows(st["pools"], st["table"], st["rows"], starts=st["starts"])
            return _kept(st)
        if "caches" not in st:
            st["caches"] = [_own_cache(st, tuple(x[i] for x in k), tuple(x[i] for x in v), S)
                            for i in range(case["layers"])]
        for c in st["caches"]:  # (the drafted rows have been appended)
            c.offset = S
        cache.keep_rows(st["caches"], S - L, st["rows"])
        return _kept(st)
    if case["form"] == "paged":
        return list(kernels.paged_dequantize(st["keys"], st["values"], st["table"], st["lens"], group_size=case["G"],
                                             bits=case["bits"], out=st["out"]))
    if "cache" not in st:
        st["cache"] = _own_cache(st, st["keys"], st["values"], S)
    return list(st["cache"].dequantized())


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "rope":
        return state["q"].copy_(_plain_rotated(state["q"], state["pos"], state["case"]))
    if kind == "write":
        return _plain_write(state)
    if kind == "tree":
        return _plain_tree_call(state)
    return _plain_keep(state) if kind == "keep" else _plain_read(state)


# ---- what a pass cannot do without

def work(case):
    kind, B, D = case["kind"], case["B"], case["D"]
    if kind == "rope":
        rows = B * case["Hq"] * case["L"]
        # (dims past the rotated ones stay where they are)
        return {"bytes": rows * case["dims"] * 4 + 4 * len(_sizes(case)) * B * case["L"], "flops": 3.0 * rows * case["dims"]}
    bits, G, Hkv = case["bits"], case["G"], case["Hkv"]
    row = 2 * 2 * D if bits == 16 else 2 * (D * bits // 8 + 4 * D // G)  # bytes of a key and its value
    if kind == "write":
        rows, L = B * Hkv * case["L"], case["L"]
        q = B * case["Hq"] * L * case["dims"] * 4
        # the new rows are read, written to the cache, read back and returned
        return {"bytes": q + rows * (2 * 2 * D + 2 * row + 2 * 2 * D) + 4 * len(_sizes(case)) * B * L,
                "flops": 3.0 * B * (case["Hq"] + Hkv) * L * case["dims"] + 6.0 * rows * 2 * D}
    if kind == "tree":
        L, S, Hq = case["L"], case["S"], case["Hq"]
        share = 0.75 if case["form"] == "paged" else 1.0  # of S rows, and of L nodes, that a sequence has
        seen = max(share * S - L, 0.0) if not case["window"] else min(max(share * S - L, 0.0), case["window"])
        nodes = share * L
        return {"bytes": B * Hkv * (seen + nodes) * row + 4.0 * B * Hq * L * D + 4.0 * B * L,
                "flops": 4.0 * D * Hq * B * nodes * (seen + min(4.0, (nodes + 1) / 2))}
    if kind == "keep":
        kept = case["M"] if case["form"] != "paged" else (case["M"] + 1) / 2
        return {"bytes": 2.0 * case["layers"] * B * Hkv * kept * row + 4.0 * B * case["M"], "flops": 0.0}
    share = 0.75 if case["form"] == "paged" else 1.0
    return {"bytes": share * B * Hkv * case["S"] * (row + 2 * 2 * D), "flops": share * 4.0 * B * Hkv * case["S"] * D}


# ---- the same in 64 bits, from the definitions

def _exact_rotated(x, pos, case):
    """x as complex numbers turned by e^(i t), pair by pair."""
    n, sizes = case["dims"], _sizes(case)
    order = []  # the axis of every pair
    if case["interleaved"]:
        waiting = [[a] * s for a, s in enumerate(sizes)]
        while any(waiting):
            order += [w.pop() for w in waiting if w]
    else:
        order = sum(([a] * s for a, s in enumerate(sizes)), [])
    turned = x.double().clone()
    count = [0] * len(sizes)
    for i, a in enumerate(order):
        e = 2.0 * (count[a] if case["restart"] else i) / (2.0 * sizes[a] if case["restart"] else n)
        count[a] += 1
        turn = torch.polar(torch.ones_like(pos[a], dtype=torch.float64), pos[a].double() * math.pow(_BASE, -e))[:, None]
        d0, d1 = (2 * i, 2 * i + 1) if case["traditional"] else (i, i + n // 2)
        z = torch.complex(x[..., d0].double(), x[..., d1].double()) * turn
        turned[..., d0], turned[..., d1] = z.real, z.imag
    return turned


def _exact_values(tr, bits, G):
    codes, s, b = tr
    n = 32 // bits
    w = codes.view(torch.int32).long() & 0xFFFFFFFF
    c = torch.stack([(w >> (bits * i)) % (1 << bits) for i in range(n)], dim=-1).flatten(-2).double()
    return c * s.double().repeat_interleave(G, -1) + b.double().repeat_interleave(G, -1)


def _exact_tree(st):
    case = st["case"]
    B, Hq, L, D = st["q"].shape
    rep, W = Hq // case["Hkv"], case["window"]
    out = torch.zeros(B, Hq, L, D, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, parents = int(st["lens"][b]), st["parents"][b].tolist()
        if case["form"] == "dense":
            k, v = st["keys"][b, :, :n].double(), st["values"][b, :, :n].double()
        elif case["form"] == "paged":
            k, v = (_exact_values([_unpaged(x, st["table"][b: b + 1])[:, :, :n].contiguous() for x in st[m]],
                                  case["bits"], case["G"])[0] for m in ("keys", "values"))
        else:
            k, v = (_exact_values([x[b: b + 1, :, :n].contiguous() for x in st[m]], case["bits"], case["G"])[0]
                    for m in ("keys", "values"))
        see = torch.zeros(L, n, dtype=torch.bool)
        for l in range(L):
            if parents[l] < -1:
                continue
            path, j = [], l
            while j >= 0:
                path.append(j)
                j = parents[j]
            at = n - L + len(path) - 1
            see[l, max(0, at - W + 1) if W else 0: n - L] = True
            see[l, [n - L + j for j in path]] = True
        hidden = ~see.cuda()
        for h in range(Hq):
            s = (st["q"][b, h].double() @ k[h // rep].t().contiguous()) * _scale(case)
            p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
            out[b, h] = torch.where(hidden.all(-1)[:, None], 0.0, p.nan_to_num(0.0) @ v[h // rep])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        return _exact_rotated(st["q"], st["pos"], case)
    if kind == "write":
        k = _exact_rotated(st["k"], st["pos"], case).to(st["k"].dtype)  # (the quantizer is given rows of its type)
        read = [_exact_values(_triple(x, case["bits"], case["G"]), case["bits"], case["G"]) for x in (k, st["v"])]
        return {"q": _exact_rotated(st["q"], st["pos"], case), "keys": read[0], "values": read[1]}
    if kind == "tree":
        return _exact_tree(st)
    if kind == "keep":  # row by row; the codes are whole numbers
        B, M = case["B"], case["M"]
        before = [x.clone() if i % 3 else None for i, x in enumerate(st["layers"][0] + st["layers"][1])]
        out = []
        for x in before:
            if x is None:
                out.append(None)
                continue
            y = torch.empty(case["layers"], B, M, case["Hkv"], x.shape[-1], dtype=torch.float64, device="cuda")
            for b in range(B):
                for i in range(M):
                    r = int(st["rows"][b, i])
                    at = int(st["starts"][b]) + (r if r >= 0 else i)
                    if case["form"] == "paged":
                        y[:, b, i] = x[:, int(st["table"][b, at // _PAGE]), :, at % _PAGE].double()
                    else:
                        y[:, b, i] = x[:, b, :, at].double()
            out.append(y.transpose(2, 3) if case["form"] != "paged" else y.permute(1, 2, 0, 3, 4))
        return out
    if case["form"] != "paged":
        return [_exact_values(st[n], case["bits"], case["G"]) for n in ("keys", "values")]
    out = []
    for n in ("keys", "values"):
        x = torch.zeros(case["B"], case["Hkv"], case["S"], case["D"], dtype=torch.float64, device="cuda")
        for b in range(case["B"]):
            m = int(st["lens"][b])
            rows = [_unpaged(y, st["table"][b: b + 1])[:, :, :m].contiguous() for y in st[n]]
            x[b, :, :m] = _exact_values(rows, case["bits"], case["G"])[0]
        out.append(x)
    return out
