"""Tree speculation (ops/tree.py) against 64-bit definitions: mask, attention, verification,
cache commit, and a whole speculative step of them."""
import math

import pytest
import torch

from vllm_xtu_moe_b200.ops import basic, tree
from vllm_xtu_moe_b200.ops import _native as N
from vllm_xtu_moe_b200.ops.tree import TreeMetadata

PAGE = 64
FP8 = torch.float8_e4m3fn
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def i32(x, device="cpu"):
    return torch.tensor(x, dtype=torch.int32, device=device)


def random_trees(lens, seed, device="cpu", back=6):
    """parents [T], q_start of trees with the given node counts."""
    g = torch.Generator().manual_seed(seed)
    par, qs = [], [0]
    for n in lens:
        for i in range(n):
            par.append(-1 if i == 0 else max(0, i - int(torch.randint(1, back + 1, (1,), generator=g))))
        qs.append(qs[-1] + n)
    return i32(par, device), i32(qs, device)


def family(parents, i):
    got = [i]
    while 0 <= parents[got[-1]] < got[-1]:
        got.append(parents[got[-1]])
    return got


# ---------------------------------------------------------------- mask
def mask_oracle(parents, q_start, W):
    par, qs = parents.tolist(), q_start.tolist()
    mask, depth = [], []
    for b in range(len(qs) - 1):
        mine = par[qs[b]:qs[b + 1]]
        for i in range(len(mine)):
            up = family(mine, i)
            words = [0] * W
            for a in up:
                words[a // 32] |= 1 << (a % 32)
            mask.append([w - 2 ** 32 if w >> 31 else w for w in words])
            depth.append(len(up) - 1)
    return i32(mask).view(-1, W), i32(depth)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [[1], [5], [32], [33, 0, 1], [64, 7, 65], [200, 3, 128, 129], [1024, 1, 1023]])
def test_mask(device, lens):
    par, qs = random_trees(lens, 1, back=6 if max(lens) < 300 else 40)
    most = max(lens)
    m0, d0 = mask_oracle(par, qs, (most + 31) // 32)
    m, d = tree.tree_mask(par.to(device), qs.to(device), most)
    assert torch.equal(m.cpu(), m0) and torch.equal(d.cpu(), d0)


@pytest.mark.parametrize("device", DEVICES)
def test_mask_odd_parents_and_rows_behind(device):
    # a root with a parent, forward and self references, a chain through all words
    par = i32([3, 0, 5, 3, -7, 4] + [-1] + list(range(69)), device)
    qs = i32([0, 6, 76], device)
    T = 80
    m = torch.full((T, 3), 77, dtype=torch.int32, device=device)
    d = torch.full((T,), 77, dtype=torch.int32, device=device)
    par = torch.cat([par, torch.zeros(T - 76, dtype=torch.int32, device=device)])
    tree.tree_mask(par, qs, 70, m, d)
    m0, d0 = mask_oracle(par.cpu(), qs.cpu(), 3)
    assert torch.equal(m[:76].cpu(), m0) and torch.equal(d[:76].cpu(), d0)
    assert (m[76:] == 77).all() and (d[76:] == 77).all()


# ---------------------------------------------------------------- attention
def make_attention(Hq, Hk, D, Dv, lens, ctx, fp8=False, seed=0, device="cpu", window=0, sinks=False, spare=3,
                   mask=None):
    g = torch.Generator().manual_seed(seed)
    par, qs = random_trees(lens, seed)
    T, most = int(qs[-1]), max(max(lens), 1)
    m, d = mask_oracle(par, qs, (most + 31) // 32)
    if mask is not None:
        m = mask(m)
    kv = [c + n for c, n in zip(ctx, lens)]
    nblk = [-(-x // PAGE) for x in kv]
    total = sum(nblk) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    bt = torch.zeros(len(lens), max(max(nblk), 1), dtype=torch.int32)
    at = 0
    for b, n in enumerate(nblk):
        bt[b, :n] = order[at:at + n]
        at += n
    q = torch.randn(T, Hq, D, generator=g).to(torch.bfloat16)
    k = torch.randn(total, Hk, PAGE, D, generator=g)
    v = torch.randn(total, Hk, Dv, PAGE, generator=g) if fp8 else torch.randn(total, Hk, PAGE, Dv, generator=g)
    ks, vs = (0.02, 0.015) if fp8 else (1.0, 1.0)
    t = FP8 if fp8 else torch.bfloat16
    meta = TreeMetadata(num_seqs=len(lens), q_start=qs, kv_len=i32(kv), block_table=bt, mask=m, max_nodes=most,
                        max_kv_len=max(kv + [1]), depth=d)
    s = dict(q=q, k=(k / ks).to(t), v=(v / vs).to(t), meta=meta, window=window, ks=ks, vs=vs,
             sinks=torch.randn(Hq, generator=g) if sinks else None)
    return to_device(s, device)


def to_device(s, device):
    import dataclasses
    m = s["meta"]
    meta = dataclasses.replace(m, **{f: getattr(m, f).to(device) for f in
                                     ("q_start", "kv_len", "block_table", "mask", "depth")})
    return {**{k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in s.items()}, "meta": meta}


def attention_oracle(s):
    """(o, sum p |v|, visible) in 64 bits: a key outside a row's view takes no part at all."""
    s = to_device(s, "cpu")
    m, w = s["meta"], s["window"]
    q, k, v = s["q"].double(), s["k"].double() * s["ks"], s["v"].double() * s["vs"]
    if s["v"].dtype == FP8:
        v = v.transpose(2, 3)
    T, Hq, D = q.shape
    Hk, Dv = k.shape[1], v.shape[3]
    o = torch.zeros(T, Hq, Dv, dtype=torch.float64)
    a = torch.zeros_like(o)
    qs, kl = m.q_start.tolist(), m.kv_len.tolist()
    for b in range(m.num_seqs):
        n = qs[b + 1] - qs[b]
        ctx = kl[b] - n
        pages = m.block_table[b].long()
        for i in range(n):
            row = qs[b] + i
            far = int(m.depth[row]) - w if w else -10 ** 9
            keys = [t for t in range(ctx) if t - ctx > far]
            for j in range(n):
                if int(m.mask[row, j // 32]) >> (j % 32) & 1 and (not w or int(m.depth[qs[b] + j]) > far):
                    keys.append(ctx + j)
            if not keys:
                continue
            t = torch.tensor(keys)
            pg, off = pages[t // PAGE], t % PAGE
            kk, vv = k[pg, :, off], v[pg, :, off]                    # [keys, Hk, D]
            for h in range(Hq):
                e = (kk[:, h // (Hq // Hk)] @ q[row, h]) * D ** -0.5
                top = e.max()
                if s["sinks"] is not None:
                    top = torch.maximum(top, s["sinks"][h].double())
                p = torch.exp(e - top)
                z = p.sum() + (torch.exp(s["sinks"][h].double() - top) if s["sinks"] is not None else 0.0)
                o[row, h] = (p / z) @ vv[:, h // (Hq // Hk)]
                a[row, h] = (p / z) @ vv[:, h // (Hq // Hk)].abs()
    return o, a


def check_attention(s, out, o=None, a=None):
    """The result's own rounding (bf16: 2^-8 of it) and P's before the second product (bf16: 2^-8
    of every p |v|; fp8 caches: f16, 2^-11, and 2^-25 absolute where p is subnormal, the
    largest p being at least 1 before the division), and 2^-12 of sum p |v| for the
    32-bit scores: products of 64 .. 256 terms of size <= 30 give |ds| < 256 * 30 * 2^-24 < 2^-11 in
    the worst case, in practice far less."""
    if o is None:
        o, a = attention_oracle(s)
    fp8 = s["v"].dtype == FP8
    tol = 2 ** -8 * o.abs() + (2 ** -11 if fp8 else 2 ** -8) * a + 2 ** -12 * a
    if fp8:
        tol = tol + 2 ** -25 * s["meta"].max_kv_len * 448 * s["vs"] / 100
    err = (out.cpu().double() - o).abs()
    worst = (err - tol).max().item() if err.numel() else -1
    assert worst <= 1e-30, (worst, err.max().item())
    assert torch.isfinite(out.float()).all()


def run_attention(s, **kw):
    return tree.tree_attention(s["q"], s["k"], s["v"], s["meta"], window=s["window"], sinks=s["sinks"],
                               k_scale=s["ks"], v_scale=s["vs"], **kw)


SHAPES = [  # Hq, Hk, D, Dv, fp8
    (4, 2, 64, 64, False), (24, 2, 128, 128, False), (16, 2, 256, 256, False), (16, 2, 192, 128, False),
    (4, 2, 64, 64, True), (24, 2, 128, 128, True), (3, 3, 128, 128, False), (48, 1, 128, 128, False)]
TREES = [([1], [0]), ([1, 1], [1, 200]), ([5], [0]), ([7, 1, 12], [63, 64, 65]), ([33, 0, 5], [127, 40, 500]),
         ([61, 17], [130, 1000])]


def test_plan():
    """Every size gets a plan within the kernels' limits; a given split count stays."""
    for B in (1, 3, 64, 2000):
        for rows in (1, 128, 129, 5000):
            for seen in (0, 1, 700, 10 ** 6):
                for d, dv in tree.HEAD_DIMS:
                    t, s = tree.tree_plan(B, 8, rows, seen, d, dv)
                    assert t in (1, 2) and 1 <= s <= tree.MAX_SPLITS and (t == 1 or (rows > 128 and dv <= 128))
                    assert tree.tree_plan(B, 8, rows, seen, d, dv, 5)[1] == 5
    assert tree.tree_plan(4, 8, 732, 14817) == (2, 3) and tree.tree_plan(8, 8, 208, 218, 192, 128)[0] == 1


@pytest.mark.parametrize("trees", TREES[:5])
def test_attention_cpu(trees):
    s = make_attention(4, 2, 64, 64, *trees, seed=2)
    check_attention(s, run_attention(s))


@pytest.mark.gpu
@pytest.mark.parametrize("trees", TREES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(shape, trees, monkeypatch):
    Hq, Hk, D, Dv, fp8 = shape
    s = make_attention(Hq, Hk, D, Dv, *trees, fp8=fp8, seed=3, device="cuda")
    o, a = attention_oracle(s)
    check_attention(s, run_attention(s), o, a)
    plan = tree.tree_plan
    for splits in (1, 3, 64):                     # more splits than pages leaves empty ones
        s["meta"].num_splits = splits
        for tiles in (1, 2) if Dv <= 128 else (1,):
            monkeypatch.setattr(tree, "tree_plan", lambda *a: (tiles, plan(*a)[1]))
            check_attention(s, run_attention(s), o, a)
    N.check_status()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("window", [1, 3, 64, 100, 5000])
@pytest.mark.parametrize("sinks", [False, True])
def test_attention_window_and_sinks(device, window, sinks):
    for Hq, Hk, D, Dv in [(4, 2, 64, 64), (16, 2, 192, 128), (24, 2, 128, 128)][:1 if device == "cpu" else 3]:
        s = make_attention(Hq, Hk, D, Dv, [9, 1, 30], [0, 63, 700], seed=4, device=device, window=window, sinks=sinks)
        check_attention(s, run_attention(s))
        s["meta"].num_splits = 2
        check_attention(s, run_attention(s))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("splits", [1, 2])
def test_attention_rows_that_see_nothing(device, splits):
    """ctx = 0 and an empty mask row: zero, with and without sinks; bits past the tree are no keys."""
    def holes(m):
        m = m.clone()
        m[::2] = 0
        m[1::2, -1] |= -2 ** 31       # bit 31 / 63: no such node
        return m
    for sinks in (False, True):
        s = make_attention(8, 2, 64, 64, [20, 40], [0, 0], seed=5, device=device, sinks=sinks, mask=holes)
        s["meta"].num_splits = splits
        out = run_attention(s)
        check_attention(s, out)
        assert (out[::2] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES[:6])
@pytest.mark.parametrize("splits", [1, 3])
def test_attention_ignores_what_a_row_does_not_see(shape, splits):
    """NaN and infinities in the slots behind the last node, in unused pages and (bf16) in the K / V
    of a node: rows that do not see them keep their value, rows that see the node do not."""
    Hq, Hk, D, Dv, fp8 = shape
    s = make_attention(Hq, Hk, D, Dv, [12, 9], [70, 0], fp8=fp8, seed=6, device="cuda")
    s["meta"].num_splits = splits
    m = s["meta"]
    o, a = attention_oracle(s)
    bad = [float("nan")] if fp8 else [float("nan"), float("inf"), float("-inf")]
    used = set()
    for b in range(2):
        for t in range(int(m.kv_len[b])):
            used.add((int(m.block_table[b, t // PAGE]), t % PAGE))
    kf, vf = s["k"].float(), s["v"].float()
    for pg in range(kf.shape[0]):
        for off in range(PAGE):
            if (pg, off) not in used:
                kf[pg, :, off] = bad[off % len(bad)]
                if fp8:
                    vf[pg, :, :, off] = bad[(off + 1) % len(bad)]
                else:
                    vf[pg, :, off] = bad[(off + 1) % len(bad)]
    t = s["k"].dtype
    clean = run_attention(s)
    s["k"], s["v"] = kf.to(t), vf.to(t)
    out = run_attention(s)
    check_attention(s, out, o, a)
    assert torch.equal(out, clean)
    # the V of node 4 of sequence 0 turns non-finite in column 1
    slot = 70 + 4
    pg, off = int(m.block_table[0, slot // PAGE]), slot % PAGE
    vf[pg][(slice(None), 1, off) if fp8 else (slice(None), off, 1)] = bad[-1]
    s["v"] = vf.to(t)
    out2 = run_attention(s)
    sees = torch.tensor([bool(int(m.mask[i, 0]) >> 4 & 1) and i < 12 for i in range(21)])
    assert torch.equal(out2[~sees], clean[~sees])
    assert not torch.isfinite(out2[sees][:, :, 1].float()).any()
    keep = [c for c in range(Dv) if c != 1]
    assert torch.equal(out2[sees][:, :, keep], clean[sees][:, :, keep])
    N.check_status()


def poison_unused(s, bad):
    """(k, v) in 32 bits with `bad` in every slot that holds no key of a sequence."""
    m, fp8 = s["meta"], s["v"].dtype == FP8
    free = torch.ones(s["k"].shape[0], PAGE, dtype=torch.bool)
    for b in range(m.num_seqs):
        t = torch.arange(int(m.kv_len[b]))
        free[m.block_table[b].cpu().long()[t // PAGE], t % PAGE] = False
    pg, off = (x.to(s["k"].device) for x in torch.nonzero(free, as_tuple=True))
    val = torch.tensor(bad, device=s["k"].device)[off % len(bad)][:, None, None]
    kf, vf = s["k"].float(), s["v"].float()
    kf[pg, :, off] = val
    if fp8:
        vf[pg, :, :, off] = val
    else:
        vf[pg, :, off] = val
    return kf, vf


RINGS = [  # shape, keys a tile, last masked tile: twice round the V slots of one row tile and further
    ((4, 2, 64, 64, False), 128, 13), ((24, 2, 128, 128, False), 128, 7), ((16, 2, 192, 128, False), 64, 9),
    ((16, 2, 256, 256, False), 64, 5), ((4, 2, 64, 64, True), 128, 7), ((24, 2, 128, 128, True), 128, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("shape,bn,last,tiles", [(*r, t) for r in RINGS for t in (1, 2) if t == 1 or r[0][3] <= 128])
@pytest.mark.parametrize("splits", [1, 2, 3])
def test_attention_of_masked_tiles_at_every_place_of_the_ring(shape, bn, last, tiles, splits, monkeypatch):
    """The first masked tile is the call's tile 0, 1, .. `last` (within a split: every place up to there), the slots
    behind the last node and a node's V hold NaN and infinities, and shared memory holds NaN from the kernel before:
    a row's value is that of the clean cache bit for bit unless it sees the node."""
    Hq, Hk, D, Dv, fp8 = shape
    ctx = [t * bn + 5 for t in range(last + 1)] + [t * bn + bn - 4 for t in range(last + 1)]
    n = 12
    s = make_attention(Hq, Hk, D, Dv, [n] * len(ctx), ctx, fp8=fp8, seed=16, device="cuda")
    m = s["meta"]
    o, a = attention_oracle(s)
    bad = [float("nan")] if fp8 else [float("nan"), float("inf"), float("-inf")]
    k, v, t = s["k"], s["v"], s["k"].dtype
    kf, vf = poison_unused(s, bad)
    vn = vf.clone()                                 # beside that, column 1 of node 4's V
    for b, c in enumerate(ctx):
        pg, off = int(m.block_table[b, (c + 4) // PAGE]), (c + 4) % PAGE
        vn[pg][(slice(None), 1, off) if fp8 else (slice(None), off, 1)] = bad[-1]
    sees = (m.mask[:, 0] >> 4 & 1).bool()
    keep = [c for c in range(Dv) if c != 1]
    dirt = torch.full((2048, 2048), float("nan"), dtype=torch.bfloat16, device="cuda")
    plan = tree.tree_plan
    m.num_splits = splits
    monkeypatch.setattr(tree, "tree_plan", lambda *x: (tiles, plan(*x)[1]))
    s["k"], s["v"] = k, v
    clean = run_attention(s)
    check_attention(s, clean, o, a)
    for _ in range(3):
        s["k"], s["v"] = k, v
        torch.mm(dirt, dirt)
        assert torch.equal(run_attention(s), clean)
        s["k"], s["v"] = kf.to(t), vf.to(t)
        torch.mm(dirt, dirt)
        assert torch.equal(run_attention(s), clean)
        s["v"] = vn.to(t)
        torch.mm(dirt, dirt)
        out = run_attention(s)
        assert torch.equal(out[~sees], clean[~sees])
        assert not torch.isfinite(out[sees][:, :, 1].float()).any()
        assert torch.equal(out[sees][:, :, keep], clean[sees][:, :, keep])
    N.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_of_a_node_with_an_infinite_value(device):
    """A node's V that some rows see and others do not."""
    s = make_attention(2, 1, 64, 64, [12], [3], seed=8, device=device)
    m = s["meta"]
    clean = run_attention(s)
    s["v"][int(m.block_table[0, 0]), :, 3 + 4, 1] = float("inf")
    out = run_attention(s)
    sees = torch.tensor([bool(int(m.mask[i, 0]) >> 4 & 1) for i in range(12)])
    assert 0 < int(sees.sum()) < 12
    assert torch.equal(out[~sees], clean[~sees]) and bool((out[sees][:, :, 1] == float("inf")).all())


@pytest.mark.gpu
def test_attention_strides_out_and_rows_behind():
    s = make_attention(24, 2, 128, 128, [5, 18], [90, 300], seed=7, device="cuda")
    o, a = attention_oracle(s)
    T = s["q"].shape[0]
    wide = torch.full((T, 24, 3, 128), float("nan"), dtype=torch.bfloat16, device="cuda")   # q inside a fused qkv row
    wide[:, :, 1] = s["q"]
    meta = s["meta"]
    # three more rows behind the last sequence
    q = torch.cat([wide, torch.full_like(wide[:3], float("nan"))])[:, :, 1]
    meta.mask = torch.cat([meta.mask, torch.full_like(meta.mask[:3], -1)])
    meta.depth = torch.cat([meta.depth, meta.depth[:3]])
    bt = torch.full((2, 12), 10 ** 6, dtype=torch.int32, device="cuda")    # a table of a larger stride
    bt[:, 3:3 + meta.block_table.shape[1]] = meta.block_table
    meta.block_table = bt[:, 3:3 + meta.block_table.shape[1]]
    for splits in (1, 4):
        meta.num_splits = splits
        out = torch.full((T + 3, 24, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        ws = torch.empty(4 * (T + 3) * 24 * 130, device="cuda")
        r = tree.tree_attention(q, s["k"], s["v"], meta, out=out, workspace=ws)
        assert r.data_ptr() == out.data_ptr() and (out[T:] == 7.0).all()
        check_attention(s, out[:T], o, a)


@pytest.mark.gpu
def test_attention_long_context_large_tree():
    """A long context in shuffled pages against an oracle over all of it."""
    for fp8 in (False, True):
        s = make_attention(12, 1, 128, 128, [64], [9000], fp8=fp8, seed=8, device="cuda")
        check_attention(s, run_attention(s))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_attention_of_the_largest_tree(fp8):
    """1024 nodes (32 mask words), several row tiles and heads of both kinds of grouping."""
    for Hq, Hk, lens in ((2, 1, [1024]), (3, 1, [1000, 1, 130])):
        s = make_attention(Hq, Hk, 64, 64, lens, [100, 0, 63][:len(lens)], fp8=fp8, seed=12, device="cuda")
        check_attention(s, run_attention(s))


@pytest.mark.gpu
def test_attention_large_scores_keep_the_maximum():
    """Scores that climb by far more than 2^8 between pages: the running maximum moves."""
    for fp8 in (False, True):
        s = make_attention(8, 2, 128, 128, [10], [500], fp8=fp8, seed=9, device="cuda")
        ramp = torch.linspace(0.1, 6.0, 512, device="cuda")
        kf = s["k"].float()
        for t in range(510):
            kf[int(s["meta"].block_table[0, t // PAGE]), :, t % PAGE] *= ramp[t]
        s["k"] = kf.clamp(-448, 448).to(s["k"].dtype)
        # scores reach |s| = 40: their 32-bit error of 128 terms is below 2^-13 of it, within the bound
        check_attention(s, run_attention(s))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_raises_the_maximum_at_every_tile(shape, monkeypatch):
    """Scores that climb by about 0.06 a key: 2^11 over 128 keys, so every tile rescales what the tiles before left.
    They reach 75, a 32-bit error of 75 * 2^-21 in the worst case: below the 2^-12 of the bound."""
    Hq, Hk, D, Dv, fp8 = shape
    s = make_attention(Hq, Hk, D, Dv, [20, 3], [1200, 500], fp8=fp8, seed=15, device="cuda")
    m, q, kf = s["meta"], s["q"], s["k"].float()
    q[:, :, 0] = 128.0
    for b in range(2):
        for t in range(int(m.kv_len[b])):
            kf[int(m.block_table[b, t // PAGE]), :, t % PAGE, 0] = 0.06 * t * D ** 0.5 / 128 / s["ks"]
    s["k"] = kf.to(s["k"].dtype)
    assert torch.isfinite(s["k"].float()).all()
    o, a = attention_oracle(s)
    plan = tree.tree_plan
    for splits in (1, 2):
        m.num_splits = splits
        for tiles in (1, 2) if Dv <= 128 else (1,):
            monkeypatch.setattr(tree, "tree_plan", lambda *x: (tiles, plan(*x)[1]))
            check_attention(s, run_attention(s), o, a)
    N.check_status()


# ---------------------------------------------------------------- verification
def verify_oracle(probs, tokens, parents, q_start, P, ua, ud, draft=None, target=None):
    par, tok, qs = parents.tolist(), tokens.tolist(), q_start.tolist()
    acc, paths, toks, last = [], [], [], []
    for b in range(len(qs) - 1):
        q0, n = qs[b], qs[b + 1] - qs[b]
        if n == 0:
            acc.append(0), paths.append([-1] * P), toks.append([-1] * P), last.append(-1)
            continue
        at, path, out = 0, [0], []
        while True:
            kids = [i for i in range(at + 1, n) if par[q0 + i] == at]
            took = None
            if target is None:
                row = probs[q0 + at].double()
                w = torch.where(row > 0, row, 0.0)
                z, dead = 1.0, set()
                d = torch.where(draft[q0 + at] > 0, draft[q0 + at].double(), 0.0) if draft is not None else None
            for c in kids:
                x, u = tok[q0 + c], float(ua[q0 + c]) if ua is not None else 0
                inside = 0 <= x and (target is not None or x < probs.shape[1])
                if target is not None:
                    hit = x == int(target[q0 + at])
                elif draft is None:
                    hit = inside and x not in dead and bool(row[x] >= 0) and u * z < float(w[x])
                else:
                    hit = inside and u * float(d[x]) * z < float(w[x])
                if hit:
                    took = c
                    break
                if target is None and draft is None and inside:
                    if x not in dead:
                        z -= float(w[x])
                    dead.add(x)
                    w[x] = 0.0
                elif target is None and draft is not None:
                    w = torch.clamp(w / z - d, min=0.0)
                    z = float(w.sum())
                    z = z if z > 0 else 1.0
            if took is None:
                break
            at = took
            path.append(took)
            out.append(tok[q0 + took])
        if target is not None:
            x = int(target[q0 + at])
        else:
            if not float(w.sum()) > 0:
                w = torch.where(row > 0, row, 0.0)
            x, run, lim = 0, 0.0, float(ud[b]) * float(w.sum())
            pos = torch.nonzero(w > 0)[:, 0]
            if len(pos):
                hit = torch.nonzero(w.cumsum(0)[pos] > lim)
                x = int(pos[hit[0, 0]]) if len(hit) else int(pos[-1])
        acc.append(len(path) - 1)
        paths.append(path + [-1] * (P - len(path)))
        toks.append(out + [x] + [-1] * (P - len(out) - 1))
        last.append(q0 + at)
    return i32(acc), i32(paths), i32(toks), i32(last)


def same_verdict(v, want):
    for got, w, name in zip((v.accepted, v.path, v.tokens, v.last_row), want, ("accepted", "path", "tokens", "last")):
        assert torch.equal(got.cpu(), w), (name, got.cpu(), w)


def verify_inputs(lens, V, mode, seed, dtype=torch.float32, sharp=2.0):
    g = torch.Generator().manual_seed(seed)
    par, qs = random_trees(lens, seed)
    T = int(qs[-1])
    logits = sharp * torch.randn(T, V, generator=g)
    probs = torch.softmax(logits, -1).to(dtype)
    guess = torch.softmax(logits + 0.5 * torch.randn(T, V, generator=g), -1)
    seq = torch.repeat_interleave(torch.arange(len(lens)), i32(lens).long())
    row = (qs[seq] + par.clamp(min=0)).long()
    draft = None
    if mode == "draft":
        tokens = torch.multinomial(guess[row], 1, generator=g)[:, 0].to(torch.int32)
        draft = guess.to(dtype)
    else:       # likely tokens, repeats among siblings on purpose
        top = guess.topk(min(4, V), -1).indices
        tokens = top[row, torch.randint(0, min(4, V), (T,), generator=g)].to(torch.int32)
    return dict(probs=probs, tokens=tokens, parents=par, q_start=qs, max_nodes=max(lens),
                u_accept=torch.rand(T, generator=g), u_draw=torch.rand(len(lens), generator=g), draft_probs=draft)


def run_verify(s, device):
    return tree.verify_tree(**{k: v.to(device) if isinstance(v, torch.Tensor) else v for k, v in s.items()})


def oracle_of(s):
    return verify_oracle(s["probs"].float(), s["tokens"], s["parents"], s["q_start"], s["max_nodes"], s["u_accept"],
                         s["u_draw"], None if s["draft_probs"] is None else s["draft_probs"].float())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mode", ["point", "draft"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 11, 500, 4097, 20003, 33024])
def test_verify(device, mode, dtype, V):
    for seed, lens in enumerate([[1], [6], [3, 0, 26, 1], [61, 12, 40]]):
        s = verify_inputs(lens, V, mode, seed, dtype)
        same_verdict(run_verify(s, device), oracle_of(s))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["point", "draft"])
def test_verify_vocabulary_of_a_model(mode):
    for dtype, V in ((torch.float32, 151552), (torch.bfloat16, 151552), (torch.float32, 152577)):
        s = verify_inputs([5, 8, 1, 3], V, mode, 11, dtype, sharp=0.5)
        same_verdict(run_verify(s, "cuda"), oracle_of(s))
    s = verify_inputs([1] * 40, 30000, mode, 12, sharp=0.1)      # flat rows: every sum counts
    same_verdict(run_verify(s, "cuda"), oracle_of(s))


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["point", "draft"])
@pytest.mark.parametrize("V", [9000, 20003, 70001])
def test_verify_many_sequences_and_many_rejections(mode, V):
    """More sequences than clusters of 8 CTAs run at a time; nodes whose children are rejected one after another."""
    s = verify_inputs([9, 4, 1, 12] * 6, V, mode, 13, sharp=1.0)
    same_verdict(run_verify(s, "cuda"), oracle_of(s))
    s = verify_inputs([40, 3, 25], V, mode, 14, sharp=1.5)
    s["parents"] = i32([-1] + [0] * 39 + [-1, 0, 0] + [-1] + [0] * 24)
    s["u_accept"].fill_(0.9995)
    v = run_verify(s, "cuda")
    same_verdict(v, oracle_of(s))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("mode", ["point", "draft"])
def test_verify_edges(device, mode):
    """All-rejecting and all-accepting numbers, u at both ends, rows without mass, NaN, negative and
    infinite entries, drafts outside the vocabulary, strided rows."""
    for V in (7, 9001):
        s = verify_inputs([6, 9, 4, 5, 1], V, mode, 20, sharp=1.0)
        for ua, ud in ((0.0, 0.0), (1.0 - 2 ** -24, 1.0 - 2 ** -24), (0.5, 2.0), (float("nan"), float("nan"))):
            s["u_accept"].fill_(ua)
            s["u_draw"].fill_(ud)
            same_verdict(run_verify(s, device), oracle_of(s))
        s = verify_inputs([6, 9, 4, 5, 1], V, mode, 21, sharp=1.0)
        s["tokens"][3], s["tokens"][8], s["tokens"][12] = -1, V, 2 ** 31 - 1
        s["probs"][0] = 0.0
        s["probs"][6] = float("nan")
        s["probs"][15, 1:] = -1.0
        s["probs"][24, 3] = float("inf")
        if mode == "draft":
            s["draft_probs"][7] = s["probs"][7]        # q = p: a rejection leaves nothing
            s["draft_probs"][15, 2] = float("nan")
        for k in range(4):
            s["u_accept"] = torch.rand(25, generator=torch.Generator().manual_seed(k))
            same_verdict(run_verify(s, device), oracle_of(s))
        wide = torch.full((25, V + 5), 9.0)
        wide[:, 2:2 + V] = s["probs"]
        s["probs"] = wide[:, 2:2 + V]
        t = {k: v.to(device) if isinstance(v, torch.Tensor) and k != "probs" else v for k, v in s.items()}
        t["probs"] = wide.to(device)[:, 2:2 + V]
        same_verdict(tree.verify_tree(**t), oracle_of(s))


@pytest.mark.parametrize("device", DEVICES)
def test_verify_chain_agrees_with_the_chain_rule(device):
    """A chain of drafts chosen outright: draft j is kept while u_j < p_j(d_j)."""
    g = torch.Generator().manual_seed(3)
    probs = torch.softmax(torch.randn(5, 50, generator=g), -1)
    toks = torch.cat([i32([0]), probs[:4].argmax(-1).to(torch.int32)])
    u = torch.rand(5, generator=g) * 0.2
    v = tree.verify_tree(probs.to(device), toks.to(device), i32([-1, 0, 1, 2, 3], device), i32([0, 5], device), 5,
                         u.to(device), torch.tensor([0.5], device=device))
    a = 0
    while a < 4 and u[a + 1] < probs[a, toks[a + 1]]:
        a += 1
    assert int(v.accepted[0]) == a and v.tokens[0, :a].tolist() == toks[1:a + 1].tolist()


def test_verify_emits_the_target_distribution():
    """One root with three drafted children, many uniform numbers: the first emitted token follows p
    for drafts chosen outright and for drafts drawn from q.  The frequency of 20000 tries of a
    token of probability p is off by more than 5 sqrt(p (1 - p) / 20000) once in 10^6."""
    n, V = 20000, 5
    g = torch.Generator().manual_seed(0)
    p, q = torch.tensor([0.4, 0.3, 0.15, 0.1, 0.05]), torch.tensor([0.1, 0.5, 0.2, 0.1, 0.1])
    kids = 3
    for mode in ("point", "draft"):
        counts = torch.zeros(V)
        ua, ud = torch.rand(n, kids + 1, generator=g).double(), torch.rand(n, generator=g).double()
        drawn = torch.multinomial(q, n * kids, replacement=True, generator=g).view(n, kids)
        for t in range(n):
            w, z = p.double(), 1.0
            x = None
            for c in range(kids):
                tok = int(drawn[t, c]) if mode == "draft" else c
                share = float(q[tok]) * z if mode == "draft" else z
                if ua[t, c + 1] * share < w[tok]:
                    x = tok
                    break
                if mode == "draft":
                    w = torch.clamp(w / z - q.double(), min=0)
                    z = float(w.sum())
                else:
                    z -= float(w[tok])
                    w = w.clone()
                    w[tok] = 0
            if x is None:
                x = int((w.cumsum(0) <= ud[t] * w.sum()).sum())
            counts[x] += 1
            if t < 300:      # the operator makes the same choices
                v = tree.verify_tree(p.repeat(kids + 1, 1),
                                     i32([0] + (drawn[t].tolist() if mode == "draft" else list(range(kids)))),
                                     i32([-1] + [0] * kids), i32([0, kids + 1]), kids + 1, ua[t].float(),
                                     ud[t:t + 1].float(), q.repeat(kids + 1, 1) if mode == "draft" else None)
                assert int(v.tokens[0, 0]) == x
        assert ((counts / n - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lens", [[1], [5, 0, 9], [64, 33, 2], [1024, 40]])
def test_verify_greedy(device, lens):
    par, qs = random_trees(lens, 5)
    g = torch.Generator().manual_seed(6)
    T = int(qs[-1])
    toks = torch.randint(0, 3, (T,), generator=g, dtype=torch.int32)
    tgt = torch.randint(0, 3, (T,), generator=g, dtype=torch.int32)
    v = tree.verify_tree_greedy(tgt.to(device), toks.to(device), par.to(device), qs.to(device), max(lens))
    same_verdict(v, verify_oracle(None, toks, par, qs, max(lens), None, None, target=tgt))
    assert int(v.accepted.max()) > 0 or max(lens) == 1


# ---------------------------------------------------------------- commit
def commit_inputs(L, Hk, D, Dv, lens, ctx, fp8, seed):
    s = make_attention(Hk, Hk, D, Dv, lens, ctx, fp8=fp8, seed=seed)
    g = torch.Generator().manual_seed(seed)
    nb = s["k"].shape[0]
    t = FP8 if fp8 else torch.bfloat16
    k = torch.randn(L, nb, Hk, PAGE, D, generator=g).to(t)
    v = torch.randn(*((L, nb, Hk, Dv, PAGE) if fp8 else (L, nb, Hk, PAGE, Dv)), generator=g).to(t)
    par, qs = random_trees(lens, seed)
    P = max(lens)
    path, acc = torch.full((len(lens), P), -1, dtype=torch.int32), []
    for b, n in enumerate(lens):
        if n == 0:
            acc.append(0)
            continue
        leaf = n - 1 - int(torch.randint(0, max(1, n // 3), (1,), generator=g))
        up = family(par[qs[b]:qs[b + 1]].tolist(), leaf)[::-1]
        path[b, :len(up)] = i32(up)
        acc.append(len(up) - 1)
    m = s["meta"]
    return k, v, path, i32(acc), qs, m.kv_len, m.block_table


def commit_oracle(k, v, path, acc, qs, kv_len, bt):
    fp8 = k.dtype == FP8
    k, v = k.double(), v.double()
    k0, v0 = k.clone(), v.clone()
    for b in range(len(acc)):
        n = int(qs[b + 1] - qs[b])
        ctx = int(kv_len[b]) - n
        for j in range(1, int(acc[b]) + 1):
            f, t = ctx + int(path[b, j]), ctx + j
            fb, tb = int(bt[b, f // PAGE]), int(bt[b, t // PAGE])
            k[:, tb, :, t % PAGE] = k0[:, fb, :, f % PAGE]
            if fp8:
                v[:, tb, :, :, t % PAGE] = v0[:, fb, :, :, f % PAGE]
            else:
                v[:, tb, :, t % PAGE] = v0[:, fb, :, f % PAGE]
    return k, v


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("L,Hk,D,Dv,lens,ctx", [(1, 2, 64, 64, [1], [5]), (3, 2, 64, 64, [9, 0, 30], [60, 4, 120]),
                                               (2, 8, 128, 128, [61, 64], [10, 63]), (70, 1, 64, 64, [12], [0]),
                                               (2, 4, 192, 128, [20], [50]), (1, 1, 64, 64, [1000, 3], [33, 64])])
def test_commit(device, fp8, L, Hk, D, Dv, lens, ctx):
    if fp8 and D != Dv:
        D = Dv
    k, v, path, acc, qs, kl, bt = commit_inputs(L, Hk, D, Dv, lens, ctx, fp8, 31)
    k1, v1 = commit_oracle(k, v, path, acc, qs, kl, bt)
    idx = [t.to(device) for t in (path, acc, qs, kl, bt)]
    ks, vs = k.to(device), v.to(device)
    kl_, vl_ = [x.clone() for x in ks], [x.clone() for x in vs]
    tree.commit_tree(ks, vs, *idx)                       # layers stacked in one tensor
    assert torch.equal(ks.cpu().double(), k1) and torch.equal(vs.cpu().double(), v1)
    tree.commit_tree(kl_, vl_, *idx)                     # one tensor per layer
    assert torch.equal(torch.stack(kl_).cpu().double(), k1) and torch.equal(torch.stack(vl_).cpu().double(), v1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fp8", [False, True])
def test_commit_moves_nothing_outside_the_tree(device, fp8):
    """accepted beyond the path, entries that do not rise, lie outside the tree or name no page."""
    k, v, path, acc, qs, kl, bt = commit_inputs(2, 2, 64, 64, [6, 6, 6], [60, 61, 3], fp8, 32)
    path[0] = i32([0, 1, 0, 9, -1, -1])
    path[1] = i32([0, 1, 2, 3, 4, 5])
    path[2] = i32([0, 2, 1, 2 ** 30, -5, 6])
    acc[:] = i32([5, 100, 5])
    k1, v1 = k.clone(), v.clone()
    p = int(bt[2, 0])
    if fp8:
        k, v, k1, v1 = (x.view(torch.uint8) for x in (k, v, k1, v1))
        v1[:, p, :, :, 4] = v[:, p, :, :, 5]
    else:
        v1[:, p, :, 4] = v[:, p, :, 5]
    k1[:, p, :, 4] = k[:, p, :, 5]                     # the one good entry: node 2 to slot 1
    kd, vd = k.to(device), v.to(device)
    t = FP8 if fp8 else torch.bfloat16
    tree.commit_tree(kd.view(t), vd.view(t), *[x.to(device) for x in (path, acc, qs, kl, bt)])
    assert torch.equal(kd.cpu(), k1) and torch.equal(vd.cpu(), v1)
    # a path that falls back after reaching the second page: the first move is good, the second is none
    k, v, path, acc, qs, kl, bt = commit_inputs(1, 2, 64, 64, [50], [40], fp8, 33)
    path[0, :3] = i32([0, 45, 2])
    acc[:] = 2
    path[0, 3:] = -1
    one = acc.clone().fill_(1)
    k1, v1 = commit_oracle(k, v, path, one, qs, kl, bt)
    kd, vd = k.to(device), v.to(device)
    tree.commit_tree(kd, vd, *[x.to(device) for x in (path, acc, qs, kl, bt)])
    assert torch.equal(kd.cpu().double(), k1) and torch.equal(vd.cpu().double(), v1)


def commit_by_slots(k, v, path, acc, qs, kl, bt):
    """commit_oracle for tables with columns and ids that name no page: a move needs both of its slots."""
    fp8 = k.dtype == FP8
    k1, v1 = (x.view(torch.uint8).clone() if fp8 else x.clone() for x in (k, v))
    k0, v0 = k1.clone(), v1.clone()
    for b in range(len(acc)):
        n = int(qs[b + 1] - qs[b])
        ctx = int(kl[b]) - n
        slot = {i: (int(bt[b, (ctx + i) // PAGE]), (ctx + i) % PAGE) for i in range(n)
                if ctx >= 0 and (ctx + i) // PAGE < bt.shape[1] and 0 <= int(bt[b, (ctx + i) // PAGE]) < k.shape[1]}
        for j in range(1, int(acc[b]) + 1):
            f, t = slot.get(int(path[b, j])), slot.get(j)
            if f is None or t is None:
                continue
            k1[:, t[0], :, t[1]] = k0[:, f[0], :, f[1]]
            if fp8:
                v1[:, t[0], :, :, t[1]] = v0[:, f[0], :, :, f[1]]
            else:
                v1[:, t[0], :, t[1]] = v0[:, f[0], :, f[1]]
    return k1, v1


BAD_PAGES = ["none", "first", "second", "beyond", "columns", "short"]


def commit_with_bad_pages(device, fp8, bad):
    """Trees over two and three pages, of which one is not there."""
    k, v, path, acc, qs, kl, bt = commit_inputs(2, 2, 64, 64, [60, 130, 9], [30, 40, 62], fp8, 34)
    for b, n in enumerate([60, 130, 9]):                     # every second node is accepted: all of them move
        path[b] = -1
        path[b, :(n + 1) // 2] = torch.arange(0, n, 2, dtype=torch.int32)
        acc[b] = (n + 1) // 2 - 1
    if bad in ("first", "second", "beyond"):
        bt[:, {"first": 0, "second": 1, "beyond": 2}[bad]] = i32([-1, k.shape[1], 10 ** 6])
    elif bad == "columns":
        bt = bt[:, :1].contiguous()
    elif bad == "short":                                     # padding: fewer keys than nodes
        kl = i32([0, 129, 3])
    k1, v1 = commit_by_slots(k, v, path, acc, qs, kl, bt)
    assert bad in ("columns", "short") or not torch.equal(k1, k.view(torch.uint8) if fp8 else k)
    kd, vd = k.to(device), v.to(device)
    tree.commit_tree(kd, vd, *[x.to(device) for x in (path, acc, qs, kl, bt)])
    if fp8:
        kd, vd = kd.view(torch.uint8), vd.view(torch.uint8)
    assert torch.equal(kd.cpu(), k1) and torch.equal(vd.cpu(), v1)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("bad", BAD_PAGES)
def test_commit_cpu_moves_nothing_from_or_to_pages_that_are_not_there(fp8, bad):
    commit_with_bad_pages("cpu", fp8, bad)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("bad", BAD_PAGES)
def test_commit_moves_k_and_v_alike_beside_pages_that_are_not_there(fp8, bad):
    """fp8: V lies transposed and takes another way than K; without the first page it was left where it lay."""
    commit_with_bad_pages("cuda", fp8, bad)


# ---------------------------------------------------------------- together
def two_layer_model(Hq, Hk, D, V, seed, device):
    g = torch.Generator().manual_seed(seed)
    H = Hq * D
    r = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(torch.bfloat16).to(device)  # noqa: E731
    return dict(emb=(torch.randn(V, H, generator=g)).to(torch.bfloat16).to(device), head=r(V, H),
                layers=[(r((Hq + 2 * Hk) * D, H), r(H, H)) for _ in range(2)], Hq=Hq, Hk=Hk, D=D,
                rope=basic.rope_cache(D, 512, 10000.0, device))


def forward(m, ids, pos, slots, caches, attend):
    h = m["emb"][ids.long()].float()
    Hq, Hk, D = m["Hq"], m["Hk"], m["D"]
    for (wqkv, wo), (kc, vc) in zip(m["layers"], caches):
        x = h / h.pow(2).mean(-1, keepdim=True).sqrt()
        qkv = (x @ wqkv.float().t()).to(torch.bfloat16).contiguous()
        T = qkv.shape[0]
        q = qkv[:, :Hq * D].view(T, Hq, D)
        k = qkv[:, Hq * D:(Hq + Hk) * D].view(T, Hk, D)
        v = qkv[:, (Hq + Hk) * D:].view(T, Hk, D)
        basic.rope_and_cache(q, k, v, pos, m["rope"], D, True, slot_mapping=slots, k_cache=kc, v_cache=vc)
        h = h + attend(q, kc, vc).reshape(T, Hq * D).float() @ wo.float().t()
    return h @ m["head"].float().t()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("sampled", [False, True])
def test_speculative_steps_match_one_token_at_a_time(device, sampled):
    """Trees of guesses (some right) verified and committed step by step give the tokens and the
    cache that decoding one token at a time gives.  Sampled: u_accept = 0 accepts any first child,
    and a chain-less root with u_draw = 0 emits the smallest token of positive probability."""
    V, Hq, Hk, D = 97, 4, 2, 64
    m = two_layer_model(Hq, Hk, D, V, 1, device)
    nb = 8
    new = lambda: [(torch.zeros(nb, Hk, PAGE, D, dtype=torch.bfloat16, device=device),   # noqa: E731
                    torch.zeros(nb, Hk, PAGE, D, dtype=torch.bfloat16, device=device)) for _ in range(2)]
    bt = i32([[5, 2, 7, 0]], device)
    slot_of = lambda t: int(bt[0, t // PAGE]) * PAGE + t % PAGE    # noqa: E731
    prompt = [3, 14, 15, 92, 65, 35] * 10                              # 60 tokens: the tree crosses a page
    steps = 14

    def nodes(caches, ctx, ids, parents):
        n = len(ids)
        par, qs = i32(parents, device), i32([0, n], device)
        mask, depth = tree.tree_mask(par, qs, n)
        meta = TreeMetadata(num_seqs=1, q_start=qs, kv_len=i32([ctx + n], device), block_table=bt, mask=mask,
                            depth=depth, max_nodes=n, max_kv_len=ctx + n)
        logits = forward(m, i32(ids, device), (depth + ctx).to(torch.int32),
                         i32([slot_of(ctx + i) for i in range(n)], device), caches,
                         lambda q, k, v: tree.tree_attention(q, k, v, meta))
        return logits, par, qs, meta

    # one token at a time
    plain = new()
    seq = list(prompt)
    nodes(plain, 0, seq[:-1], list(range(-1, len(seq) - 2)))
    for _ in range(steps):
        logits, *_ = nodes(plain, len(seq) - 1, seq[-1:], [-1])
        seq.append(int(logits[0].argmax()))
    want = seq[len(prompt):]
    # trees: node 1 a wrong guess, 2 the right one, 3 below the wrong one, 4 right below 2, 5 wrong below 4
    spec = new()
    got = list(prompt)
    nodes(spec, 0, got[:-1], list(range(-1, len(got) - 2)))
    taken = []
    while len(got) < len(prompt) + steps:
        at = len(got) - len(prompt)
        nxt = (want + [0] * 3)[at:at + 3]
        wrong = [(x + 1) % V for x in nxt]
        ids, parents = [got[-1], wrong[0], nxt[0], nxt[1], nxt[1], wrong[2]], [-1, 0, 0, 1, 2, 4]
        ctx = len(got) - 1
        logits, par, qs, meta = nodes(spec, ctx, ids, parents)
        if sampled:   # a distribution that puts all on the greedy token
            probs = torch.nn.functional.one_hot(logits.argmax(-1), V).float()
            ver = tree.verify_tree(probs, i32(ids, device), par, qs, 6, torch.rand(6, device=device),
                                   torch.rand(1, device=device))
        else:
            ver = tree.verify_tree_greedy(logits.argmax(-1).to(torch.int32), i32(ids, device), par, qs, 6)
        tree.commit_tree([k for k, _ in spec], [v for _, v in spec], ver.path, ver.accepted, qs, meta.kv_len, bt)
        a = int(ver.accepted[0])
        taken.append(a)
        got += ver.tokens[0, :a + 1].tolist()
    assert max(taken) == 2, "the right branch is accepted"
    assert got[len(prompt):len(prompt) + steps] == want
    # the committed keys are those of the same tokens one at a time (bf16 roundings of other batches apart)
    for (k0, v0), (k1, v1) in zip(plain, spec):
        for t in range(len(prompt) + steps - 1):
            pg, off = int(bt[0, t // PAGE]), t % PAGE
            for x, y in ((k0, k1), (v0, v1)):
                a, b = x[pg, :, off].float(), y[pg, :, off].float()
                assert (a - b).abs().max() <= 2 ** -5 * a.abs().max()


# ---------------------------------------------------------------- streams, graphs
@pytest.mark.gpu
def test_step_in_a_graph_and_on_two_streams():
    """The four calls captured once and replayed on new inputs; two captured graphs and two streams
    at a time give what one call at a time gives."""
    sets = []
    for seed in (40, 41):
        s = make_attention(24, 2, 128, 128, [9, 16], [300, 2100], seed=seed, device="cuda")
        par, qs = random_trees([9, 16], seed, "cuda")
        ver = {k: v.cuda() if isinstance(v, torch.Tensor) else v
               for k, v in verify_inputs([9, 16], 30000, "draft", seed).items()}
        kc, vc = s["k"].clone()[None], s["v"].clone()[None]

        def step(s=s, par=par, qs=qs, ver=ver, kc=kc, vc=vc):
            mask, depth = tree.tree_mask(par, qs, 16)
            o = run_attention(s)
            v = tree.verify_tree(**ver)
            kc.copy_(s["k"][None]), vc.copy_(s["v"][None])
            tree.commit_tree(kc, vc, v.path, v.accepted, qs, s["meta"].kv_len, s["meta"].block_table)
            return [mask, depth, o, v.accepted, v.path, v.tokens, v.last_row, kc, vc]
        sets.append((step, ver))
    want = [[t.clone() for t in step()] for step, _ in sets]
    graphs = []
    for step, _ in sets:
        s0 = torch.cuda.Stream()
        s0.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s0):
            step()
        torch.cuda.current_stream().wait_stream(s0)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in sets]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(20):                                       # both graphs at once
        for (g, _), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), w in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w))
    got = [None, None]
    for _ in range(20):                                       # eager calls on two streams
        for i, ((step, _), st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i] = step()
    torch.cuda.synchronize()
    for out, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(out, w))
    # a replay reads the inputs of the day
    ver = sets[0][1]
    ver["u_draw"].fill_(0.999)
    graphs[0][0].replay()
    v = tree.verify_tree(**ver)
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1][5], v.tokens)
    N.check_status()


# ---------------------------------------------------------------- refusals
def test_refusals():
    s = make_attention(4, 2, 64, 64, [5, 3], [10, 70], seed=50)
    m, q, k, v = s["meta"], s["q"], s["k"], s["v"]
    import dataclasses

    def no(what, f):
        with pytest.raises(ValueError, match=what):
            f()
    no("max_nodes", lambda: tree.tree_mask(i32([-1]), i32([0, 1]), 0))
    no("max_nodes", lambda: tree.tree_mask(i32([-1]), i32([0, 1]), 1025))
    no("parents", lambda: tree.tree_mask(torch.zeros(3, dtype=torch.int64), i32([0, 3]), 3))
    no("mask", lambda: tree.tree_mask(i32([-1]), i32([0, 1]), 40, i32([[0]])))
    no("do not match", lambda: tree.tree_attention(q, k, v[:, :1].contiguous(), m))
    no("K and a V", lambda: tree.tree_attention(q, k, None, m))
    no("divide", lambda: tree.tree_attention(q[:, :3].contiguous(), k, v, m))
    no("depths", lambda: tree.tree_attention(q, k, v, dataclasses.replace(m, depth=None), window=8))
    no("too narrow", lambda: tree.tree_attention(q, k, v, dataclasses.replace(m, max_nodes=33)))
    no("kv_len", lambda: tree.tree_attention(q, k, v, dataclasses.replace(m, kv_len=m.kv_len.long())))
    no("mask", lambda: tree.tree_attention(q, k, v, dataclasses.replace(m, mask=m.mask[:-1])))
    no("sinks", lambda: tree.tree_attention(q, k, v, m, sinks=torch.zeros(3)))
    no("out", lambda: tree.tree_attention(q, k, v, m, out=torch.zeros(8, 4, 64)))
    t, p = i32([0, 1, 2]), i32([-1, 0, 0])
    pr, u = torch.full((3, 4), 0.25), torch.rand(3)
    no("u_draw", lambda: tree.verify_tree(pr, t, p, i32([0, 3]), 3, u, u))
    no("probs", lambda: tree.verify_tree(pr.double(), t, p, i32([0, 3]), 3, u, u[:1]))
    no("draft_probs", lambda: tree.verify_tree(pr, t, p, i32([0, 3]), 3, u, u[:1], pr[:, :3]))
    no("tokens", lambda: tree.verify_tree(pr, t.long(), p, i32([0, 3]), 3, u, u[:1]))
    no("target", lambda: tree.verify_tree_greedy(t[:2], t, p, i32([0, 3]), 3))
    c = (i32([[0, 1]]), i32([1]), i32([0, 2]), i32([5]), i32([[0]]))
    no("as many", lambda: tree.commit_tree([k], [], *c))
    no("alike", lambda: tree.commit_tree([k, k[:1]], [v, v], *c))
    no("64 tokens", lambda: tree.commit_tree([k[:, :, :32]], [v[:, :, :32]], *c))
    no("contiguous", lambda: tree.commit_tree([k.transpose(0, 1).contiguous().transpose(0, 1)], [v], *c))


@pytest.mark.gpu
def test_refusals_gpu():
    s = make_attention(4, 2, 64, 64, [5, 3], [10, 70], seed=51, device="cuda")
    m, q, k, v = s["meta"], s["q"], s["k"], s["v"]

    def no(what, f):
        with pytest.raises(ValueError, match=what):
            f()
    no("head sizes", lambda: tree.tree_attention(torch.zeros(8, 4, 128, dtype=torch.bfloat16, device="cuda"),
                                                 torch.zeros(2, 2, 64, 128, dtype=torch.bfloat16, device="cuda"), v[:2], m))
    no("bfloat16", lambda: tree.tree_attention(q.float(), k, v, m))
    no("bfloat16", lambda: tree.tree_attention(q, k.half(), v.half(), m))
    no("64 tokens", lambda: tree.tree_attention(q, k[:, :, :32].contiguous(), v[:, :, :32].contiguous(), m))
    no("16-byte", lambda: tree.tree_attention(torch.zeros(8 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:]
                                              .view(8, 4, 64), k, v, m))
    no("on cuda", lambda: tree.tree_attention(q, k.cpu(), v.cpu(), m))
    # sizes that the device finds wrong are told: rows past the tensors, more nodes than max_nodes, keys
    # past the table
    import dataclasses

    def told():
        with pytest.raises(RuntimeError, match="bounds"):
            N.check_status()
    for change in (dict(q_start=i32([0, 5, 9], "cuda")), dict(q_start=i32([0, 5, 3], "cuda")), dict(max_nodes=4),
                   dict(block_table=m.block_table[:, :1])):
        tree.tree_attention(q, k, v, dataclasses.replace(m, **change))
        told()
    par, tok = random_trees([5, 3], 2, "cuda")[0], torch.ones(8, dtype=torch.int32, device="cuda")
    pr, u = torch.full((8, 20), 0.05, device="cuda"), torch.zeros(8, device="cuda")
    for qs in (i32([0, 5, 9], "cuda"), i32([-1, 3], "cuda"), i32([0, 5, 3], "cuda")):
        B = len(qs) - 1
        tree.tree_mask(par, qs, 5)
        told()
        v1 = tree.verify_tree_greedy(tok, tok, par, qs, 5)
        told()
        v2 = tree.verify_tree(pr, tok, par, qs, 5, u, u[:B])
        told()
        for vd in (v1, v2):                      # such a sequence has no nodes
            assert int(vd.last_row[B - 1]) == -1 and int(vd.accepted[B - 1]) == 0
            assert bool((vd.path[B - 1] == -1).all()) and bool((vd.tokens[B - 1] == -1).all())
    # a tree larger than max_nodes is cut and reported
    par, qs = random_trees([9], 1, "cuda")
    tree.tree_mask(par, qs, 4)
    with pytest.raises(RuntimeError, match="bounds"):
        N.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("shape", SHAPES[:6])
def test_attention_goes_on_beside_what_it_leaves_out(shape, splits):
    """A sequence outside the call's tensors is reported and left out.  The other sequences of the call, and calls after
    it whose caller has not asked for the status yet, keep their results although their waits are long."""
    import dataclasses
    Hq, Hk, D, Dv, fp8 = shape
    s = make_attention(Hq, Hk, D, Dv, [12, 3, 9, 12], [6000, 2500, 70, 4000], fp8=fp8, seed=53, device="cuda")
    m = s["meta"]
    m.num_splits = splits
    clean = run_attention(s)
    N.check_status()
    row = lambda t: torch.cat([t, t[:1]])                                     # noqa: E731
    wrong = dataclasses.replace(m, num_seqs=5, q_start=torch.cat([m.q_start, i32([48], "cuda")]), kv_len=row(m.kv_len),
                                block_table=row(m.block_table).contiguous())
    for _ in range(10):
        assert torch.equal(run_attention({**s, "meta": wrong}), clean)
        assert torch.equal(run_attention(s), clean)                           # the report still stands
    with pytest.raises(RuntimeError, match="bounds"):
        N.check_status()
    assert torch.equal(run_attention(s), clean)
    N.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("lens,starts,most,good", [
    ([5, 3], [0, 5, 3], 5, range(5)), ([5, 3], [0, 5, 9], 5, range(5)), ([5, 3], [-1, 5, 8], 5, range(5, 8)),
    ([5, 3], [0, 5, 8], 4, [0, 1, 2, 3, 5, 6, 7]), ([5, 3], [0, 5, 8], 2, [0, 1, 5, 6]), ([3] * 40, None, 2, None)])
def test_attention_leaves_out_only_what_it_reports(lens, starts, most, good, splits):
    """Bounds that fall or lie outside q, and more nodes than max_nodes: the other rows are those of a clean call, the
    rows left out keep what `out` held."""
    import dataclasses
    if starts is None:                                        # more sequences than lanes, each cut
        starts, good = list(range(0, 121, 3)), [3 * b + i for b in range(40) for i in range(2)]
    for Hq, Hk, D, Dv, fp8 in SHAPES[:6]:
        s = make_attention(Hq, Hk, D, Dv, lens, [700 + 3 * b for b in range(len(lens))], fp8=fp8, seed=54, device="cuda")
        m = s["meta"]
        m.num_splits = splits
        clean = run_attention(s)
        N.check_status()
        out = torch.full_like(clean, 7.0)
        ws = torch.full((splits * clean.numel() // Dv * (Dv + 2),), float("nan"), device="cuda")
        wrong = dataclasses.replace(m, q_start=i32(starts, "cuda"), max_nodes=most)
        run_attention({**s, "meta": wrong}, out=out, workspace=ws)
        with pytest.raises(RuntimeError, match="bounds"):
            N.check_status()
        kept = torch.zeros(len(clean), dtype=torch.bool)
        kept[list(good)] = True
        assert torch.equal(out[kept], clean[kept]) and bool((out[~kept] == 7.0).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("splits", [1, 2])
@pytest.mark.parametrize("window,sinks", [(0, False), (3, True)])
def test_attention_of_a_padded_batch(device, splits, window, sinks):
    """Padding sequences: no nodes, or nodes without keys, whose rows are zero; with fewer keys than nodes the keys are
    the last nodes'.  The other sequences keep their rows."""
    s = make_attention(4, 2, 64, 64, [9, 4, 0, 5, 6], [70, 0, 0, 130, 0], seed=55, device=device, window=window, sinks=sinks)
    m = s["meta"]
    m.num_splits = splits
    clean = run_attention(s)
    m.kv_len[1] = 0
    out = run_attention(s)
    assert bool((out[9:13] == 0).all()) and torch.equal(out[:9], clean[:9]) and torch.equal(out[13:], clean[13:])
    # the last two of sequence 4's six nodes, as a tree whose first four nodes nobody sees
    m.kv_len[4] = 2
    out = run_attention(s)
    k, v, pg = s["k"].clone(), s["v"].clone(), int(m.block_table[4, 0])
    k[pg, :, 4:6], v[pg, :, 4:6] = s["k"][pg, :, :2], s["v"][pg, :, :2]
    m.mask[18:, 0] &= ~0xF
    m.kv_len[4] = 6
    same = run_attention({**s, "k": k, "v": v})
    # check_attention's bound for each of the two, with sum p |v| <= max |v|
    assert (out[18:].float() - same[18:].float()).abs().max() <= (2 ** -6 + 2 ** -11) * v[pg, :, 4:6].float().abs().max()
    assert torch.equal(out[:18], same[:18])
    if device == "cuda":
        N.check_status()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_window_wider_than_any_context(device):
    s = make_attention(4, 2, 64, 64, [9, 4], [70, 300], seed=56, device=device)
    clean = run_attention(s)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 40):
        assert torch.equal(run_attention({**s, "window": window}), clean)


def test_the_attention_entry_refuses_unaligned_tensors():
    """q, out and the workspace are read and written 16 bytes at a time; the entry says so before it starts anything."""
    base = dict(q=256, o=256, ws=256)
    for name in base:
        a = {**base, name: 264}
        with pytest.raises(RuntimeError, match="code -5"):
            N.call_packed("xtu_tree_attention", a["q"], 512, 64, 256, 256, 0, a["o"], 0, 0, 0, 1, 1, 0, 1, 0, 0, 1, 1, 1, 4, 2,
                          64, 64, 1, 1.0, 1.0, 1.0, 0, 1, 2, a["ws"], 0, 0)


@pytest.mark.gpu
def test_attention_refuses_an_unaligned_out():
    s = make_attention(4, 2, 64, 64, [5, 3], [10, 70], seed=52, device="cuda")
    for splits in (1, 2):
        s["meta"].num_splits = splits
        out = torch.zeros(8 * 4 * 64 + 8, dtype=torch.bfloat16, device="cuda")
        for odd in (1, 4):
            with pytest.raises(ValueError, match="16-byte"):
                run_attention(s, out=out[odd:odd + 8 * 4 * 64].view(8, 4, 64))
        check_attention(s, run_attention(s, out=out[8:].view(8, 4, 64)))
