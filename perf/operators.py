"""Measured operators of tree speculation: a step that verifies a tree of drafted tokens.

A decode step may verify a *tree* of drafted tokens per sequence instead of a chain.  Node 0
is the last emitted token, every other node has a parent of lower index, and a node stands
for the continuation that its ancestors spell.  Four operators of ``vllm_xtu_moe_b200.ops.tree``
make up such a step beside the model's own layers:

* ``tree_mask``       parents -> ancestor bit rows and depths,
* ``tree_attention``  the nodes' queries over the paged KV cache (committed context + ancestors),
* ``verify_tree``     acceptance of the drafts against the target's probabilities,
* ``commit_tree``     the accepted path's K / V rows moved behind the committed context.

``run`` computes each in a plain form (elementary torch operations), or, with ``own`` set, by
the framework's call.
"""
import math

import torch

own = False

PAGE = 64                       # tokens per KV-cache block

# (query heads, KV heads, K width, V width) of the repository's model presets
HEADS = {"tiny": (4, 2, 64, 64), "glm": (96, 8, 128, 128), "qwen": (16, 2, 256, 256), "mimo": (64, 8, 192, 128)}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _attn(name, heads, batch, ctx_lo, ctx_hi, nodes, fp8=False, window=0, sinks=False):
    return {"name": name, "op": "attention", "heads": heads, "batch": batch, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi,
            "nodes": nodes, "fp8": fp8, "window": window, "sinks": sinks}


def _verify(name, mode, batch, nodes, vocab, bf16=False):
    return {"name": name, "op": "verify", "mode": mode, "batch": batch, "nodes": nodes, "vocab": vocab, "bf16": bf16}


def _commit(name, heads, layers, batch, nodes, ctx_hi, fp8):
    return {"name": name, "op": "commit", "heads": heads, "layers": layers, "batch": batch, "nodes": nodes,
            "ctx_hi": ctx_hi, "fp8": fp8}


def _mask(name, batch, nodes):
    return {"name": name, "op": "mask", "batch": batch, "nodes": nodes}


def listed():
    return [
        # one short chat with a handful of drafts on the smallest preset: pure latency
        _attn("attn_tiny_b1", "tiny", 1, 100, 100, 5),
        # the repository's headline decode (4 requests, 14.5K prompts) with a small tree
        _attn("attn_glm_b4_n16", "glm", 4, 14500, 14756, 16),
        # the same requests with the usual 60 drafts and the root: the largest attention
        _attn("attn_glm_b4_n61", "glm", 4, 14500, 14756, 61),
        # the same small tree over the fp8 cache
        _attn("attn_glm_fp8_b4_n16", "glm", 4, 14500, 14756, 16, fp8=True),
        # a sliding-window layer with learned sinks: most of the context is out of sight
        _attn("attn_mimo_swa_b8_n26", "mimo", 8, 2000, 8000, 26, window=128, sinks=True),
        # many requests of very different lengths, wide heads
        _attn("attn_qwen_ragged_b16_n9", "qwen", 16, 1, 12001, 9),
        # one sampled request with a chain of 4 greedy drafts
        _verify("verify_chain_b1", "point", 1, 5, 151552),
        # a full batch whose children were drawn from the drafter's own distributions
        _verify("verify_tree_b32", "draft", 32, 26, 151552),
        # the accepted path of 4 requests in every layer's bf16 cache
        _commit("commit_glm_b4", "glm", 46, 4, 16, 150, False),
        # a batch of large trees in fp8 caches (V transposed inside each block)
        _commit("commit_glm_fp8_b16", "glm", 46, 16, 61, 150, True),
        # one small tree
        _mask("mask_b1", 1, 16),
        # a large batch of large trees
        _mask("mask_b64_n200", 64, 200),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "verify", "verify", "commit", "mask"])
    if op == "attention":
        heads = rng.choice(sorted(HEADS))
        fp8 = heads in ("tiny", "glm") and rng.random() < 0.35
        win = rng.choice([0, 128, 1000]) if heads == "mimo" or rng.random() < 0.15 else 0
        batch = _log(rng, 1, 16)
        hi = _log(rng, 2, 57000 // batch)
        c = _attn("", heads, batch, rng.randint(0, hi), hi, _log(rng, 1, 61), fp8, win,
                  heads == "mimo" or rng.random() < 0.15)
    elif op == "verify":
        mode = rng.choice(["point", "draft", "greedy"])
        c = _verify("", mode, _log(rng, 1, 32), _log(rng, 1, 26), rng.choice([_log(rng, 500, 163840), 151552]),
                    mode != "greedy" and rng.random() < 0.4)
    elif op == "commit":
        heads = rng.choice(sorted(HEADS))
        c = _commit("", heads, rng.randint(1, 46 if heads != "qwen" else 12), _log(rng, 1, 16), _log(rng, 2, 61),
                    _log(rng, 2, 150), heads in ("tiny", "glm") and rng.random() < 0.4)
    else:
        c = _mask("", _log(rng, 1, 64), _log(rng, 9, 256))
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _trees(g, batch, nodes):
    """Node counts (the last sequence has `nodes`, the others up to a quarter fewer, the same for
    every seed: they set the outputs' shapes) and random parents: a node hangs below one of
    the 6 nodes before it, which gives branching paths several deep."""
    lens = nodes - 5 * torch.arange(batch - 1, -1, -1, device="cuda") % (nodes // 4 + 1)
    q_start = torch.zeros(batch + 1, dtype=torch.int32, device="cuda")
    q_start[1:] = lens.cumsum(0)
    T = int(q_start[-1])
    seq = torch.repeat_interleave(torch.arange(batch, device="cuda"), lens)
    i = torch.arange(T, device="cuda") - q_start[seq]
    back = torch.randint(1, 7, (T,), generator=g, device="cuda")
    parents = torch.where(i > 0, (i - back).clamp(min=0), -1).to(torch.int32)
    return lens, q_start, seq, i, parents, T


def _prepare_attention(case, g):
    Hq, Hk, D, Dv = HEADS[case["heads"]]
    B, N = case["batch"], case["nodes"]
    lens, q_start, _, _, parents, T = _trees(g, B, N)
    ctx = torch.randint(case["ctx_lo"], case["ctx_hi"] + 1, (B,), generator=g, device="cuda")
    kv_len = (ctx + lens).to(torch.int32)
    mb = -(-(case["ctx_hi"] + N) // PAGE)
    nblk = (kv_len + PAGE - 1) // PAGE
    total = int(nblk.sum())
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    bt = torch.zeros(B, mb, dtype=torch.int32, device="cuda")
    have = torch.arange(mb, device="cuda")[None] < nblk[:, None]
    bt[have] = order
    q = torch.randn(T, Hq, D, generator=g, device="cuda").to(torch.bfloat16)
    k = torch.randn(total, Hk, PAGE, D, generator=g, device="cuda")
    v = torch.randn(*((total, Hk, Dv, PAGE) if case["fp8"] else (total, Hk, PAGE, Dv)), generator=g, device="cuda")
    ks, vs = (0.0125, 0.0145) if case["fp8"] else (1.0, 1.0)
    t = torch.float8_e4m3fn if case["fp8"] else torch.bfloat16
    # the mask and depths that tree_mask gives for these parents, made here the plain way
    mask, depth = _plain_mask(parents, q_start, B, N)
    return {"q": q, "k": (k / ks).to(t), "v": (v / vs).to(t), "q_start": q_start, "kv_len": kv_len, "bt": bt,
            "mask": mask, "depth": depth, "B": B, "N": N, "max_kv": case["ctx_hi"] + N, "window": case["window"],
            "sinks": torch.randn(Hq, generator=g, device="cuda") if case["sinks"] else None, "ks": ks, "vs": vs,
            "scale": D ** -0.5, "Dv": Dv}


def _prepare_verify(case, g):
    B, N, V = case["batch"], case["nodes"], case["vocab"]
    _, q_start, seq, i, parents, T = _trees(g, B, N)
    logits = torch.randn(T, V, generator=g, device="cuda") * 3.0
    row = (q_start[seq] + parents.clamp(min=0)).long()
    s = {"q_start": q_start, "parents": parents, "B": B, "N": N, "mode": case["mode"], "probs": None, "draft": None,
         "u_accept": torch.rand(T, generator=g, device="cuda"), "u_draw": torch.rand(B, generator=g, device="cuda")}
    # the drafter agrees with the target up to noise
    guess = logits + 0.7 * torch.randn(T, V, generator=g, device="cuda")
    dt = torch.bfloat16 if case["bf16"] else torch.float32
    if case["mode"] == "draft":          # children drawn from the drafter's distribution at their parent
        qd = torch.softmax(guess, -1)
        s["tokens"] = torch.multinomial(qd[row], 1, generator=g)[:, 0].to(torch.int32)
        s["draft"] = qd.to(dt)
    else:                                # children are the drafter's most likely tokens at their parent
        top = guess.topk(min(6, V), dim=-1).indices
        s["tokens"] = top[row, (i.long() % min(6, V))].to(torch.int32)
    if case["mode"] == "greedy":
        s["target"] = logits.argmax(-1).to(torch.int32)
    else:
        s["probs"] = torch.softmax(logits, -1).to(dt)
    s["max_children"] = min(6, N - 1)    # a node's children lie within the 6 nodes after it
    return s


def _prepare_commit(case, g):
    _, Hk, D, Dv = HEADS[case["heads"]]
    B, N, L = case["batch"], case["nodes"], case["layers"]
    lens, q_start, seq, i, parents, T = _trees(g, B, N)
    ctx = torch.randint(1, case["ctx_hi"] + 1, (B,), generator=g, device="cuda")
    mb = -(-(case["ctx_hi"] + N) // PAGE)
    bt = torch.randperm(B * mb, generator=g, device="cuda").view(B, mb).to(torch.int32)
    # accept a random node and its ancestors
    leaf = (torch.rand(B, generator=g, device="cuda") * lens).long()
    anc, depth = _closure(parents, q_start, B, N)
    on = anc[torch.arange(B, device="cuda"), leaf]                               # [B, N]
    pos = torch.where(on, depth, N)
    path = torch.full((B, N + 1), -1, dtype=torch.int32, device="cuda")
    path.scatter_(1, pos, torch.arange(N, dtype=torch.int32, device="cuda").expand(B, N).contiguous())
    path = path[:, :N].contiguous()
    acc = (on.sum(1) - 1).to(torch.int32)
    t = torch.float8_e4m3fn if case["fp8"] else torch.bfloat16
    k = torch.randn(L, B * mb, Hk, PAGE, D, generator=g, device="cuda", dtype=torch.bfloat16).to(t)
    v = torch.randn(*((L, B * mb, Hk, Dv, PAGE) if case["fp8"] else (L, B * mb, Hk, PAGE, Dv)), generator=g,
                    device="cuda", dtype=torch.bfloat16).to(t)
    path = torch.where(torch.arange(N, device="cuda")[None] <= acc[:, None], path, -1)
    return {"k": k, "v": v, "path": path, "accepted": acc, "q_start": q_start, "kv_len": (ctx + lens).to(torch.int32),
            "bt": bt, "B": B, "N": N}


def _prepare_mask(case, g):
    _, q_start, _, _, parents, _ = _trees(g, case["batch"], case["nodes"])
    return {"parents": parents, "q_start": q_start, "B": case["batch"], "N": case["nodes"]}


_PREPARE = {"attention": _prepare_attention, "verify": _prepare_verify, "commit": _prepare_commit,
            "mask": _prepare_mask}


def prepare(case, seed):
    s = _PREPARE[case["op"]](case, _gen(seed))
    s["op"] = case["op"]
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _padded(q_start, B, N):
    """[B, N] row of every (sequence, node), and which exist (the others point at row 0)."""
    i = torch.arange(N, device=q_start.device)[None]
    rows = q_start[:B, None].long() + i
    ok = rows < q_start[1:, None]
    return torch.where(ok, rows, 0), ok


def _closure(parents, q_start, B, N):
    """anc [B, N, N]: node j is i or an ancestor of i; depth [B, N]."""
    rows, ok = _padded(q_start, B, N)
    par = torch.where(ok, parents[rows].long(), -1)
    n = torch.arange(N, device=parents.device)
    m = ((par[:, :, None] == n) | (n[:, None] == n)).float() * ok[:, :, None]
    for _ in range(max(1, (N - 1).bit_length())):      # paths of length 1, 2, 4, ...
        m = (torch.matmul(m, m) > 0).float()
    anc = m > 0
    return anc, anc.sum(-1) - 1


def _plain_mask(parents, q_start, B, N):
    anc, depth = _closure(parents, q_start, B, N)
    W = (N + 31) // 32
    bits = torch.nn.functional.pad(anc, (0, 32 * W - N)).view(B, N, W, 32).long()
    words = (bits << torch.arange(32, device=parents.device)).sum(-1)
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
    rows, ok = _padded(q_start, B, N)
    T = parents.shape[0]
    mask = torch.zeros(T + 1, W, dtype=torch.int32, device=parents.device)
    dep = torch.zeros(T + 1, dtype=torch.int32, device=parents.device)
    at = torch.where(ok, rows, T)
    mask[at] = words
    dep[at] = depth.to(torch.int32)
    return mask[:T], dep[:T]


def _plain_attention(s):
    q, B, N, Dv = s["q"], s["B"], s["N"], s["Dv"]
    T, Hq, D = q.shape
    Hk = s["k"].shape[1]
    G = Hq // Hk
    dev = q.device
    rows, ok = _padded(s["q_start"], B, N)
    bt = s["bt"].long()
    L = bt.shape[1] * PAGE
    k = (s["k"].float() * s["ks"])[bt].transpose(1, 2).reshape(B, Hk, L, D)
    v = s["v"].float() * s["vs"]
    if s["v"].dtype == torch.float8_e4m3fn:
        v = v.transpose(2, 3)
    v = v[bt].transpose(1, 2).reshape(B, Hk, L, Dv)
    qq = q.float()[rows].view(B, N, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * N, D)
    sc = (torch.matmul(qq, k.transpose(2, 3)) * s["scale"]).view(B, Hk, G, N, L)
    # which keys a node sees: the context inside its window, and its ancestors' bits
    ctx = (s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1])).long()[:, None, None]
    t = torch.arange(L, device=dev)[None, None]
    j = t - ctx                                                                    # [B, 1, L] node index
    words = s["mask"].long()[rows]                                                 # [B, N, W]
    jc = j.clamp(0, 32 * words.shape[2] - 1).expand(B, N, L)
    see = ((words.gather(2, jc >> 5) >> (jc & 31)) & 1).bool() & (j >= 0) & (t < s["kv_len"].long()[:, None, None])
    inside = j < 0
    if s["window"]:
        dep = s["depth"].long()[rows]
        far = dep[:, :, None] - s["window"]                # a key deeper than this is inside the window
        inside = inside & (j > far)
        dkey = torch.where(ok, dep, 0).gather(1, j.clamp(0, N - 1).expand(B, 1, L)[:, 0])[:, None]
        see = see & (dkey > far)
    see = (see | inside)[:, None, None]                                            # [B, 1, 1, N, L]
    sc = torch.where(see, sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sk = s["sinks"].float().view(1, Hk, G, 1, 1)
        m = torch.maximum(m, sk)
    m = torch.where(torch.isinf(m), 0.0, m)
    p = torch.exp(sc - m)
    tot = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        tot = tot + torch.exp(sk - m)
    p = p / torch.where(tot > 0, tot, 1.0)
    o = torch.matmul(p.view(B, Hk, G * N, L), v).view(B, Hk, G, N, Dv).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, Dv)
    out = torch.zeros(T + 1, Hq, Dv, dtype=q.dtype, device=dev)
    out[torch.where(ok, rows, T)] = o.to(q.dtype)
    return out[:T]


def _plain_verify(s):
    B, N = s["B"], s["N"]
    dev = s["tokens"].device
    rows, ok = _padded(s["q_start"], B, N)
    par = torch.where(ok, s["parents"].long()[rows], -1)
    tok = s["tokens"].long()[rows]
    n = torch.arange(N, device=dev)
    child = par >= 0
    sib = (par[:, :, None] == par[:, None, :]) & child[:, :, None] & (n[:, None] > n)     # j an earlier sibling of i
    prow = rows.gather(1, par.clamp(min=0))                                               # row of the parent
    if s["mode"] == "greedy":
        test = child & (tok == s["target"].long()[prow])
    else:
        u = s["u_accept"].double()[rows]
        pt = s["probs"][prow, tok].double()
        if s["mode"] == "point":
            first = child & ~(sib & (tok[:, :, None] == tok[:, None, :])).any(-1)
            gone = (sib * (pt * first)[:, None, :]).sum(-1)
            test = first & (u * (1.0 - gone) < pt)
        else:
            rank = sib.sum(-1)
            p, q = s["probs"], s["draft"]
            qt = q[prow, tok].double()
            w, z = p.double(), torch.ones(p.shape[0], dtype=torch.float64, device=dev)
            test = torch.zeros_like(child)
            for r in range(s["max_children"]):
                test = test | (child & (rank == r) & (u * qt * z[prow] < w[prow, tok]))
                w = (w / z[:, None] - q.double()).clamp_(min=0)
                z = w.sum(-1)
                z = torch.where(z > 0, z, 1.0)
    won = test & ~(sib & test[:, None, :]).any(-1) & ok                  # the first sibling that passes
    root = ok & (n == 0)
    anc, depth = _closure(s["parents"], s["q_start"], B, N)
    on = ((~anc) | (won | root)[:, None, :]).all(-1) & ok & (child | root)
    acc = (on.sum(1) - 1).clamp(min=0)
    last = torch.where(on, n, 0).amax(1)
    vrow = rows.gather(1, last[:, None])[:, 0]
    if s["mode"] == "greedy":
        x = s["target"].long()[vrow]
    else:
        w = s["probs"][vrow].double()
        if s["mode"] == "point":
            kids = (par == last[:, None]) & child
            w = torch.nn.functional.pad(w, (0, 1)).scatter(1, torch.where(kids, tok, w.shape[1]), 0.0)[:, :-1]
        else:
            left = ((par == last[:, None]) & child).sum(1)
            z, q = torch.ones_like(w[:, :1]), s["draft"][vrow].double()
            for r in range(s["max_children"]):
                w2 = (w / z - q).clamp_(min=0)
                w = torch.where(left[:, None] > r, w2, w)
                z2 = w.sum(1, keepdim=True)
                z = torch.where(left[:, None] > r, torch.where(z2 > 0, z2, 1.0), z)
        w = torch.where(w.sum(1, keepdim=True) > 0, w, s["probs"][vrow].double())
        cum = w.cumsum(1)
        x = (cum <= s["u_draw"].double()[:, None] * cum[:, -1:]).sum(1)
        lastpos = torch.where(w > 0, torch.arange(w.shape[1], device=dev), 0).amax(1)
        x = torch.minimum(x, lastpos)
    path = torch.full((B, N + 1), -1, dtype=torch.int32, device=dev)
    path.scatter_(1, torch.where(on, depth, N), n.to(torch.int32).expand(B, N).contiguous())
    out = torch.full((B, N + 1), -1, dtype=torch.int32, device=dev)
    out.scatter_(1, torch.where(on & (depth > 0), depth - 1, N), tok.to(torch.int32))
    out.scatter_(1, acc[:, None], x[:, None].to(torch.int32))
    path, out = path[:, :N], out[:, :N]
    keep = n[None] <= acc[:, None]
    return {"accepted": acc.to(torch.int32), "path": torch.where(keep, path, -1), "tokens": torch.where(keep, out, -1),
            "last_row": vrow.to(torch.int32)}


def _plain_commit(s):
    B, N = s["B"], s["N"]
    dev = s["path"].device
    ctx = (s["kv_len"] - (s["q_start"][1:] - s["q_start"][:-1])).long()[:, None]
    j = torch.arange(1, N, device=dev)[None]
    ok = j <= s["accepted"][:, None]
    src = ctx + torch.where(ok, s["path"][:, 1:].long(), 0)      # the others: the root onto itself
    dst = ctx + torch.where(ok, j, 0)
    fp8 = s["k"].dtype == torch.float8_e4m3fn
    k, v = (s["k"].view(torch.uint8), s["v"].view(torch.uint8)) if fp8 else (s["k"], s["v"])
    sb, db = s["bt"].long().gather(1, src // PAGE), s["bt"].long().gather(1, dst // PAGE)
    so, do = src % PAGE, dst % PAGE
    k[:, db, :, do] = k[:, sb, :, so]
    if fp8:
        v[:, db, :, :, do] = v[:, sb, :, :, so]
    else:
        v[:, db, :, do] = v[:, sb, :, so]
    return s["k"], s["v"]


def run(state):
    s = state
    op = s["op"]
    if not own:
        if op == "attention":
            return _plain_attention(s)
        if op == "verify":
            return _plain_verify(s)
        if op == "commit":
            return _plain_commit(s)
        return _plain_mask(s["parents"], s["q_start"], s["B"], s["N"])
    from vllm_xtu_moe_b200.ops import tree
    if op == "attention":
        meta = tree.TreeMetadata(num_seqs=s["B"], q_start=s["q_start"], kv_len=s["kv_len"], block_table=s["bt"],
                                 mask=s["mask"], depth=s["depth"], max_nodes=s["N"], max_kv_len=s["max_kv"])
        return tree.tree_attention(s["q"], s["k"], s["v"], meta, scale=s["scale"], window=s["window"],
                                   sinks=s["sinks"], k_scale=s["ks"], v_scale=s["vs"])
    if op == "verify":
        if s["mode"] == "greedy":
            r = tree.verify_tree_greedy(s["target"], s["tokens"], s["parents"], s["q_start"], s["N"])
        else:
            r = tree.verify_tree(s["probs"], s["tokens"], s["parents"], s["q_start"], s["N"], s["u_accept"],
                                 s["u_draw"], draft_probs=s["draft"])
        return {"accepted": r.accepted, "path": r.path, "tokens": r.tokens, "last_row": r.last_row}
    if op == "commit":
        tree.commit_tree(s["k"], s["v"], s["path"], s["accepted"], s["q_start"], s["kv_len"], s["bt"])
        return s["k"], s["v"]
    return tree.tree_mask(s["parents"], s["q_start"], s["N"])


# ---------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------
def _family(parents, i):
    """Node i and its ancestors, as a list from i up."""
    got = [i]
    while parents[got[-1]] >= 0:
        got.append(parents[got[-1]])
    return got


def _exact_attention(s):
    q = s["q"].double()
    T, Hq, D = q.shape
    Hk, dev = s["k"].shape[1], q.device
    G = Hq // Hk
    qs, kl, dep = s["q_start"].tolist(), s["kv_len"].tolist(), s["depth"].tolist()
    mask = [[w & 0xFFFFFFFF for w in r] for r in s["mask"].tolist()]
    out = torch.zeros(T, Hq, s["Dv"], dtype=torch.float64, device=dev)
    for b in range(s["B"]):
        n, ctx = qs[b + 1] - qs[b], kl[b] - (qs[b + 1] - qs[b])
        if n == 0:
            continue
        see = torch.zeros(n, kl[b], dtype=torch.bool)
        for i in range(n):
            row = qs[b] + i
            low = max(0, ctx + dep[row] - s["window"] + 1) if s["window"] else 0
            see[i, low:ctx] = True
            for j in range(n):
                if mask[row][j // 32] >> (j % 32) & 1 and (not s["window"] or dep[qs[b] + j] > dep[row] - s["window"]):
                    see[i, ctx + j] = True
        see = see.to(dev)
        blocks = s["bt"][b, :-(-kl[b] // PAGE)].long()
        for h in range(Hk):
            kk = (s["k"][blocks, h].double() * s["ks"]).reshape(-1, D)[:kl[b]]
            vv = s["v"][blocks, h].double() * s["vs"]
            if s["v"].dtype == torch.float8_e4m3fn:
                vv = vv.transpose(1, 2)
            vv = vv.reshape(-1, s["Dv"])[:kl[b]]
            for g in range(G):
                e = (q[qs[b]:qs[b + 1], h * G + g] @ kk.t()) * s["scale"]
                e = e.masked_fill(~see, -math.inf)
                top = e.amax(1, keepdim=True)
                sk = s["sinks"][h * G + g].double() if s["sinks"] is not None else None
                if sk is not None:
                    top = torch.maximum(top, sk)
                top = torch.where(torch.isinf(top), 0.0, top)
                e = torch.exp(e - top)
                z = e.sum(1, keepdim=True) + (torch.exp(sk - top) if sk is not None else 0.0)
                out[qs[b]:qs[b + 1], h * G + g] = (e / torch.where(z > 0, z, 1.0)) @ vv
    return out


def _exact_verify(s):
    B, N = s["B"], s["N"]
    qs, par, tok = s["q_start"].tolist(), s["parents"].tolist(), s["tokens"].tolist()
    ua, ud = s["u_accept"].tolist(), s["u_draw"].tolist()
    accepted, paths, tokens, last_row = [], [], [], []
    for b in range(B):
        q0, n = qs[b], qs[b + 1] - qs[b]
        at, path, emitted, w = 0, [0], [], None
        while True:
            kids = [i for i in range(n) if par[q0 + i] == at and i > 0]
            step = None
            if s["mode"] != "greedy":
                w, z = s["probs"][q0 + at].double().clone(), 1.0
                d = s["draft"][q0 + at].double() if s["mode"] == "draft" else None
            for i in kids:
                x = tok[q0 + i]
                if s["mode"] == "greedy":
                    if x == int(s["target"][q0 + at]):
                        step = i
                        break
                    continue
                share = z if d is None else z * float(d[x])
                if ua[q0 + i] * share < float(w[x]):
                    step = i
                    break
                if d is None:
                    z -= float(w[x])
                    w[x] = 0.0
                else:
                    w = torch.clamp(w / z - d, min=0)
                    z = float(w.sum())
                    z = z if z > 0 else 1.0
            if step is None:
                break
            at = step
            path.append(step)
            emitted.append(tok[q0 + step])
        if s["mode"] == "greedy":
            x = int(s["target"][q0 + at])
        else:
            if float(w.sum()) <= 0:
                w = s["probs"][q0 + at].double()
            cum = w.cumsum(0)
            x = int((cum <= ud[b] * float(cum[-1])).sum())
            x = min(x, int(torch.nonzero(w > 0)[-1]))
        accepted.append(len(path) - 1)
        paths.append(path + [-1] * (N - len(path)))
        tokens.append(emitted + [x] + [-1] * (N - len(emitted) - 1))
        last_row.append(q0 + at)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=s["tokens"].device)  # noqa: E731
    return {"accepted": t(accepted), "path": t(paths), "tokens": t(tokens), "last_row": t(last_row)}


def _exact_commit(s):
    k, v = s["k"].double(), s["v"].double()
    k0, v0 = k.clone(), v.clone()
    qs, kl, acc = s["q_start"].tolist(), s["kv_len"].tolist(), s["accepted"].tolist()
    path, bt = s["path"].tolist(), s["bt"].tolist()
    fp8 = s["v"].dtype == torch.float8_e4m3fn
    for b in range(s["B"]):
        ctx = kl[b] - (qs[b + 1] - qs[b])
        for j in range(1, acc[b] + 1):
            f, t = ctx + path[b][j], ctx + j
            fb, tb = bt[b][f // PAGE], bt[b][t // PAGE]
            k[:, tb, :, t % PAGE] = k0[:, fb, :, f % PAGE]
            if fp8:
                v[:, tb, :, :, t % PAGE] = v0[:, fb, :, :, f % PAGE]
            else:
                v[:, tb, :, t % PAGE] = v0[:, fb, :, f % PAGE]
    return k, v


def _exact_mask(s):
    par, qs = s["parents"].tolist(), s["q_start"].tolist()
    W = (s["N"] + 31) // 32
    mask, depth = [], []
    for b in range(s["B"]):
        mine = par[qs[b]:qs[b + 1]]
        for i in range(len(mine)):
            up = _family(mine, i)
            words = [0] * W
            for a in up:
                words[a // 32] |= 1 << (a % 32)
            mask.append([w - 2 ** 32 if w >= 2 ** 31 else w for w in words])
            depth.append(len(up) - 1)
    dev = s["parents"].device
    return torch.tensor(mask, dtype=torch.int32, device=dev), torch.tensor(depth, dtype=torch.int32, device=dev)


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "verify": _exact_verify, "commit": _exact_commit,
            "mask": _exact_mask}[case["op"]](s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "attention":
        Hq, Hk, D, Dv = HEADS[case["heads"]]
        B, N = case["batch"], case["nodes"]
        n = B * N * 7 / 8                                      # nodes in all, on average
        ctx = (case["ctx_lo"] + case["ctx_hi"]) / 2
        seen = min(ctx, case["window"]) if case["window"] else ctx
        size = 1 if case["fp8"] else 2
        kv = B * (seen + N) * Hk * (D + Dv) * size
        return {"bytes": kv + n * Hq * (D + Dv) * 2 + n * ((N + 31) // 32) * 4,
                "flops": 2.0 * n * Hq * (seen + N / 4) * (D + Dv)}
    if case["op"] == "verify":
        B, N, V = case["batch"], case["nodes"], case["vocab"]
        size = 2 if case["bf16"] else 4
        nodes = B * N * 16.0
        if case["mode"] == "greedy":
            return {"bytes": nodes + 8 * B * N, "flops": 0}
        # the row (with the drafter's: both rows) from which the last token is drawn
        rows = 2 if case["mode"] == "draft" else 1
        return {"bytes": B * V * size * rows + nodes + 8 * B * N, "flops": 2.0 * B * V * rows}
    if case["op"] == "commit":
        _, Hk, D, Dv = HEADS[case["heads"]]
        moved = case["batch"] * max(1.0, case["nodes"] / 7)     # a random node's depth: 3.5 nodes a level
        return {"bytes": 2.0 * moved * case["layers"] * Hk * (D + Dv) * (1 if case["fp8"] else 2), "flops": 0}
    n = case["batch"] * case["nodes"] * 7 / 8
    return {"bytes": n * (4 + 4 + 4 * ((case["nodes"] + 31) // 32)), "flops": 0}
