"""Tree speculation: one step verifies a tree of drafted tokens per sequence.

A chain of drafts (``engine/spec_decode.py``) gives up at its first wrong token; a tree keeps
alternatives.  The nodes of sequence b are the rows ``q_start[b] .. q_start[b+1] - 1`` of the step:
node 0 the root (the last emitted token), every other node a drafted token below a parent of
lower index (``parents``, node indices inside the sequence, -1 for the root).  A step

1. ``tree_mask``       turns the parents into ancestor bit rows and depths (a node's position is
                       context length + depth),
2. writes the nodes' K / V behind the context, node i at slot context + i
   (``basic.rope_and_cache`` with those slots and positions),
3. ``tree_attention``  attends from every node to the context and to its ancestors, beside
                       :func:`attention.paged_attention` and over the same paged caches,
4. ``verify_tree_greedy`` / ``verify_tree``  choose the accepted path and the token after it,
5. ``commit_tree``     moves the accepted nodes' K / V to the slots behind the context, in every layer.

The kernels are in ``csrc/cuda/tree.cu`` and ``csrc/cuda/tree_attention.cu``; on CPU tensors the
``*_ref`` restatements run.  All calls work on the current stream of their tensors' device, copy
nothing to the host and can be captured into a CUDA graph.
"""
from __future__ import annotations

import functools
import math
from array import array
from dataclasses import dataclass

import torch

from . import _native as N
from .attention import KV_BLOCK, _gather_kv, dequant_fp8_cache

MAX_NODES = 1024          # nodes of one sequence's tree
MAX_SPLITS = 64
_FP8, _BF16, _F32, _I32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.int32
# (K width, V width) that the GPU kernels serve
HEAD_DIMS = ((64, 64), (128, 128), (192, 128), (256, 256))
FP8_HEAD_DIMS = ((64, 64), (128, 128))


@dataclass
class TreeMetadata:
    """A step's trees.  ``kv_len`` counts the context and the nodes, as in ``AttnMetadata``."""
    num_seqs: int
    q_start: torch.Tensor        # int32 [B+1]
    kv_len: torch.Tensor         # int32 [B] context + nodes
    block_table: torch.Tensor    # int32 [B, max_blocks]
    mask: torch.Tensor           # int32 [T, W] bit j of row i: node i sees node j (of its sequence)
    max_nodes: int               # largest tree of the step
    max_kv_len: int
    depth: torch.Tensor | None = None   # int32 [T]; sliding-window layers need it
    num_splits: int = 0          # KV splits; 0: chosen from the sizes


@dataclass
class TreeVerdict:
    accepted: torch.Tensor       # int32 [B] accepted drafts
    path: torch.Tensor           # int32 [B, max_nodes] the root and the accepted nodes, then -1
    tokens: torch.Tensor         # int32 [B, max_nodes] accepted tokens and the one after them, then -1
    last_row: torch.Tensor       # int32 [B] row of the last accepted node (-1: a sequence without nodes)


# A step makes these calls once per layer and their kernels take a few microseconds, so the checks are
# written to cost little where they pass: messages are put together only for a refusal, and devices are
# compared by their index (-1: the CPU), which costs less than torch.device objects.
def _name(dev: int) -> str:
    return "cpu" if dev < 0 else f"cuda:{dev}"


def _ints(name: str, t: torch.Tensor, shape: tuple, dev: int) -> None:
    if t.dtype is not _I32 or t.shape != shape or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape} on {_name(dev)}, not "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")


def _table(bt: torch.Tensor, B: int, dev: int) -> tuple[int, int]:
    """(row stride, columns) of a block table."""
    shape, stride = bt.shape, bt.stride()
    if bt.dtype is not _I32 or len(shape) != 2 or shape[0] < B or stride[1] != 1 or bt.get_device() != dev:
        raise ValueError(f"block_table must be int32 [{B}, blocks] with contiguous rows on {_name(dev)}")
    return stride[0], shape[1]


def _max_nodes(n: int) -> None:
    if not 1 <= n <= MAX_NODES:
        raise ValueError(f"max_nodes must be 1 .. {MAX_NODES}, not {n}")


def _elsewhere(dev: int) -> bool:
    return dev != torch._C._cuda_getDevice()


def _ptr(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _status(dev: int) -> int:
    st = N._status.get(dev)
    return (st if st is not None else N.status_buffer(dev)).data_ptr()


def _stream(dev: int) -> int:
    return torch._C._cuda_getCurrentRawStream(dev)


# ---------------------------------------------------------------------------
# mask
# ---------------------------------------------------------------------------
def tree_mask_ref(parents: torch.Tensor, q_start: torch.Tensor, max_nodes: int, mask: torch.Tensor,
                  depth: torch.Tensor) -> None:
    par, qs = parents.tolist(), q_start.tolist()
    W = mask.shape[1]
    for b in range(len(qs) - 1):
        rows = []
        for i in range(qs[b + 1] - qs[b]):
            p = par[qs[b] + i]
            rows.append((rows[p] if 0 <= p < i else 0) | 1 << i)
            words = [rows[i] >> 32 * w & 0xFFFFFFFF for w in range(W)]
            mask[qs[b] + i] = torch.tensor([w - (1 << 32) if w >> 31 else w for w in words], dtype=torch.int32)
            depth[qs[b] + i] = rows[i].bit_count() - 1


def tree_mask(parents: torch.Tensor, q_start: torch.Tensor, max_nodes: int, mask: torch.Tensor | None = None,
              depth: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """parents int32 [T] -> (mask int32 [T, ceil(max_nodes / 32)], depth int32 [T]).

    Bit j of row i: j is node i or an ancestor of it.  A parent that is negative or not below its
    node means none.  Rows behind the last sequence are left as they are."""
    _max_nodes(max_nodes)
    dev = parents.get_device()
    T, B = len(parents), len(q_start) - 1
    _ints("parents", parents, (T,), dev)
    _ints("q_start", q_start, (B + 1,), dev)
    W = (max_nodes + 31) // 32
    mask = mask if mask is not None else parents.new_empty((T, W))
    depth = depth if depth is not None else torch.empty_like(parents)
    _ints("mask", mask, (T, W), dev)
    _ints("depth", depth, (T,), dev)
    if dev < 0:
        tree_mask_ref(parents, q_start, max_nodes, mask, depth)
        return mask, depth
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return tree_mask(parents, q_start, max_nodes, mask, depth)
    N.call_packed("xtu_tree_mask", parents.data_ptr(), q_start.data_ptr(), B, T, max_nodes, W, mask.data_ptr(),
                  depth.data_ptr(), _status(dev), _stream(dev))
    return mask, depth


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def tree_attention_ref(q, k_cache, v_cache, meta: TreeMetadata, scale: float, out: torch.Tensor, window: int = 0,
                       sinks: torch.Tensor | None = None, k_scale: float = 1.0, v_scale: float = 1.0) -> torch.Tensor:
    """q [T, Hq, D] -> out [T, Hq, Dv] (fp32 math, sequence by sequence)."""
    if k_cache.dtype == _FP8:
        k_cache, v_cache = dequant_fp8_cache(k_cache, v_cache, k_scale, v_scale)
    Hk = k_cache.shape[1]
    G = q.shape[1] // Hk
    qs, kl = meta.q_start.tolist(), meta.kv_len.tolist()
    for b in range(meta.num_seqs):
        r0, n = qs[b], qs[b + 1] - qs[b]
        if n == 0:
            continue
        if kl[b] <= 0:
            out[r0:r0 + n] = 0
            continue
        ctx = kl[b] - n
        k = _gather_kv(k_cache, meta.block_table[b], kl[b]).float().repeat_interleave(G, dim=1)
        v = _gather_kv(v_cache, meta.block_table[b], kl[b]).float().repeat_interleave(G, dim=1)
        node = torch.arange(n, device=q.device)
        tree = (meta.mask[r0:r0 + n].long()[:, node >> 5] >> (node & 31) & 1).bool()            # [i, j]
        see = torch.ones(n, kl[b], dtype=torch.bool, device=q.device)
        first = max(0, -ctx)          # (fewer keys than nodes, padding: the last nodes' keys are there)
        if window > 0:
            deep = meta.depth[r0:r0 + n].long().clamp(0, n - 1)
            far = deep[:, None] - window
            see[:, :max(0, ctx)] = torch.arange(max(0, ctx), device=q.device)[None] > ctx + far
            tree &= deep[None] > far
        see[:, max(0, ctx):] = tree[:, first:]
        s = torch.einsum("qhd,khd->hqk", q[r0:r0 + n].float(), k) * scale
        s = s.masked_fill(~see[None], float("-inf"))
        m = s.amax(-1, keepdim=True)
        if sinks is not None:
            sk = sinks.float()[:, None, None]
            m = torch.maximum(m, sk)
        m = m.masked_fill(m == float("-inf"), 0.0)
        p = torch.exp(s - m)
        z = p.sum(-1, keepdim=True)
        if sinks is not None:
            z = z + torch.exp(sk - m)
        p = torch.where(z == 0.0, 0.0, p / z)
        # a key that a row does not see must not reach it as 0 * NaN
        if torch.isfinite(v).all():
            o = torch.einsum("hqk,khd->qhd", p, v)
        else:
            o = torch.stack([torch.einsum("hk,khd->hd", p[:, i, see[i]], v[see[i]]) for i in range(n)])
        out[r0:r0 + n] = o.to(out.dtype)
    return out


@functools.lru_cache(maxsize=4096)
def _plan(groups: int, rows: int, keys: int, one: bool, one_us: float, splits: int, num_sms: int) -> tuple[int, int]:
    best = None
    for tiles in ((1,) if one or rows <= 128 else (1, 2)):
        ctas = max(1, -(-rows // (128 * tiles)) * groups)
        for s in ((splits,) if splits else range(1, max(1, min(MAX_SPLITS, keys)) + 1)):
            cost = -(-ctas * s // num_sms) * (-(-keys // s) * (1.8 if tiles == 2 else one_us) + 9) + (7 if s > 1 else 0)
            if best is None or cost < best[0]:
                best = (cost, tiles, s)
    return best[1], best[2]


def tree_plan(num_seqs: int, num_kv_heads: int, rows: int, seen: int, d: int = 128, dv: int = 128, splits: int = 0,
              fp8: bool = False, num_sms: int = 148) -> tuple[int, int]:
    """(row tiles of a CTA, KV splits) of a step.  ``rows``: query rows of the largest tree per KV head,
    ``seen``: keys that a sequence attends to, ``splits``: a split count that is given.

    One CTA per SM takes one or two 128-row tiles of a (sequence, KV head, split).  In microseconds a
    key tile costs about 1.8 for two row tiles and 0.85 for one (1.55 from fp8, 1.2 of 256-wide heads),
    a CTA's start and end 9 and the merge of the splits 7, so the time is about
    waves * (key tiles per split * that + 9) + 7.  Measured (4 x 14.6K keys, 8 KV heads, cold caches),
    one / two row tiles at their best splits: 192 rows 74 / 82 us, 480 rows 115 / 137, 732 rows 184 /
    182; fp8: 192 rows 117 / 90, 60 rows 66 / 70."""
    one_us = 1.55 if fp8 else 0.85 if dv <= 128 else 1.2
    return _plan(num_seqs * num_kv_heads, rows, -(-seen // (128 if d <= 128 else 64)), dv > 128, one_us, splits, num_sms)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, meta: TreeMetadata,
                   scale: float | None = None, out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                   window: int = 0, sinks: torch.Tensor | None = None, k_scale: float = 1.0,
                   v_scale: float = 1.0) -> torch.Tensor:
    """Tree nodes' queries q [T, Hq, D] bf16 over the paged cache -> [T, Hq, Dv] bf16.

    Node i sees its sequence's context and the nodes of its mask row; with ``window`` > 0 only
    keys at positions above its own minus the window (node j lies at context + ``meta.depth[j]``).
    ``sinks`` fp32 [Hq]: learned logits in the denominator.  A row that sees nothing (or only
    scores of minus infinity) is zero.
    Keys outside a row's view never reach it, whatever the cache holds there; rows behind the
    last sequence are left as they are.  On the GPU ``_native.check_status`` reports a sequence whose
    rows lie outside q and nodes past ``meta.max_nodes``, whose rows stay as they are too, and keys past
    the block table, which no row sees.  Rows of a sequence with a ``kv_len`` of 0 (padding) are zero.

    Scores, softmax statistics and sums are held in 32 bits; the weights of the second product are rounded to the
    type of its operands, bf16 (half a step: 2^-8 of each) over bf16 caches, fp16 (2^-11) over fp8 ones.

    Caches as in :func:`attention.paged_attention`: bf16 ``[blocks, Hkv, 64, D]`` / ``[.., Dv]`` with
    (D, Dv) in ``HEAD_DIMS``, or fp8 (e4m3) K and per-block transposed V with ``FP8_HEAD_DIMS`` (their
    products take q as fp16: magnitudes up to 65504).  MLA latent caches are not served.
    ``out``: bf16 [T, Hq, Dv], contiguous, on a 16-byte boundary.
    ``workspace``: fp32, ``splits * T * Hq * (Dv + 2)`` elements when the KV range is split; allocated
    when None or too small.  One that is passed in belongs to the call until its work is done: calls
    that may overlap take one each."""
    dev = q.get_device()
    if q.dim() != 3 or (dev >= 0 and q.dtype is not _BF16):
        raise ValueError("q must be [T, Hq, D] bfloat16")
    T, Hq, D = q.shape
    if k_cache.dim() != 4 or v_cache is None or v_cache.dim() != 4:
        raise ValueError("tree attention takes a K and a V cache [blocks, Hkv, 64, D]")
    nb, Hk, bs, Dk = k_cache.shape
    kt, vshape = k_cache.dtype, v_cache.shape
    fp8 = kt is _FP8
    Dv = vshape[2] if fp8 else vshape[3]
    if vshape != ((nb, Hk, Dv, bs) if fp8 else (nb, Hk, bs, Dv)) or Dk != D or v_cache.dtype is not kt:
        raise ValueError(f"caches {tuple(k_cache.shape)} and {tuple(vshape)} do not match each other or q")
    if Hq % Hk:
        raise ValueError(f"{Hq} query heads do not divide over {Hk} KV heads")
    if k_cache.get_device() != dev or v_cache.get_device() != dev:
        raise ValueError(f"the caches must be on {_name(dev)}")
    B, most = meta.num_seqs, meta.max_nodes
    q_start, kv_len, bt, mask = meta.q_start, meta.kv_len, meta.block_table, meta.mask
    _max_nodes(most)
    _ints("q_start", q_start, (B + 1,), dev)
    _ints("kv_len", kv_len, (B,), dev)
    bt_stride, bt_cols = _table(bt, B, dev)
    W = mask.shape[-1]
    _ints("mask", mask, (T, W), dev)
    if 32 * W < most:
        raise ValueError(f"a mask of {W} words is too narrow for {most} nodes")
    if window > 0:
        if meta.depth is None:
            raise ValueError("a sliding window needs the nodes' depths")
        _ints("depth", meta.depth, (T,), dev)
    if sinks is not None and (sinks.dtype is not _F32 or not sinks.is_contiguous() or sinks.numel() != Hq
                              or sinks.get_device() != dev):
        raise ValueError(f"sinks must be contiguous fp32 [{Hq}] on {_name(dev)}")
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if not (scale > 0 and k_scale > 0):
        raise ValueError("scales must be positive")
    if out is None:
        out = torch.empty_like(q) if Dv == D and q.is_contiguous() else q.new_empty((T, Hq, Dv))
    elif out.shape != (T, Hq, Dv) or out.dtype is not q.dtype or not out.is_contiguous() or out.get_device() != dev:
        raise ValueError(f"out must be contiguous {q.dtype} [{T}, {Hq}, {Dv}] on {_name(dev)}")
    if dev < 0:
        return tree_attention_ref(q, k_cache, v_cache, meta, scale, out, window, sinks, k_scale, v_scale)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return tree_attention(q, k_cache, v_cache, meta, scale, out, workspace, window, sinks, k_scale, v_scale)
    if not fp8 and kt is not _BF16:
        raise ValueError(f"the cache must be bfloat16 or float8_e4m3fn, not {kt}")
    if (D, Dv) not in (FP8_HEAD_DIMS if fp8 else HEAD_DIMS):
        raise ValueError(f"{'fp8 ' if fp8 else ''}head sizes {D} / {Dv} are not served "
                         f"({FP8_HEAD_DIMS if fp8 else HEAD_DIMS})")
    if bs != KV_BLOCK:
        raise ValueError(f"the GPU kernels read KV blocks of {KV_BLOCK} tokens, not {bs}")
    kp, vp, qp = k_cache.data_ptr(), v_cache.data_ptr(), q.data_ptr()
    if (kp | vp) & 15 or not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError("the caches must be contiguous and start on 16-byte boundaries")
    if not 0 < (nb + 1) * Hk * max(bs, Dv) < 2 ** 31:
        raise ValueError("the cache is empty or has more rows than 31 bits count")
    q_ts, q_hs, q1 = q.stride()
    if q1 != 1 or (q_ts | q_hs) & 7 or qp & 15:
        raise ValueError("q rows must be contiguous and start on 16-byte boundaries")
    op = out.data_ptr()
    if op & 15:
        raise ValueError("out must start on a 16-byte boundary")
    rows = most * (Hq // Hk)
    seen = min(meta.max_kv_len, window + most + KV_BLOCK) if window > 0 else meta.max_kv_len
    tiles, splits = tree_plan(B, Hk, rows, seen, D, Dv, meta.num_splits, fp8)
    if not 1 <= splits <= MAX_SPLITS:
        raise ValueError(f"1 .. {MAX_SPLITS} splits, not {splits}")
    ws = None
    if splits > 1:
        need = splits * T * Hq * (Dv + 2)
        ws = workspace
        if ws is not None and (ws.dtype is not _F32 or not ws.is_contiguous() or ws.get_device() != dev
                               or ws.data_ptr() & 15):
            raise ValueError(f"workspace must be contiguous fp32 on {_name(dev)}, on a 16-byte boundary")
        if ws is None or ws.numel() < need:
            ws = q.new_empty(need, dtype=_F32)
    N.call_packed("xtu_tree_attention", qp, q_ts, q_hs, kp, vp, fp8, op, q_start.data_ptr(), kv_len.data_ptr(),
                  bt.data_ptr(), bt_stride, bt_cols, mask.data_ptr(), W, _ptr(meta.depth), min(window, 2 ** 31 - 1), B,
                  most, T, Hq, Hk, D, Dv, nb, scale, k_scale, v_scale, _ptr(sinks), tiles, splits, _ptr(ws),
                  _status(dev), _stream(dev))
    return out


# ---------------------------------------------------------------------------
# verification
# ---------------------------------------------------------------------------
def _verdict(B: int, max_nodes: int, like: torch.Tensor) -> TreeVerdict:
    accepted, path = like.new_empty(B), like.new_empty((B, max_nodes))
    return TreeVerdict(accepted, path, torch.empty_like(path), torch.empty_like(accepted))


def _children(parents: list, n: int, at: int) -> list:
    return [i for i in range(1, n) if parents[i] == at and at < i]


def _walk(tokens, parents, q_start, max_nodes, choose, final) -> TreeVerdict:
    """The verification of every sequence on the host: ``choose(row, children)`` -> the accepted
    child or None, ``final(row, children, b)`` -> the token after the path."""
    qs, par, tok = q_start.tolist(), parents.tolist(), tokens.tolist()
    v = _verdict(len(qs) - 1, max_nodes, tokens)
    for t in (v.path, v.tokens, v.last_row):
        t.fill_(-1)
    v.accepted.zero_()
    for b in range(len(qs) - 1):
        q0, n = qs[b], qs[b + 1] - qs[b]
        if n == 0:
            continue
        mine, path = par[q0:q0 + n], [0]
        while True:
            kids = _children(mine, n, path[-1])
            c = choose(q0, path[-1], kids)
            if c is None:
                break
            path.append(c)
        v.accepted[b] = len(path) - 1
        v.path[b, :len(path)] = torch.tensor(path, dtype=torch.int32)
        v.tokens[b, :len(path)] = torch.tensor([tok[q0 + i] for i in path[1:]] + [final(q0, path[-1], kids, b)],
                                               dtype=torch.int32)
        v.last_row[b] = q0 + path[-1]
    return v


def _tree_args(tokens, parents, q_start, max_nodes):
    _max_nodes(max_nodes)
    T, B, dev = len(tokens), len(q_start) - 1, tokens.get_device()
    _ints("tokens", tokens, (T,), dev)
    _ints("parents", parents, (T,), dev)
    _ints("q_start", q_start, (B + 1,), dev)
    return T, B, dev


def verify_tree_greedy_ref(target, tokens, parents, q_start, max_nodes) -> TreeVerdict:
    tgt, tok = target.tolist(), tokens.tolist()
    return _walk(tokens, parents, q_start, max_nodes,
                 lambda q0, at, kids: next((c for c in kids if tok[q0 + c] == tgt[q0 + at]), None),
                 lambda q0, at, kids, b: tgt[q0 + at])


def verify_tree_greedy(target: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, q_start: torch.Tensor,
                       max_nodes: int) -> TreeVerdict:
    """Greedy verification: ``target`` int32 [T] holds the model's token after every node.  From the
    root the path takes the first child (lowest index) whose token is the target's, and ends
    with the target's token after the last accepted node (``verify_greedy`` for trees)."""
    T, B, dev = _tree_args(tokens, parents, q_start, max_nodes)
    _ints("target", target, (T,), dev)
    if dev < 0:
        return verify_tree_greedy_ref(target, tokens, parents, q_start, max_nodes)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return verify_tree_greedy(target, tokens, parents, q_start, max_nodes)
    v = _verdict(B, max_nodes, tokens)
    N.call_packed("xtu_tree_verify_greedy", target.data_ptr(), tokens.data_ptr(), parents.data_ptr(),
                  q_start.data_ptr(), B, T, max_nodes, v.accepted.data_ptr(), v.path.data_ptr(), v.tokens.data_ptr(),
                  v.last_row.data_ptr(), _status(dev), _stream(dev))
    return v


def verify_tree_ref(probs, tokens, parents, q_start, max_nodes, u_accept, u_draw, draft_probs=None) -> TreeVerdict:
    tok, ua, ud = tokens.tolist(), u_accept.tolist(), u_draw.tolist()
    V = probs.shape[1]
    state = {}

    def weights(row):       # NaN and negative entries weigh nothing
        w = probs[row].double()
        return torch.where(w > 0, w, 0.0)

    def choose(q0, at, kids):
        w, z, gone = weights(q0 + at), 1.0, 0.0
        d = None
        if draft_probs is not None:
            d = draft_probs[q0 + at].double()
            d = torch.where(d > 0, d, 0.0)
        state["w"] = w
        for c in kids:
            x = tok[q0 + c]
            p = float(w[x]) if 0 <= x < V else 0.0
            if d is None:
                seen = any(tok[q0 + e] == x for e in kids[:kids.index(c)])
                if 0 <= x < V and not seen and float(probs[q0 + at, x]) >= 0 and ua[q0 + c] * (1.0 - gone) < p:
                    return c
                if 0 <= x < V:
                    gone += p
                    w[x] = 0.0
            else:
                if 0 <= x < V and ua[q0 + c] * float(d[x]) * z < p:
                    return c
                w = torch.clamp(w / z - d, min=0)
                z = float(w.sum())
                z = z if z > 0 else 1.0
                state["w"] = w
        return None

    def final(q0, at, kids, b):
        w = state["w"]
        if not float(w.sum()) > 0:
            w = weights(q0 + at)
        pos = torch.nonzero(w > 0)
        if pos.numel() == 0:
            return 0
        cum = w.cumsum(0)
        hit = torch.nonzero((cum > ud[b] * float(cum[-1])) & (w > 0))
        return int(hit[0]) if hit.numel() else int(pos[-1])

    return _walk(tokens, parents, q_start, max_nodes, choose, final)


def verify_tree(probs: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor, q_start: torch.Tensor,
                max_nodes: int, u_accept: torch.Tensor, u_draw: torch.Tensor,
                draft_probs: torch.Tensor | None = None) -> TreeVerdict:
    """Rejection-sampling verification with given random numbers (``verify_sampled`` for trees).

    probs [T, V] fp32 or bf16: the request's (filtered) sampling distribution after every node;
    u_accept fp32 [T] one uniform number in [0, 1) per node, u_draw fp32 [B] one per sequence.
    At a node the children are tried in index order:

    * ``draft_probs`` None, drafts chosen outright (a greedy drafter's likeliest tokens): child c
      with token x is accepted when u_c (1 - r) < p(x), r the probability of the siblings
      rejected before it; a rejected token's probability is removed.  A sibling that repeats
      a rejected token is rejected.
    * ``draft_probs`` [T, V] (the type of probs): the children of a node were drawn independently
      from its row q.  With w = p and Z = 1 at first, a child is accepted when u_c q(x) Z < w(x);
      each rejection sets w to max(0, w / Z - q) and Z to its sum.

    A node whose children are all rejected (or that has none) ends the path and emits the smallest
    token t with w(0) + .. + w(t) > u_draw * sum(w), in the weights that are left (in p when
    nothing is left of them).  Every emitted token is then a sample of the target's
    distribution.  NaN and negative entries weigh nothing, and a draft outside the vocabulary is
    never accepted."""
    T, B, dev = _tree_args(tokens, parents, q_start, max_nodes)
    shape, stride, dtype = probs.shape, probs.stride(), probs.dtype
    if (len(shape) != 2 or shape[0] != T or shape[1] < 1 or probs.get_device() != dev or stride[1] != 1
            or not (dtype is _F32 or dtype is _BF16)):
        raise ValueError(f"probs must be fp32 or bf16 [{T}, V] with contiguous rows on {_name(dev)}")
    if draft_probs is not None and (draft_probs.shape != shape or draft_probs.dtype is not dtype
                                    or draft_probs.get_device() != dev or draft_probs.stride(1) != 1):
        raise ValueError("draft_probs must match probs in shape and type, with contiguous rows")
    for name, u, n in (("u_accept", u_accept, T), ("u_draw", u_draw, B)):
        if u.dtype is not _F32 or u.shape != (n,) or not u.is_contiguous() or u.get_device() != dev:
            raise ValueError(f"{name} must be contiguous fp32 [{n}] on {_name(dev)}")
    if dev < 0:
        return verify_tree_ref(probs, tokens, parents, q_start, max_nodes, u_accept, u_draw, draft_probs)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return verify_tree(probs, tokens, parents, q_start, max_nodes, u_accept, u_draw, draft_probs)
    v = _verdict(B, max_nodes, tokens)
    N.call_packed("xtu_tree_verify", probs.data_ptr(), stride[0], _ptr(draft_probs),
                  0 if draft_probs is None else draft_probs.stride(0), dtype is _BF16, shape[1], tokens.data_ptr(),
                  parents.data_ptr(), q_start.data_ptr(), u_accept.data_ptr(), u_draw.data_ptr(), B, T, max_nodes,
                  v.accepted.data_ptr(), v.path.data_ptr(), v.tokens.data_ptr(), v.last_row.data_ptr(), _status(dev),
                  _stream(dev))
    return v


# ---------------------------------------------------------------------------
# cache commit
# ---------------------------------------------------------------------------
def commit_tree_ref(k_caches, v_caches, path, accepted, q_start, kv_len, block_table) -> None:
    qs, kl, acc, pth, bt = q_start.tolist(), kv_len.tolist(), accepted.tolist(), path.tolist(), block_table.tolist()
    fp8, nb = k_caches[0].dtype == _FP8, k_caches[0].shape[0]

    def page(b, slot):      # -1: the cache has none
        col = slot // KV_BLOCK
        return bt[b][col] if col < len(bt[b]) and 0 <= bt[b][col] < nb else -1

    for b in range(len(kl)):
        n = qs[b + 1] - qs[b]
        ctx = kl[b] - n
        if ctx < 0:
            continue
        for j in range(1, min(acc[b], path.shape[1] - 1, n - 1) + 1):
            if not j < pth[b][j] < n:
                continue
            f, t = ctx + pth[b][j], ctx + j
            fb, tb = page(b, f), page(b, t)
            if fb < 0 or tb < 0:
                continue
            for k, v in zip(k_caches, v_caches):
                if fp8:
                    k, v = k.view(torch.uint8), v.view(torch.uint8)
                    v[tb, :, :, t % KV_BLOCK] = v[fb, :, :, f % KV_BLOCK]
                else:
                    v[tb, :, t % KV_BLOCK] = v[fb, :, f % KV_BLOCK]
                k[tb, :, t % KV_BLOCK] = k[fb, :, f % KV_BLOCK]


def commit_tree(k_caches, v_caches, path: torch.Tensor, accepted: torch.Tensor, q_start: torch.Tensor,
                kv_len: torch.Tensor, block_table: torch.Tensor) -> None:
    """Move the accepted nodes' K / V behind the context, in place: of every sequence and layer slot
    context + path[j] to slot context + j, j = 1 .. accepted (``path`` and ``accepted`` of a
    :class:`TreeVerdict`; ``q_start``, ``kv_len``, ``block_table`` those of the step).

    k_caches / v_caches: one cache per layer, of one shape (layers of other head counts take a
    call of their own), as sequences of tensors or as one tensor with the layers in front; bf16
    or fp8 (V transposed inside each block).  A path must rise (a parent lies below its
    children): entry j names a node above j, or j itself, which is in place.  Entries that name
    none such, and moves from or to a slot outside the table or the cache, move nothing; nor does a
    sequence of fewer keys than nodes (padding)."""
    stacked = isinstance(k_caches, torch.Tensor) and isinstance(v_caches, torch.Tensor)
    if stacked:
        if k_caches.dim() != 5 or v_caches.dim() != 5:
            raise ValueError("stacked caches are [layers, blocks, Hkv, 64, D]")
        k0, v0 = k_caches, v_caches
        L, *kshape = k0.shape
        Lv, *vshape = v0.shape
    else:
        L, Lv = len(k_caches), len(v_caches)
        if L == 0 or L != Lv:
            raise ValueError("commit_tree takes as many K as V caches")
        k0, v0 = k_caches[0], v_caches[0]
        kshape, vshape = list(k0.shape), list(v0.shape)
        if len(kshape) != 4 or len(vshape) != 4:
            raise ValueError("caches are [blocks, Hkv, 64, D] per layer")
    if L == 0 or L != Lv:
        raise ValueError("commit_tree takes as many K as V caches")
    dev, dtype = k0.get_device(), k0.dtype
    nb, Hk, bs, D = kshape
    fp8 = dtype is _FP8
    Dv = vshape[2] if fp8 else vshape[3]
    if vshape != ([nb, Hk, Dv, bs] if fp8 else [nb, Hk, bs, Dv]):
        raise ValueError(f"K and V caches {tuple(kshape)} and {tuple(vshape)} do not match")
    if bs != KV_BLOCK:
        raise ValueError(f"KV blocks hold 64 tokens, not {bs}")
    if not fp8 and dtype is not _BF16 and dev >= 0:
        raise ValueError(f"the caches must be bfloat16 or float8_e4m3fn, not {dtype}")
    B, P = path.shape
    _ints("path", path, (B, P), dev)
    _ints("accepted", accepted, (B,), dev)
    _ints("q_start", q_start, (B + 1,), dev)
    _ints("kv_len", kv_len, (B,), dev)
    bt_stride, bt_cols = _table(block_table, B, dev)
    kfull, vfull = k0.shape, v0.shape
    for k, v in ((k0, v0),) if stacked else zip(k_caches, v_caches):
        if (k.shape != kfull or v.shape != vfull or k.dtype is not dtype or v.dtype is not dtype
                or k.get_device() != dev or v.get_device() != dev):
            raise ValueError("the layers' caches must be alike")
        if not k.is_contiguous() or not v.is_contiguous():
            raise ValueError("the caches must be contiguous")
    if dev < 0:
        commit_tree_ref(k_caches, v_caches, path, accepted, q_start, kv_len, block_table)
        return
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return commit_tree(k_caches, v_caches, path, accepted, q_start, kv_len, block_table)
    es = k0.element_size()
    if D * es % 16 or (not fp8 and Dv * es % 16):
        raise ValueError("head rows must be multiples of 16 bytes")
    kp = vp = kb = ks = vb = vs = 0
    if stacked:
        kb, ks, vb, vs = k0.data_ptr(), k_caches.stride(0) * es, v0.data_ptr(), v_caches.stride(0) * es
        odd = (kb | ks | vb | vs) & 15
    else:
        kl, vl = [k.data_ptr() for k in k_caches], [v.data_ptr() for v in v_caches]
        lists = array("q", kl + vl)            # (lives until the call is over)
        kp = lists.buffer_info()[0]
        vp = kp + 8 * L
        odd = any(x & 15 for x in kl) or any(x & 15 for x in vl)
    if odd:
        raise ValueError("the caches must start on 16-byte boundaries")
    N.call_packed("xtu_tree_commit", kp, vp, kb, ks, vb, vs, L, path.data_ptr(), P, accepted.data_ptr(),
                  q_start.data_ptr(), kv_len.data_ptr(), block_table.data_ptr(), bt_stride, bt_cols, B, nb, Hk, D * es,
                  Dv * es, fp8, Dv, _stream(dev))
