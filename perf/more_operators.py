"""Workloads of the operators that bound the context of ordinary attention layers: attention with a sliding window and a
few first tokens that stay visible (sinks), and the eviction of cached rows by the attention weight they have gathered.

Four operators, as a decoder over long texts uses them:

  window   causal attention over prompts, query i of a sequence over keys j with i - j < W or j < sinks,
           forward and backward                                                   ``causal_attention(window=, sinks=)``
  decode   single tokens or drafted ones over a paged cache, with such a window, or adding the weights that the
           cached rows got to a sum for each                                      ``tree_attention(window=, sinks=, weights=)``
  sums     the weight that each key of a prompt got from all queries              ``key_weights``
  evict    the rows of a cache that gathered most weight stay and close ranks     ``cache_evict``

``mode`` is "forward" or "train" (forward and backward).  ``own`` false: the plain torch forms, in 32 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

# The largest listed cases: products of a forward and of a training step, bytes of a cache
_MOST_FLOPS = 8 * 32768 * 4096 * 4 * 128
_MOST_TRAIN_FLOPS = 16 * 8192 * 512 * 14 * 128
_MOST_SCORES = 1 << 31                   # of the plain forms
_MOST_CACHE = 600 << 20


def listed():
    rows = (
        # a unit-test sized batch in full precision, one sequence empty and one a single token
        ("window_small_fp32_train", dict(op="window", mode="train", dtype="fp32", packed=True, S=4, T=323, L=0, tail=5,
                                         H=4, HK=2, D=64, W=48, sinks=2, mix=1)),
        # the middle-sized layer of the benchmark's sweeps, with the keys' window of its 2-simplicial layers, no sinks
        ("window_middle_train", dict(op="window", mode="train", dtype="bf16", packed=False, S=2, T=4096, L=2048, tail=0,
                                     H=8, HK=8, D=64, W=512, sinks=0, mix=2)),
        # prompts of a serving batch, packed, with the rows behind the last one that its padding leaves
        ("window_prompts", dict(op="window", mode="forward", dtype="bf16", packed=True, S=6, T=8100, L=0, tail=92,
                                H=16, HK=4, D=128, W=1024, sinks=4, mix=3)),
        # a training step at the benchmark's headline length, heads and window
        ("window_headline_train", dict(op="window", mode="train", dtype="bf16", packed=False, S=1, T=8192, L=8192, tail=0,
                                       H=16, HK=4, D=128, W=512, sinks=4, mix=4)),
        # one long prompt
        ("window_long", dict(op="window", mode="forward", dtype="fp16", packed=False, S=1, T=32768, L=32768, tail=0,
                             H=8, HK=2, D=128, W=4096, sinks=4, mix=5)),
        # single tokens of a small serving batch whose caches are much longer than the window
        ("decode_window_tokens", dict(op="decode", dtype="bf16", S=8, T=1, H=16, HK=4, D=128, page=16, cap=32768, W=1024,
                                      sinks=4, add=False, mix=6)),
        # drafted trees over middle lengths, head_dim 64, no pages
        ("decode_window_trees", dict(op="decode", dtype="fp16", S=5, T=23, H=8, HK=8, D=64, page=0, cap=3000, W=512,
                                     sinks=1, add=False, mix=7)),
        # single tokens of a serving batch that adds up the weights its cached rows get
        ("decode_weights", dict(op="decode", dtype="bf16", S=16, T=1, H=16, HK=4, D=128, page=64, cap=4096, W=0, sinks=0,
                                add=True, mix=8)),
        # what the keys of a unit-test sized batch were worth
        ("sums_small_fp32", dict(op="sums", dtype="fp32", packed=True, S=3, T=217, L=0, tail=0, H=4, HK=2, D=64, W=0,
                                 sinks=0, mix=9)),
        # the same of a serving batch's prompts, before their keys go into the cache
        ("sums_prompts", dict(op="sums", dtype="bf16", packed=True, S=6, T=8100, L=0, tail=92, H=16, HK=4, D=128, W=0,
                              sinks=0, mix=10)),
        # a serving batch's full caches halved
        ("evict_batch", dict(op="evict", dtype="bf16", S=8, HK=4, D=128, page=16, cap=2048, keep=1024, first=4, recent=256,
                             shared=False, mix=11)),
        # long caches cut to a quarter
        ("evict_long", dict(op="evict", dtype="bf16", S=4, HK=4, D=128, page=64, cap=65536, keep=16384, first=4,
                            recent=1024, shared=False, mix=12)),
    )
    return [dict(case, name=name) for name, case in rows]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        c = {"window": _draw_window, "decode": _draw_decode, "sums": _draw_sums, "evict": _draw_evict}[
            rng.choice(("window", "window", "window", "decode", "decode", "sums", "evict"))](rng)
        if c is not None:
            return c


def _draw_heads(rng):
    hk = rng.choice((1, 2, 4, 8))
    return hk * rng.choice((1, 2, 3, 4, 8)), hk


def _draw_rows(rng):
    packed = rng.random() < 0.5
    H, HK = _draw_heads(rng)
    S, L = _log_int(rng, 1, 12), _log_int(rng, 1, 32768)
    return dict(dtype=rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32")), packed=packed, S=S, T=S * L, L=0 if packed else L,
                tail=rng.choice((0, 0, 37)) if packed else 0, H=H, HK=HK, D=rng.choice((32, 64, 64, 80, 128, 128)),
                mix=rng.randrange(1 << 20))


def _draw_window(rng):
    c = dict(op="window", mode=rng.choice(("forward", "train")), **_draw_rows(rng))
    c["W"] = rng.choice((_log_int(rng, 1, 4096), 1 << rng.randint(4, 12)))
    c["sinks"] = rng.choice((0, 1, 4, 4, rng.randint(1, 150)))
    if c["mode"] == "train" and (c["W"] < 2 or max(_lengths(c)) < 2):     # (nothing but each row's own key: dq and dk are zero)
        return None
    most = _MOST_FLOPS if c["mode"] == "forward" else _MOST_TRAIN_FLOPS
    return c if work(c)["flops"] * (8 if c["dtype"] == "fp32" else 1) <= most and _scores(c) <= _MOST_SCORES and c["T"] * (c["H"] + c["HK"]) <= 32768 * 20 else None


def _draw_sums(rng):
    c = dict(op="sums", **_draw_rows(rng))
    c["W"], c["sinks"] = rng.choice(((0, 0), (0, 0), (_log_int(rng, 16, 2048), 4)))
    return c if work(c)["flops"] * (8 if c["dtype"] == "fp32" else 1) <= _MOST_FLOPS / 4 and _scores(c) <= _MOST_SCORES / 2 and c["T"] * (c["H"] + c["HK"]) <= 32768 * 20 else None


def _draw_decode(rng):
    H, HK = _draw_heads(rng)
    page = rng.choice((0, 16, 16, 64, 256))
    cap = _log_int(rng, 16, 65536)
    cap = cap if page == 0 else -(-cap // page) * page
    add = rng.random() < 0.4
    T = 1 if add else rng.choice((1, 1, _log_int(rng, 2, 64)))
    W, sinks = (_log_int(rng, 1, 8192), rng.choice((0, 1, 4, 40))) if not add or rng.random() < 0.3 else (0, 0)
    c = dict(op="decode", dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), S=_log_int(rng, 1, 16), T=T, H=H, HK=HK,
             D=rng.choice((32, 64, 80, 128)), page=page, cap=cap, W=W, sinks=sinks, add=add, mix=rng.randrange(1 << 20))
    seen = min(cap, W + sinks) if W else cap
    return c if 2 * c["S"] * cap * HK * c["D"] * _SIZE[c["dtype"]] <= _MOST_CACHE and c["S"] * T * H * seen <= 1 << 26 else None


def _draw_evict(rng):
    page = rng.choice((0, 16, 64, 256))
    cap = _log_int(rng, 16, 65536)
    cap = cap if page == 0 else -(-cap // page) * page
    keep = rng.randint(max(1, cap // 8), cap)
    c = dict(op="evict", dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")), S=_log_int(rng, 1, 16), HK=rng.choice((1, 2, 4, 8)),
             D=rng.choice((32, 64, 80, 128)), page=page, cap=cap, keep=keep, first=min(keep, rng.choice((0, 1, 4))), recent=0,
             shared=rng.random() < 0.3, mix=rng.randrange(1 << 20))
    c["recent"] = rng.randint(0, (c["keep"] - c["first"]) // 2)
    return c if 2 * c["S"] * cap * c["HK"] * c["D"] * _SIZE[c["dtype"]] <= _MOST_CACHE else None


def _lengths(c):
    """Lengths of the packed sequences, summing to T: from four on one of them is empty, from three on one a single token."""
    S, T = c["S"], c["T"]
    if c.get("L"):
        return [c["L"]] * S
    rng = random.Random(c["mix"])
    fixed = [0] * (S >= 4) + [1] * (S >= 3 and T >= 1)
    parts = [rng.expovariate(1.0) + 0.2 for _ in range(S - len(fixed))]
    left = T - sum(fixed)
    lens = [int(left * p / sum(parts)) for p in parts]
    lens[0] += left - sum(lens)
    return lens[:1] + fixed + lens[1:]


def _cached(c):
    """Rows that each sequence of a cache holds: any number up to what leaves room, one of them none; full ones to evict from."""
    rng = random.Random(c["mix"] + 1)
    room = c["cap"] - c.get("T", 0)
    room = max(room, 0)
    held = [int(room * rng.uniform(0.9 if c["op"] == "evict" else 0.5, 1.0)) for _ in range(c["S"])]
    if c["S"] >= 5:
        held[2] = 0
    return held


def _parents(c):
    """A drafted tree per sequence: node 0 hangs on the last cached token, most others on an earlier node, some on the
    cached token too; sequences from the second on may have fewer nodes, the places left over are -2."""
    rng = random.Random(c["mix"] + 3)
    rows = []
    for s in range(c["S"]):
        n = c["T"] if s == 0 else rng.randint(max(1, c["T"] // 2), c["T"])
        rows.append([-1] + [rng.choice((-1, rng.randrange(i), rng.randrange(i), i - 1, i - 1)) for i in range(1, n)] + [-2] * (c["T"] - n))
    return rows


def _pairs(c):
    """Visible pairs of query and key of a prompt's head, summed over its sequences."""
    total = 0
    for n in _lengths(c):
        w = min(c["W"], n) if c["W"] else n
        total += w * (w + 1) // 2 + (n - w) * w
        if c["W"] and n > w:
            total += sum(min(c["sinks"], i - w + 1) for i in range(w, min(n, w + c["sinks"]))) + max(0, n - w - c["sinks"]) * c["sinks"]
    return total


def _block(c, L):
    """Queries of a block of the plain forms, and the keys that one gathers."""
    if not c["W"] or c["W"] >= L:
        return L, L
    rows = min(L, max(c["W"], 64))
    return rows, c["W"] - 1 + rows + c["sinks"]


def _scores(c):
    L = max(max(_lengths(c)), 1)
    rows, keys = _block(c, L)
    return c["S"] * c["H"] * -(-L // rows) * rows * keys


def prepare(case, seed):
    c, dev = case, torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    D, state = c["D"], {"case": c}
    if c["op"] in ("window", "sums"):
        ends = [0]
        for n in _lengths(c):
            ends.append(ends[-1] + n)
        state["cu"] = ints(ends)
        lead = (c["T"] + c["tail"],) if c["packed"] else (c["S"], c["L"])
        leaves = [normal(*lead, h, D) for h in ((c["H"], c["HK"], c["HK"]) if c["op"] == "window" else (c["H"], c["HK"]))]
        if c["op"] == "sums":
            state["q"], state["k"] = leaves
            state["lse"] = _log_sums(c, state)         # the attention that ran before left it
            return state
        if c["mode"] == "train":
            leaves = [t.requires_grad_(True) for t in leaves]
            state["dout"] = normal(*lead, c["H"], D)
        state["q"], state["k"], state["v"] = leaves
        return state
    # a cache: pages in no order, or one piece per sequence
    S, page = c["S"], c["page"]
    state["lengths"] = ints(_cached(c))
    shape = (S, c["cap"], c["HK"], D) if page == 0 else (S * c["cap"] // page, page, c["HK"], D)
    state["k_cache"], state["v_cache"] = normal(*shape), normal(*shape)
    state["pages"] = None
    if page:
        state["pages"] = torch.randperm(shape[0], generator=g, device=dev).to(torch.int32).view(S, -1)
    heads = 1 if c["op"] == "evict" and c["shared"] else c["HK"]
    if c["op"] == "evict" or c["add"]:
        # what rows gather: a few much, most little, those behind a window nothing at all (equal ones)
        gathered = torch.randn(S, heads, c["cap"], generator=g, device=dev).mul_(2).exp_()
        gathered *= torch.rand(S, heads, c["cap"], generator=g, device=dev) > 0.1
        state["weights"] = gathered
    if c["op"] == "evict":
        return state
    state["q"], state["k"], state["v"] = normal(S, c["T"], c["H"], D), normal(S, c["T"], c["HK"], D), normal(S, c["T"], c["HK"], D)
    state["parents"] = ints(_parents(c))
    return state


def run(state):
    c = state["case"]
    return {"window": _run_window, "decode": _run_decode, "sums": _run_sums, "evict": _run_evict}[c["op"]](c, state)


# ---- prompts ---------------------------------------------------------------------------------------------------------

def _sides(c, cu):
    """(spread, gather): rows of a batch or of packed sequences to [S, heads, L, D] in 32 bits, padded to the longest, and back."""
    L = max(_lengths(c))
    if not c["packed"]:
        return (lambda t: t.detach().float().transpose(1, 2),
                lambda t, like: t.transpose(1, 2).to(like.dtype).contiguous())
    rows = cu[:-1, None] + torch.arange(L, device=cu.device, dtype=torch.int32)
    valid = rows < cu[1:, None]
    rows = torch.where(valid, rows, 0).long()
    return (lambda t: (t.detach().float()[rows] * valid[..., None, None]).transpose(1, 2),
            lambda t, like: torch.zeros(like.shape, dtype=like.dtype, device=like.device).index_put_(
                (rows[valid],), t.transpose(1, 2)[valid].to(like.dtype)))


def _band(c, L, dev):
    """Blocks of queries and the keys that each gathers: (rows of a block, blocks, key of [block, place], visible [block, row, place])."""
    rows, _ = _block(c, L)
    blocks = -(-L // rows)
    query = torch.arange(blocks * rows, device=dev).view(blocks, rows, 1)
    W, sinks = c["W"], c["sinks"]
    if not W or W >= L:
        at = torch.arange(L, device=dev).view(1, 1, L)
        return rows, blocks, at[:, 0], at <= query
    near = torch.arange(blocks, device=dev)[:, None] * rows - (W - 1) + torch.arange(W - 1 + rows, device=dev)
    first = torch.arange(sinks, device=dev).expand(blocks, sinks)
    seen_near = (near[:, None] >= 0) & (near[:, None] <= query) & (query - near[:, None] < W)
    seen_first = query - first[:, None] >= W
    return rows, blocks, torch.cat((near, first), 1).clamp(0, L - 1), torch.cat((seen_near, seen_first), 2)


def _blocks_of(t, c, rows, blocks):
    """[S, H, L, ...] as [S, HK, blocks, G * rows, ...], zeros behind the last row."""
    t = torch.nn.functional.pad(t, (0, 0, 0, blocks * rows - t.shape[2]))
    t = t.unflatten(1, (c["HK"], -1)).unflatten(3, (blocks, rows))
    return t.transpose(2, 3).flatten(3, 4)


def _rows_of(t, c, rows, L):
    """The other way."""
    return t.unflatten(3, (-1, rows)).transpose(2, 3).flatten(3, 4).flatten(1, 2)[:, :, :L]


def _band_scores(c, q, k, L):
    rows, blocks, at, visible = _band(c, L, q.device)
    qb, kb = _blocks_of(q, c, rows, blocks), k[:, :, at.flatten()].unflatten(2, at.shape)
    scores = torch.matmul(qb, kb.transpose(-1, -2)) * (1.0 / math.sqrt(c["D"]))
    scores.masked_fill_(~visible.repeat(1, c["H"] // c["HK"], 1), float("-inf"))
    return rows, blocks, at, qb, kb, scores


def _run_window(c, s):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        import simplical_attn_amd as sa
        out = sa.causal_attention(q, k, v, cu_seqlens=s["cu"] if c["packed"] else None, window=c["W"], sinks=c["sinks"])
        if c["mode"] == "forward":
            return out
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), s["dout"]))
    L = max(_lengths(c))
    spread, gather = _sides(c, s["cu"])
    kf, vf = spread(k), spread(v)
    rows, blocks, at, qb, kb, weights = _band_scores(c, spread(q), kf, L)
    vb = vf[:, :, at.flatten()].unflatten(2, at.shape)
    weights.sub_(weights.amax(-1, keepdim=True)).exp_()
    weights /= weights.sum(-1, keepdim=True)
    out = _rows_of(torch.matmul(weights, vb), c, rows, L)
    if c["mode"] == "forward":
        return gather(out, q)
    db = _blocks_of(spread(s["dout"]), c, rows, blocks)
    dscores = torch.matmul(db, vb.transpose(-1, -2))
    dscores = weights * (dscores - (weights * dscores).sum(-1, keepdim=True)) * (1.0 / math.sqrt(c["D"]))
    dq = _rows_of(torch.matmul(dscores, kb), c, rows, L)
    back = lambda t: torch.zeros_like(kf).index_add_(2, at.flatten(), t.flatten(2, 3))  # noqa: E731
    dk, dv = back(torch.matmul(dscores.transpose(-1, -2), qb)), back(torch.matmul(weights.transpose(-1, -2), db))
    return gather(out, q.detach()), gather(dq, q.detach()), gather(dk, k.detach()), gather(dv, v.detach())


def _log_sums(c, s):
    """log sum e^score of each query, [S, H, L] or packed [H, rows] (minus infinity in rows of no sequence)."""
    L = max(_lengths(c))
    spread, _ = _sides(c, s["cu"])
    rows, _, _, _, _, scores = _band_scores(c, spread(s["q"]), spread(s["k"]), L)
    top = scores.amax(-1, keepdim=True)
    lse = _rows_of((scores.sub_(top).exp_().sum(-1, keepdim=True).log_() + top), c, rows, L)[..., 0]
    if not c["packed"]:
        return lse.contiguous()
    out = torch.full((c["T"] + c["tail"], c["H"]), float("-inf"), device=lse.device)
    return _sides(c, s["cu"])[1](lse[..., None], out[..., None])[..., 0].T.contiguous().masked_fill_(
        torch.arange(len(out), device=lse.device) >= s["cu"][-1], float("-inf"))


def _run_sums(c, s):
    q, k, lse = s["q"], s["k"], s["lse"]
    if own:
        import simplical_attn_amd as sa
        return sa.key_weights(q, k, lse, cu_seqlens=s["cu"] if c["packed"] else None, window=c["W"] or None, sinks=c["sinks"])
    L = max(_lengths(c))
    spread, gather = _sides(c, s["cu"])
    rows, blocks, at, _, _, weights = _band_scores(c, spread(q), spread(k), L)
    lses = spread(lse.T[..., None].clamp_min(-1e30)) if c["packed"] else lse[..., None]
    weights.sub_(_blocks_of(lses, c, rows, blocks)).exp_()
    if c["packed"]:                                                     # queries behind a sequence have no weights
        real = torch.arange(L, device=q.device) < s["cu"].diff()[:, None]
        real = real[:, None, :, None].expand(-1, c["H"], -1, -1).float()
        weights *= _blocks_of(real, c, rows, blocks)
    elif blocks * rows > L:
        weights *= _blocks_of(torch.ones_like(lses), c, rows, blocks)
    sums = torch.zeros(c["S"], c["HK"], L, device=q.device).index_add_(2, at.flatten(), weights.sum(3).flatten(2, 3))
    if not c["packed"]:
        return sums
    return gather(sums[..., None], lse.new_empty(c["T"] + c["tail"], c["HK"], 1))[..., 0].T.contiguous()


# ---- cache -----------------------------------------------------------------------------------------------------------

def _places(c, pages, sequence, position):
    """(first index, second index) into a cache of the rows at `position` of `sequence`."""
    if pages is None:
        return sequence, position
    return pages[sequence, position // c["page"]].long(), position % c["page"]


def _run_decode(c, s):
    window = c["W"] or None
    if own:
        import simplical_attn_amd as sa
        out = sa.tree_attention(s["q"], s["k"], s["v"], s["parents"], s["k_cache"], s["v_cache"], s["lengths"],
                                page_table=s["pages"], window=window, sinks=c["sinks"], weights=s.get("weights"))
        return (out, s["weights"]) if c["add"] else out
    S, T, G, dev = c["S"], c["T"], c["H"] // c["HK"], s["q"].device
    held = s["lengths"][:, None].long()
    # the cached rows that some node sees: all of them, or the first ones and those of the first node's window
    if window and c["sinks"] + window - 1 < c["cap"]:
        near = held - (window - 1) + torch.arange(window - 1, device=dev)
        first = torch.arange(c["sinks"], device=dev).expand(S, -1)
        place = torch.cat((first, near), 1)
        there = torch.cat((first < held, near >= c["sinks"]), 1)
        place = place.clamp(0, c["cap"] - 1)
    else:
        place = torch.arange(c["cap"], device=dev).expand(S, -1)
        there = place < held
    at = _places(c, s["pages"], torch.arange(S, device=dev)[:, None].expand(place.shape), place)
    keys = torch.cat((s["k_cache"][at], s["k"]), 1).float().transpose(1, 2).contiguous()       # [S, HK, rows + T, D]
    values = torch.cat((s["v_cache"][at], s["v"]), 1).float().transpose(1, 2).contiguous()
    # node i sees itself and its ancestors: the steps to a parent, taken any number of times; its position counts them
    nodes = torch.arange(T, device=dev, dtype=torch.int32)
    seen = (s["parents"][:, :, None] == nodes).double() + (nodes[:, None] == nodes).double()
    seen = (torch.linalg.matrix_power(seen, T) > 0).double()
    rooted = torch.matmul(seen, (s["parents"] == -1).double()[..., None]) > 0                   # [S, T, 1]
    position = held + seen.sum(-1).long() - 1                                                   # [S, T]
    reach = window or 1 << 40
    visible = there[:, None] & ((position[..., None] - place[:, None] < reach) | (place[:, None] < c["sinks"]))
    drafted = (seen > 0) & ((position[..., None] - position[:, None] < reach) | (position[:, None] < c["sinks"]))
    visible = torch.cat((visible, drafted), 2) & rooted
    q = s["q"].float().view(S, T, c["HK"], G, c["D"]).permute(0, 2, 1, 3, 4).reshape(S, c["HK"], T * G, c["D"])
    scores = (torch.matmul(q, keys.transpose(-1, -2)) / math.sqrt(c["D"])).unflatten(2, (T, G))
    scores.masked_fill_(~visible[:, None, :, None], torch.finfo(torch.float32).min)
    weights = (scores - scores.amax(-1, keepdim=True)).exp_() * visible[:, None, :, None]
    sums = weights.sum(-1, keepdim=True)
    weights /= torch.where(sums > 0, sums, 1.0)
    out = torch.matmul(weights.flatten(2, 3), values).unflatten(2, (T, G))
    out = out.permute(0, 2, 1, 3, 4).reshape(S, T, c["H"], c["D"]).to(s["q"].dtype)
    if not c["add"]:
        return out
    each = weights.sum((2, 3))                                          # [S, HK, rows + 1]
    to = torch.cat((torch.where(there, place, c["cap"]), held.clamp(max=c["cap"])), 1)[:, None].expand(-1, c["HK"], -1)
    wide = torch.nn.functional.pad(s["weights"], (0, 1))
    s["weights"].copy_(wide.scatter_add_(2, to, each)[..., :-1])
    return out, s["weights"]


def _run_evict(c, s):
    if own:
        import simplical_attn_amd as sa
        kept, weights = sa.cache_evict(s["k_cache"], s["v_cache"], s["weights"], s["lengths"], c["keep"], first=c["first"],
                                       recent=c["recent"], page_table=s["pages"])
        return kept, weights, s["k_cache"], s["v_cache"]
    S, cap, keep, dev = c["S"], c["cap"], c["keep"], s["weights"].device
    held = s["lengths"][:, None, None].long()
    place = torch.arange(cap, device=dev)
    rank = s["weights"].masked_fill((place < c["first"]) | (place >= held - c["recent"]), float("inf"))
    rank = rank.masked_fill(place >= held, float("-inf"))
    kept = rank.sort(dim=-1, descending=True, stable=True)[1][..., :keep].sort(-1)[0]               # the lowest of equal ones first
    slot = torch.arange(keep, device=dev)
    none = slot >= held
    kept = torch.where(none, slot, kept)                                # (rows that stay where they are)
    weights = torch.zeros_like(s["weights"])
    weights[..., :keep] = s["weights"].gather(2, kept) * ~none
    rows = kept.expand(S, c["HK"], keep)
    sequence = torch.arange(S, device=dev)[:, None, None].expand(rows.shape)
    head = torch.arange(c["HK"], device=dev)[:, None].expand(rows.shape)
    source, to = (_places(c, s["pages"], sequence, r) for r in (rows, slot.expand(rows.shape)))
    for cache in (s["k_cache"], s["v_cache"]):
        cache[(*to, head)] = cache[(*source, head)]
    return kept.masked_fill(none, -1).int(), weights, s["k_cache"], s["v_cache"]


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"window": _exact_window, "decode": _exact_decode, "sums": _exact_sums, "evict": _exact_evict}[case["op"]](case, s)


def _near(c, lo, hi, first, n, dev):
    """What queries lo .. hi-1 see of keys first .. n-1."""
    i, j = torch.arange(lo, hi, device=dev)[:, None], torch.arange(first, n, device=dev)
    seen = j <= i
    return seen & ((i - j < c["W"]) | (j < c["sinks"])) if c["W"] else seen


def _exact_window(c, s):
    G, train, W, step = c["H"] // c["HK"], c["mode"] == "train", c["W"], 2048
    if sum(min(n, step) * (min(n, step) + W + c["sinks"]) * -(-n // step) for n in _lengths(c)) * c["H"] * c["D"] * (20 if train else 4) > 2e13:
        return None
    flat = lambda t: t.detach().reshape(-1, t.shape[-2], t.shape[-1]).double()  # noqa: E731
    q, k, v = flat(s["q"]), flat(s["k"]), flat(s["v"])
    do = flat(s["dout"]) if train else None
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    start = 0
    for n in _lengths(c):
        for h in range(c["H"]):
            for lo in range(0, n, step):
                hi = min(n, lo + step)
                low = max(0, lo - W + 1)
                at = torch.cat((torch.arange(min(c["sinks"], low)), torch.arange(low, hi))).to(q.device)
                seen = _near(c, lo, hi, 0, hi, q.device)[:, at]
                rows, at = slice(start + lo, start + hi), at + start
                Q, K, V = q[rows, h], k[at, h // G], v[at, h // G]
                P = torch.softmax((Q @ K.T / math.sqrt(c["D"])).masked_fill(~seen, -math.inf), -1)
                out[rows, h] = P @ V
                if train:
                    dO = do[rows, h]
                    dS = P * (dO @ V.T - (dO * out[rows, h]).sum(-1, keepdim=True)) / math.sqrt(c["D"])
                    dq[rows, h] = dS @ K
                    dk[at, h // G] += dS.T @ Q
                    dv[at, h // G] += P.T @ dO
        start += n
    outs = [out.view(s["q"].shape)]
    if train:
        outs += [dq.view(s["q"].shape), dk.view(s["k"].shape), dv.view(s["v"].shape)]
    return tuple(outs) if train else outs[0]


def _exact_sums(c, s):
    G = c["H"] // c["HK"]
    flat = lambda t: t.reshape(-1, t.shape[-2], t.shape[-1]).double()  # noqa: E731
    q, k = flat(s["q"]), flat(s["k"])
    lse = s["lse"].double() if c["packed"] else s["lse"].double().transpose(0, 1).flatten(1)     # [H, rows]
    sums = torch.zeros(c["HK"], k.shape[0], dtype=torch.float64, device=k.device)
    start = 0
    for n in _lengths(c):
        for h in range(c["H"]):
            for lo in range(0, n, 2048):
                hi = min(n, lo + 2048)
                score = q[start + lo:start + hi, h] @ k[start:start + hi, h // G].T / math.sqrt(c["D"]) - lse[h, start + lo:start + hi, None]
                sums[h // G, start:start + hi] += (score.exp() * _near(c, lo, hi, 0, hi, k.device)).sum(0)
        start += n
    return sums if c["packed"] else sums.unflatten(1, (c["S"], c["L"])).transpose(0, 1)


def _exact_decode(c, s):
    G, held, parents, W = c["H"] // c["HK"], _cached(c), _parents(c), c["W"] or 1 << 40
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    sums = torch.nn.functional.pad(s["weights"].double(), (0, 1)) if c["add"] else None
    for b in range(c["S"]):
        n = held[b]
        rows = [s["k_cache"], s["v_cache"]]
        if s["pages"] is None:
            rows = [t[b, :n] for t in rows]
        else:
            used = s["pages"][b, :-(-n // c["page"])].long()
            rows = [t[used].flatten(0, 1)[:n] for t in rows]
        K, V = (torch.cat((a, new[b])).double() for a, new in zip(rows, (s["k"], s["v"])))
        mask = torch.zeros(c["T"], n + c["T"], dtype=torch.bool)
        family, depth = [], []
        for i, p in enumerate(parents[b]):                             # a parent stands before its children
            family.append(([] if p < 0 else family[p]) + [i])
            depth.append(len(family[i]) - 1)
            if p != -2:
                at = n + depth[i]
                mask[i, max(0, at - W + 1):n] = True
                mask[i, :min(c["sinks"], n)] = True
                for j in family[i]:
                    mask[i, n + j] = depth[i] - depth[j] < W or n + depth[j] < c["sinks"]
        mask = mask.to(K.device)
        real = torch.tensor([p != -2 for p in parents[b]], device=K.device)
        for h in range(c["H"]):
            score = (s["q"][b, :, h].double() @ K[:, h // G].T / math.sqrt(c["D"])).masked_fill(~mask, -math.inf)
            P = torch.softmax(score[real], -1)
            out[b, real, h] = P @ V[:, h // G]
            if c["add"]:
                sums[b, h // G, :n + 1] += P[0]
    return (out, sums[..., :-1]) if c["add"] else out


def _exact_evict(c, s):
    held = _cached(c)
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    weights = s["weights"].double().cpu()
    new = torch.zeros_like(weights)
    for b in range(c["S"]):
        for h in range(weights.shape[1]):
            n = held[b]
            row = weights[b, h, :n]
            taken = list(range(n))
            if n > c["keep"]:
                sure = list(range(c["first"])) + list(range(n - c["recent"], n))
                free = torch.arange(c["first"], n - c["recent"])
                order = free[torch.argsort(-row[free], stable=True)]
                taken = sorted(sure + order[:c["keep"] - len(sure)].tolist())
            taken = torch.tensor(taken, dtype=torch.int64)
            new[b, h, :len(taken)] = row[taken]
            taken = taken.to(caches[0].device)
            to = torch.arange(len(taken), device=taken.device)
            for cache in caches:
                heads = slice(None) if c["shared"] else slice(h, h + 1)
                if s["pages"] is None:
                    cache[b, to, heads] = cache[b, taken, heads]
                else:
                    lines, pages = cache.flatten(0, 1)[:, heads], s["pages"][b].long()
                    line = lambda r: pages[r // c["page"]] * c["page"] + r % c["page"]  # noqa: E731
                    lines[line(to)] = lines[line(taken)]
    return None, new, caches[0], caches[1]


def work(case):
    c = case
    size, D = _SIZE[c["dtype"]], c["D"]
    if c["op"] in ("window", "sums"):
        pairs = _pairs(c) * c["H"]
        q, kv = (c["T"] + c["tail"]) * c["H"] * D, (c["T"] + c["tail"]) * c["HK"] * D
        if c["op"] == "sums":
            return {"bytes": (q + kv) * size + (c["T"] + c["tail"]) * (c["H"] + c["HK"]) * 4, "flops": 2 * pairs * D}
        train = c["mode"] == "train"
        # forward reads q, k, v and writes out; backward reads those and dout and writes three gradients
        return {"bytes": (2 * q + 2 * kv + (4 * q + 4 * kv if train else 0)) * size, "flops": (14 if train else 4) * pairs * D}
    held = _cached(c)
    if c["op"] == "evict":
        # rows that are kept are moved down, their weights too; all weights are read
        kept = sum(min(n, c["keep"]) for n in held if n > c["keep"])
        heads = 1 if c["shared"] else c["HK"]
        return {"bytes": 4 * kept * c["HK"] * D * size + (sum(held) + c["S"] * (c["cap"] + c["keep"])) * heads * 4, "flops": 0}
    nodes = c["S"] * c["T"]
    keys = sum((min(n, c["W"] - 1 + c["sinks"]) if c["W"] else n) + c["T"] for n in held)
    return {"bytes": (2 * keys * c["HK"] + 2 * nodes * c["H"]) * D * size + (8 * keys * c["HK"] if c["add"] else 0), "flops": 4 * keys * c["T"] * c["H"] * D}
