"""Workloads of the operators of ordinary attention layers that stand between 2-simplicial ones.

Four operators, as a decoder uses them one after the other:

  rotary     rotation of q and k by the angles of their positions            ``rotary_embedding``
  attention  causal attention over whole prompts, grouped heads, sequences
             of one length in a batch or packed one behind the other         ``causal_attention``
  append     new keys and values into the pages of a cache                   ``cache_append``
  tree       drafted tokens (or single ones) over the cache                  ``tree_attention``

``mode`` is "forward" or "train" (forward and backward).  ``own`` false: the plain torch forms, in 32 bits.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}

# The largest listed cases: heads * (longest sequence)^2 * sequences of a prompt, bytes of a cache, elements of a rotation
_MOST_SCORES = 8 * 16384 ** 2
_MOST_TRAIN_SCORES = 16 * 8192 ** 2
_MOST_CACHE = 1 << 30
_MOST_ROTATED = 16384 * 20 * 128


def listed():
    rows = (
        # four sequences that get one token each: latency, the angles of far positions
        ("rotary_tokens", dict(op="rotary", mode="forward", dtype="bf16", S=4, T=4, tail=0, H=16, HK=4, D=128, rot=128,
                               interleaved=False, positions="far", mix=1)),
        # q and k of a packed training batch as views of one fused projection, half of each head rotated
        ("rotary_train", dict(op="rotary", mode="train", dtype="bf16", S=7, T=16384, tail=0, H=16, HK=4, D=128, rot=64,
                              interleaved=True, positions="packed", mix=2)),
        # a unit-test sized batch in full precision, one sequence of a single token among it
        ("attention_small_fp32_train", dict(op="attention", mode="train", dtype="fp32", packed=True, S=4, T=323, L=0,
                                            tail=5, H=4, HK=2, D=64, mix=3)),
        # the middle-sized layer of the benchmark's sweeps: B2 H8 N2048, head_dim 64, every head its own keys
        ("attention_middle_train", dict(op="attention", mode="train", dtype="bf16", packed=False, S=2, T=4096, L=2048,
                                        tail=0, H=8, HK=8, D=64, mix=4)),
        # prompts of a serving batch, packed, with the rows behind the last one that its padding leaves
        ("attention_prompts", dict(op="attention", mode="forward", dtype="bf16", packed=True, S=6, T=8100, L=0,
                                   tail=92, H=16, HK=4, D=128, mix=5)),
        # a training step at the benchmark's headline length and heads
        ("attention_headline_train", dict(op="attention", mode="train", dtype="bf16", packed=False, S=1, T=8192, L=8192,
                                          tail=0, H=16, HK=4, D=128, mix=6)),
        # one long prompt
        ("attention_long", dict(op="attention", mode="forward", dtype="fp16", packed=False, S=1, T=16384, L=16384,
                                tail=0, H=8, HK=2, D=128, mix=7)),
        # accepted draft tokens of a serving batch
        ("append_accepted", dict(op="append", mode="rows", dtype="bf16", S=16, T=16, HK=4, D=128, page=16, cap=2048, mix=8)),
        # the prompts of a serving batch
        ("append_prompts", dict(op="append", mode="packed", dtype="bf16", S=6, T=8100, HK=4, D=128, page=64, cap=8192, mix=9)),
        # single tokens of a small serving batch
        ("tree_single_tokens", dict(op="tree", mode="forward", dtype="bf16", S=8, T=1, H=16, HK=4, D=128, page=16,
                                    cap=4096, mix=10)),
        # drafted trees over middle lengths, head_dim 64, no pages, sequences with fewer drafts than others
        ("tree_middle", dict(op="tree", mode="forward", dtype="fp16", S=5, T=23, H=8, HK=8, D=64, page=0, cap=3000, mix=11)),
        # large trees over long caches
        ("tree_long", dict(op="tree", mode="forward", dtype="bf16", S=4, T=48, H=16, HK=4, D=128, page=64, cap=65536, mix=12)),
    )
    return [dict(case, name=name) for name, case in rows]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        c = {"rotary": _draw_rotary, "attention": _draw_attention, "append": _draw_append, "tree": _draw_tree}[
            rng.choice(("rotary", "attention", "attention", "append", "tree", "tree"))](rng)
        if c is not None:
            return c


def _draw_heads(rng):
    hk = rng.choice((1, 2, 4, 8))
    return hk * rng.choice((1, 2, 3, 4, 8)), hk


def _draw_rotary(rng):
    H, HK = _draw_heads(rng)
    D = rng.choice((32, 64, 80, 128))
    S = _log_int(rng, 1, 16)
    T = max(S, _log_int(rng, 1, 16384))
    if T * (H + HK) * D > _MOST_ROTATED:
        return None
    return dict(op="rotary", mode=rng.choice(("forward", "train")), dtype=rng.choice(("bf16", "bf16", "fp16", "fp32")),
                S=S, T=T, tail=0, H=H, HK=HK, D=D, rot=rng.choice((D, D // 2)), interleaved=rng.random() < 0.5,
                positions=rng.choice(("far", "packed")), mix=rng.randrange(1 << 20))


def _draw_attention(rng):
    H, HK = _draw_heads(rng)
    mode = rng.choice(("forward", "train"))
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp32"))
    packed = rng.random() < 0.5
    S, L = _log_int(rng, 1, 12), _log_int(rng, 1, 16384)
    c = dict(op="attention", mode=mode, dtype=dtype, packed=packed, S=S, T=S * L, L=0 if packed else L,
             tail=rng.choice((0, 0, 37)) if packed else 0, H=H, HK=HK, D=rng.choice((32, 64, 64, 80, 128, 128)),
             mix=rng.randrange(1 << 20))
    most = _MOST_SCORES if mode == "forward" else _MOST_TRAIN_SCORES
    longest = max(_lengths(c))
    if S * H * longest ** 2 * (8 if dtype == "fp32" else 1) > most or S * L * (H + HK) > 16384 * 40:
        return None
    return c


def _draw_append(rng):
    hk, D = rng.choice((1, 2, 4, 8)), rng.choice((32, 64, 80, 128))
    mode = rng.choice(("rows", "packed"))
    S, page = _log_int(rng, 1, 16), rng.choice((0, 16, 64, 256))
    T = _log_int(rng, 1, 64) if mode == "rows" else S * _log_int(rng, 1, 2048)
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    c = dict(op="append", mode=mode, dtype=dtype, S=S, T=T, HK=hk, D=D, page=page, cap=0, mix=rng.randrange(1 << 20))
    cap = 2 * (T if mode == "rows" else max(_lengths(c))) + rng.randint(16, 1024)
    c["cap"] = cap if page == 0 else -(-cap // page) * page
    return c if 2 * S * c["cap"] * hk * D * _SIZE[dtype] <= _MOST_CACHE else None


def _draw_tree(rng):
    H, HK = _draw_heads(rng)
    page = rng.choice((0, 16, 16, 64, 256))
    cap = _log_int(rng, 16, 65536)
    cap = cap if page == 0 else -(-cap // page) * page
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    c = dict(op="tree", mode="forward", dtype=dtype, S=_log_int(rng, 1, 16), T=rng.choice((1, 1, _log_int(rng, 2, 64))),
             H=H, HK=HK, D=rng.choice((32, 64, 80, 128)), page=page, cap=cap, mix=rng.randrange(1 << 20))
    return c if 2 * c["S"] * cap * HK * c["D"] * _SIZE[dtype] <= _MOST_CACHE and c["S"] * c["T"] * H * cap <= 1 << 28 else None


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
    lens = lens[:1] + fixed + lens[1:]
    return lens


def _cached(c):
    """Rows that each sequence of a cache holds already: any number up to what leaves room, one of them none."""
    rng = random.Random(c["mix"] + 1)
    room = c["cap"] - (c["T"] if c["mode"] == "rows" else max(_lengths(c)) if c["mode"] == "packed" else 0)
    held = [int(room * rng.uniform(0.5, 1.0)) for _ in range(c["S"])]
    if c["S"] >= 4:
        held[2] = 0
    return held


def _taken(c):
    """Accepted nodes of each sequence's draft, as rows of the draft in the order of their path."""
    rng = random.Random(c["mix"] + 2)
    return [sorted(rng.sample(range(c["T"]), rng.randint(0 if c["S"] > 1 else 1, min(c["T"], 8)))) for _ in range(c["S"])]


def _parents(c):
    """A drafted tree per sequence: node 0 hangs on the last cached token, most others on an earlier node, some on the
    cached token too; sequences from the second on may have fewer nodes, the places left over are -2."""
    rng = random.Random(c["mix"] + 3)
    rows = []
    for s in range(c["S"]):
        n = c["T"] if s == 0 else rng.randint(max(1, c["T"] // 2), c["T"])
        rows.append([-1] + [rng.choice((-1, rng.randrange(i), rng.randrange(i), i - 1, i - 1)) for i in range(1, n)] + [-2] * (c["T"] - n))
    return rows


def prepare(case, seed):
    c, dev = case, torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(seed)
    dtype = _DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    def ints(x, kind=torch.int32):
        return torch.tensor(x, dtype=kind, device=dev)

    D, state = c["D"], {"case": c}
    if c["op"] in ("rotary", "attention") or c["mode"] == "packed":
        ends = [0]
        for n in _lengths(c):
            ends.append(ends[-1] + n)
        state["cu"] = ints(ends)
    if c["op"] == "rotary":
        fused = normal(c["T"], c["H"] + 2 * c["HK"], D)               # what the projection leaves: q, k and v side by side
        leaves = [fused[:, :c["H"]], fused[:, c["H"]:c["H"] + c["HK"]]]
        state["frequencies"] = 10000.0 ** (-torch.arange(0, c["rot"], 2, device=dev, dtype=torch.float64) / c["rot"])
        state["positions"] = None
        if c["positions"] == "far":
            state["positions"] = torch.randint(0, 1 << 20, (c["T"],), generator=g, device=dev, dtype=torch.int32)
        if c["mode"] == "train":
            leaves = [t.detach().requires_grad_(True) for t in leaves]
            state["douts"] = [normal(c["T"], c["H"], D), normal(c["T"], c["HK"], D)]
        state["q"], state["k"] = leaves
        return state
    if c["op"] == "attention":
        lead = (c["T"] + c["tail"],) if c["packed"] else (c["S"], c["L"])
        leaves = [normal(*lead, h, D) for h in (c["H"], c["HK"], c["HK"])]
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
    if c["op"] == "append":
        lead = (S, c["T"]) if c["mode"] == "rows" else (c["T"],)
        state["k"], state["v"] = normal(*lead, c["HK"], D), normal(*lead, c["HK"], D)
        if c["mode"] == "rows":
            state["rows"] = ints([r + [-1] * (8 - len(r)) for r in _taken(c)])
        return state
    state["q"], state["k"], state["v"] = normal(S, c["T"], c["H"], D), normal(S, c["T"], c["HK"], D), normal(S, c["T"], c["HK"], D)
    state["parents"] = ints(_parents(c))
    return state


def run(state):
    c = state["case"]
    return {"rotary": _run_rotary, "attention": _run_attention, "append": _run_append, "tree": _run_tree}[c["op"]](c, state)


# ---- rotary ----------------------------------------------------------------------------------------------------------

def _run_rotary(c, s):
    q, k = s["q"], s["k"]
    if own:
        import simplical_attn_amd as sa
        q2, k2 = sa.rotary_embedding(q, k, s["frequencies"], positions=s["positions"],
                                     cu_seqlens=None if s["positions"] is not None else s["cu"], interleaved=c["interleaved"])
        if c["mode"] == "forward":
            return q2, k2
        return (q2.detach(), k2.detach(), *torch.autograd.grad((q2, k2), (q, k), s["douts"]))
    positions = s["positions"]
    if positions is None:
        rows = torch.arange(c["T"], device=q.device, dtype=torch.int32)
        sequence = torch.searchsorted(s["cu"], rows, right=True) - 1
        positions = rows - s["cu"][sequence]
    angles = positions.double()[:, None] * s["frequencies"]            # far positions: 64 bits
    cos, sin = angles.cos().float()[:, None], angles.sin().float()[:, None]
    q2, k2 = _rotated(q, cos, sin, c), _rotated(k, cos, sin, c)
    if c["mode"] == "forward":
        return q2, k2
    dq, dk = s["douts"]
    return q2.detach(), k2.detach(), _rotated(dq, cos, -sin, c), _rotated(dk, cos, -sin, c)


def _rotated(x, cos, sin, c):
    rot = c["rot"]
    y = x.detach().float()
    out = y.clone()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if c["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
    out[..., a] = y[..., a] * cos - y[..., b] * sin
    out[..., b] = y[..., b] * cos + y[..., a] * sin
    return out.to(x.dtype)


# ---- attention -------------------------------------------------------------------------------------------------------

def _run_attention(c, s):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        import simplical_attn_amd as sa
        out = sa.causal_attention(q, k, v, cu_seqlens=s["cu"] if c["packed"] else None)
        if c["mode"] == "forward":
            return out
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), s["dout"]))
    G, L = c["H"] // c["HK"], max(_lengths(c))
    scale = 1.0 / math.sqrt(c["D"])
    if c["packed"]:                                                     # sequences side by side, padded to the longest
        rows = s["cu"][:-1, None] + torch.arange(L, device=q.device, dtype=torch.int32)
        valid = rows < s["cu"][1:, None]
        rows = torch.where(valid, rows, 0).long()
        spread = lambda t: (t.detach().float()[rows] * valid[..., None, None]).transpose(1, 2).contiguous()  # noqa: E731
        gather = lambda t, like: torch.zeros(like.shape, dtype=like.dtype, device=like.device).index_put_(  # noqa: E731
            (rows[valid],), t.transpose(1, 2)[valid].to(like.dtype))
    else:
        spread = lambda t: t.detach().float().transpose(1, 2).contiguous()  # noqa: E731
        gather = lambda t, like: t.transpose(1, 2).to(like.dtype).contiguous()  # noqa: E731
    shared = lambda t: t.repeat_interleave(G, dim=1)  # noqa: E731
    qf, kf, vf = spread(q), shared(spread(k)), shared(spread(v))
    scores = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    hidden = torch.ones(L, L, dtype=torch.bool, device=q.device).triu(1)
    scores.masked_fill_(hidden, float("-inf"))
    weights = (scores - scores.amax(-1, keepdim=True)).exp_()
    weights /= weights.sum(-1, keepdim=True)
    del scores
    out = torch.matmul(weights, vf)
    if c["mode"] == "forward":
        return gather(out, q)
    df = spread(s["dout"])
    grouped = lambda t: t.unflatten(1, (c["HK"], G)).sum(2)  # noqa: E731
    dv = grouped(torch.matmul(weights.transpose(-1, -2), df))
    dweights = torch.matmul(df, vf.transpose(-1, -2))
    dscores = weights * (dweights - (weights * dweights).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(dscores, kf)
    dk = grouped(torch.matmul(dscores.transpose(-1, -2), qf))
    return gather(out, q.detach()), gather(dq, q.detach()), gather(dk, k.detach()), gather(dv, v.detach())


# ---- cache -----------------------------------------------------------------------------------------------------------

def _places(c, pages, sequence, position):
    """(first index, second index) into a cache of the rows at `position` of `sequence`."""
    if pages is None:
        return sequence, position
    return pages[sequence, position // c["page"]].long(), position % c["page"]


def _run_append(c, s):
    if own:
        import simplical_attn_amd as sa
        sa.cache_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["lengths"], page_table=s["pages"],
                        rows=s.get("rows"), cu_seqlens=s.get("cu"))
        return s["k_cache"], s["v_cache"]
    if c["mode"] == "rows":
        kept = s["rows"] >= 0
        sequence, place = kept.nonzero(as_tuple=True)
        source = (sequence, s["rows"][kept].long())
        position = s["lengths"].long()[sequence] + place
    else:
        rows = torch.arange(c["T"], device=s["k"].device, dtype=torch.int32)
        sequence = torch.searchsorted(s["cu"], rows, right=True) - 1
        source = (rows.long(),)
        position = (s["lengths"][sequence] + rows - s["cu"][sequence]).long()
    at = _places(c, s["pages"], sequence, position)
    s["k_cache"][at] = s["k"][source]
    s["v_cache"][at] = s["v"][source]
    return s["k_cache"], s["v_cache"]


def _run_tree(c, s):
    if own:
        import simplical_attn_amd as sa
        return sa.tree_attention(s["q"], s["k"], s["v"], s["parents"], s["k_cache"], s["v_cache"], s["lengths"],
                                 page_table=s["pages"])
    S, T, G, cap, dev = c["S"], c["T"], c["H"] // c["HK"], c["cap"], s["q"].device
    sequence = torch.arange(S, device=dev)[:, None].expand(S, cap)
    at = _places(c, s["pages"], sequence, torch.arange(cap, device=dev).expand(S, cap))
    keys = torch.cat((s["k_cache"][at], s["k"]), 1).float().transpose(1, 2).contiguous()       # [S, HK, cap + T, D]
    values = torch.cat((s["v_cache"][at], s["v"]), 1).float().transpose(1, 2).contiguous()
    # node i sees itself and its ancestors: the steps to a parent, taken any number of times
    nodes = torch.arange(T, device=dev, dtype=torch.int32)
    seen = (s["parents"][:, :, None] == nodes).double() + (nodes[:, None] == nodes).double()
    seen = (torch.linalg.matrix_power(seen, T) > 0).double()
    rooted = torch.matmul(seen, (s["parents"] == -1).double()[..., None]) > 0                   # [S, T, 1]
    held = torch.arange(cap, device=dev) < s["lengths"][:, None]
    visible = torch.cat((held[:, None].expand(S, T, cap), seen > 0), 2) & rooted
    q = s["q"].float().view(S, T, c["HK"], G, c["D"]).permute(0, 2, 1, 3, 4).reshape(S, c["HK"], T * G, c["D"])
    scores = (torch.matmul(q, keys.transpose(-1, -2)) / math.sqrt(c["D"])).unflatten(2, (T, G))
    scores.masked_fill_(~visible[:, None, :, None], torch.finfo(torch.float32).min)
    weights = (scores - scores.amax(-1, keepdim=True)).exp_() * rooted[:, None, :, None]
    sums = weights.sum(-1, keepdim=True)
    weights /= torch.where(sums > 0, sums, 1.0)
    out = torch.matmul(weights.flatten(2, 3), values).unflatten(2, (T, G))
    return out.permute(0, 2, 1, 3, 4).reshape(S, T, c["H"], c["D"]).to(s["q"].dtype)


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "attention": _exact_attention, "append": _exact_append, "tree": _exact_tree}[case["op"]](case, s)


def _exact_rotary(c, s):
    if s["positions"] is not None:
        positions = s["positions"].double()
    else:
        positions = torch.cat([torch.arange(n, dtype=torch.float64, device=s["q"].device) for n in _lengths(c)])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=positions.device), torch.outer(positions, s["frequencies"]))[:, None]

    def rotate(x, turn):
        x = x.detach().double()
        head, rest = x[..., :c["rot"]], x[..., c["rot"]:]
        pairs = head.unflatten(-1, (-1, 2)) if c["interleaved"] else torch.stack(head.chunk(2, -1), -1)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        head = z.flatten(-2) if c["interleaved"] else torch.cat((z[..., 0], z[..., 1]), -1)
        return torch.cat((head, rest), -1)

    outs = [rotate(s["q"], turn), rotate(s["k"], turn)]
    if c["mode"] == "train":
        outs += [rotate(d, turn.conj()) for d in s["douts"]]
    return tuple(outs)


def _exact_attention(c, s):
    lens, G = _lengths(c), c["H"] // c["HK"]
    train = c["mode"] == "train"
    if sum(n * n for n in lens) * c["H"] * c["D"] * (20 if train else 4) > 2e13:
        return None
    flat = lambda t: t.detach().reshape(-1, t.shape[-2], t.shape[-1]).double()  # noqa: E731
    q, k, v = flat(s["q"]), flat(s["k"]), flat(s["v"])
    do = flat(s["dout"]) if train else None
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    start = 0
    for n in lens:
        r = slice(start, start + n)
        start += n
        for h in range(c["H"] if n else 0):
            Q, K, V = q[r, h], k[r, h // G], v[r, h // G]
            P = torch.softmax((Q @ K.T / math.sqrt(c["D"])).masked_fill(~torch.ones(n, n, dtype=torch.bool, device=q.device).tril(), -math.inf), -1)
            out[r, h] = P @ V
            if train:
                dO = do[r, h]
                dS = P * (dO @ V.T - (dO * out[r, h]).sum(-1, keepdim=True)) / math.sqrt(c["D"])
                dq[r, h] = dS @ K
                dk[r, h // G] += dS.T @ Q
                dv[r, h // G] += P.T @ dO
    outs = [out.view(s["q"].shape)]
    if train:
        outs += [dq.view(s["q"].shape), dk.view(s["k"].shape), dv.view(s["v"].shape)]
    return tuple(outs) if train else outs[0]


def _exact_append(c, s):
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    held, ends = _cached(c), [0]
    for n in (_lengths(c) if c["mode"] == "packed" else []):
        ends.append(ends[-1] + n)
    for b in range(c["S"]):
        source = (b, torch.tensor(_taken(c)[b], dtype=torch.int64)) if c["mode"] == "rows" else slice(ends[b], ends[b + 1])
        for cache, new in zip(caches, (s["k"], s["v"])):
            rows = new[source].double()
            at = torch.arange(held[b], held[b] + len(rows), device=cache.device)
            if s["pages"] is None:
                cache[b, at] = rows
            else:
                cache.flatten(0, 1)[s["pages"][b].long()[at // c["page"]] * c["page"] + at % c["page"]] = rows
    return tuple(caches)


def _exact_tree(c, s):
    G, held, parents = c["H"] // c["HK"], _cached(c), _parents(c)
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
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
        for i, p in enumerate(parents[b]):                             # a parent stands before its children
            if p != -2:
                mask[i, :n] = True
                mask[i, n:] = mask[p, n:] if p >= 0 else False
                mask[i, n + i] = True
        mask = mask.to(K.device)
        real = torch.tensor([p != -2 for p in parents[b]], device=K.device)
        for h in range(c["H"]):
            score = (s["q"][b, :, h].double() @ K[:, h // G].T / math.sqrt(c["D"])).masked_fill(~mask, -math.inf)
            out[b, real, h] = torch.softmax(score[real], -1) @ V[:, h // G]
    return out


def work(case):
    c = case
    size, D = _SIZE[c["dtype"]], c["D"]
    if c["op"] == "rotary":
        elements = c["T"] * (c["H"] + c["HK"]) * D * (2 if c["mode"] == "train" else 1)
        return {"bytes": 2 * elements * size + c["T"] * 4, "flops": 3 * elements}
    if c["op"] == "attention":
        pairs = sum(n * (n + 1) // 2 for n in _lengths(c)) * c["H"]
        q, kv, train = (c["T"] + c["tail"]) * c["H"] * D, (c["T"] + c["tail"]) * c["HK"] * D, c["mode"] == "train"
        # forward reads q, k, v and writes out; backward reads those and dout and writes three gradients
        return {"bytes": (2 * q + 2 * kv + (4 * q + 4 * kv if train else 0)) * size, "flops": (14 if train else 4) * pairs * D}
    if c["op"] == "append":
        rows = sum(len(r) for r in _taken(c)) if c["mode"] == "rows" else c["T"]
        return {"bytes": 4 * rows * c["HK"] * D * size, "flops": 0}
    nodes, seen = c["S"] * c["T"], _cached(c)
    keys = sum(n + c["T"] for n in seen)
    return {"bytes": (2 * keys * c["HK"] + 2 * nodes * c["H"]) * D * size, "flops": 4 * keys * c["T"] * c["H"] * D}
