"""Measured cases of the operators on the hot side of the paged KV pool (``ztcp_b200.kvcache``).

Four operators, one serving step each: ``append`` (norms of queries and keys per head, position rotation, K/V written
into their pool slots), ``attend`` (new tokens of ragged sequences over a paged pool, decode and prefill chunks, with
the log-sum-exp), ``mass`` (attention weight accumulated per page) and ``select`` (the coldest pages of every sequence,
as the block table that the egress takes, and the compacted tables).  Shapes are those of the codec's own page
configurations: GQA pages 64 x 8 x 128, MLA pages 64 x 1 x 576 with the 64 RoPE columns first and no V, and smaller
generic ones; keys carry four RoPE channels per head scaled x15, as the codec's workload does.
"""
from __future__ import annotations

import random

import torch

own = False

F16, BF16 = "float16", "bfloat16"


# ---- cases ------------------------------------------------------------------------------------------------------
def _attend(name, dtype, batch, heads, kv_heads, dim, rope, page, q_max, kv_min, kv_max, lens, op="attend"):
    return {"name": name, "op": op, "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "rope": rope, "page": page, "q_max": q_max, "kv_min": kv_min, "kv_max": kv_max, "lens": lens}


def _append(name, dtype, tokens, heads, kv_heads, dim, rope, page, interleaved, norm_from, max_pos):
    return {"name": name, "op": "append", "dtype": dtype, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "rope": rope, "page": page, "interleaved": interleaved, "norm_from": norm_from,
            "max_pos": max_pos}


def _select(name, batch, page, kv_min, kv_max, keep, sink, recent, lens):
    return {"name": name, "op": "select", "batch": batch, "page": page, "kv_min": kv_min, "kv_max": kv_max,
            "keep": keep, "sink": sink, "recent": recent, "lens": lens}


def listed():
    return [
        # one user's next token over a short prefix: a latency-bound call
        _attend("attend_decode_one", BF16, 1, 32, 8, 128, 0, 64, 1, 1021, 1021, 1),
        # a serving batch's next tokens, ragged contexts
        _attend("attend_decode_batch", BF16, 48, 32, 8, 128, 0, 64, 1, 1024, 8192, 2),
        # the same step on MLA pages (V is the latent part of K)
        _attend("attend_decode_mla", BF16, 32, 16, 1, 576, 64, 64, 1, 1000, 8100, 3),
        # prefill chunks of several requests over prefixes restored from cold pages
        _attend("attend_chunk_ragged", BF16, 5, 32, 8, 128, 0, 64, 777, 800, 8192, 4),
        # one long chunk over a long restored prefix, in the type that ingress writes
        _attend("attend_chunk_long", F16, 1, 32, 8, 128, 0, 64, 2048, 32768, 32768, 5),
        # attention weight of one decode step, per page, for a serving batch
        _attend("mass_decode_batch", BF16, 48, 32, 8, 128, 0, 64, 1, 1024, 8192, 6, "mass"),
        # attention weight of a prompt's last queries (the observation window) over long prompts
        _attend("mass_window", F16, 4, 32, 8, 128, 0, 64, 64, 9001, 32768, 7, "mass"),
        # one user's pages: a latency-bound call
        _select("select_one", 1, 64, 16384, 16384, 128, 1, 2, 8),
        # a serving batch with long contexts and small pages
        _select("select_batch", 64, 16, 1500, 65536, 1000, 4, 8, 9),
        # next tokens of a serving batch
        _append("append_decode", BF16, 48, 32, 8, 128, 128, 64, False, 0, 32768),
        # a prefill chunk's tokens, rotation of the leading half of the columns in interleaved pairs
        _append("append_chunk", F16, 8191, 32, 8, 128, 64, 64, True, 0, 65536),
        # MLA: the latent columns are normed, the 64 leading columns rotated
        _append("append_mla", BF16, 4096, 16, 1, 576, 64, 64, False, 64, 32768),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "mass", "mass", "select", "append", "append"])
    dtype = rng.choice([F16, BF16])
    if op == "select":
        page = rng.choice([16, 64])
        kv = _log(rng, 20 * page, 1 << 16)
        pages = -(-kv // page)
        return _select("", _log(rng, 1, 64), page, max(1, kv // 9), kv, max(8, int(pages * rng.uniform(0.2, 0.9))),
                       rng.randint(0, 4), rng.randint(1, 8), rng.randrange(1 << 30)) | {"op": op}
    mla = rng.random() < 0.2
    kv_heads = 1 if mla else rng.choice([1, 2, 4, 8])
    heads = rng.choice([16, 16, 32, 64, 128]) if mla else kv_heads * rng.choice([1, 2, 4, 8])
    dim, rope = (576, 64) if mla else (rng.choice([64, 128, 128]), 0)
    page = rng.choice([16, 64, 64])
    if op == "append":
        rope = 64 if mla else rng.choice([32, 64, dim])
        return _append("", dtype, _log(rng, 1, 8191), heads, kv_heads, dim, rope, page, rng.random() < 0.5,
                       64 if mla else 0, 32768)
    chunk = rng.random() < 0.5
    batch = _log(rng, 1, 4) if chunk else _log(rng, 1, 32)
    kv_max = _log(rng, 65, 16384 if batch <= 8 else 6000)
    q_max = 1
    if chunk:  # no more pairs of rows and keys than the longest listed chunk has
        most = 2048 * 32768 * 32 // (batch * heads * kv_max * (5 if mla else 1))
        q_max = min(_log(rng, 2, 64 if op == "mass" else 1500), most)
    return _attend("", dtype, batch, heads, kv_heads, dim, rope, page, q_max, max(1, kv_max // 7), kv_max,
                   rng.randrange(1 << 30), op)


def _lens(case):
    """Context length and new tokens of every sequence; the new tokens are the context's last ones."""
    r = random.Random(case["lens"])
    kv = [case["kv_max"]] + [r.randint(case["kv_min"], case["kv_max"]) for _ in range(case["batch"] - 1)]
    top = case.get("q_max", 1)
    q = [top] + [r.randint(max(1, top // 8), top) for _ in range(case["batch"] - 1)]
    return kv, [min(a, b) for a, b in zip(q, kv)]


# ---- inputs -----------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(shape, g, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _tables(lens, page, g):
    """A shuffled block table [batch, pages of the longest] over a pool a little larger than needed; unused -1."""
    pages = [-(-n // page) for n in lens]
    pool = sum(pages) + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(pages)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pool


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_attend(case, g):
    dtype = getattr(torch, case["dtype"])
    kv, q_len = _lens(case)
    T, H, D = case["page"], case["kv_heads"], case["dim"]
    table, pool = _tables(kv, T, g)
    k = torch.randn((pool, T, H, D), generator=g, device="cuda", dtype=torch.bfloat16)
    hot = torch.randint(0, case["rope"] or D // 2, (H, 4), generator=g, device="cuda")
    gain = torch.ones((H, D), device="cuda").scatter_(1, hot, 15.0)
    k = (k * gain.to(torch.bfloat16)).to(dtype)
    v = None if case["rope"] else torch.randn((pool, T, H, D), generator=g, device="cuda", dtype=dtype)
    starts = [0]
    for n in q_len:
        starts.append(starts[-1] + n)
    s = {"op": case["op"], "q": _randn((starts[-1], case["heads"], D), g, dtype), "k": k, "v": v, "table": table,
         "kv_lens": _int32(kv), "starts": _int32(starts), "q_max": max(q_len), "rope": case["rope"],
         "scale": D ** -0.5}
    if case["op"] == "attend":
        dv = D - case["rope"]
        s["out"] = torch.empty((starts[-1], case["heads"], dv), dtype=dtype, device="cuda")
        s["lse"] = torch.empty((starts[-1], case["heads"]), dtype=torch.float32, device="cuda")
    else:
        s["lse"] = _scores(s)[1]
        s["mass"] = torch.rand(table.shape, generator=g, device="cuda") * 4
        s["decay"] = 0.875
        s["out"] = torch.empty_like(s["mass"])
    return s


def _prepare_append(case, g):
    dtype = getattr(torch, case["dtype"])
    n, T, H, D, R = case["tokens"], case["page"], case["kv_heads"], case["dim"], case["rope"]
    pool = -(-n // T) + 2
    split = case["heads"] * D, H * D, (0 if case["norm_from"] else H * D)
    qkv = _randn((n, sum(split)), g, dtype)  # one projection's output; q, k and v are views of its rows
    q, k, v = (t.unflatten(1, (-1, D)) if t.shape[1] else None for t in qkv.split(split, dim=1))
    width = D - case["norm_from"]
    angle = torch.arange(case["max_pos"], device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    zeros = lambda: torch.zeros((pool, T, H, D), dtype=dtype, device="cuda")  # noqa: E731
    return {"op": "append", "q": q, "k": k, "v": v, "k_pool": zeros(), "v_pool": None if v is None else zeros(),
            "slots": torch.randperm(pool * T, generator=g, device="cuda")[:n].contiguous(),
            "positions": torch.randint(0, case["max_pos"], (n,), generator=g, device="cuda", dtype=torch.int32),
            "rope_table": torch.cat([angle.cos(), angle.sin()], dim=1).float(), "rope": R,
            "interleaved": case["interleaved"], "norm_from": case["norm_from"], "eps": 1e-6,
            "q_weight": None if case["norm_from"] else 1 + 0.1 * torch.randn(width, generator=g, device="cuda"),
            "k_weight": 1 + 0.1 * torch.randn(width, generator=g, device="cuda"),
            "q_out": torch.empty((n, case["heads"], D), dtype=dtype, device="cuda")}


def _prepare_select(case, g):
    kv, _ = _lens(case)
    table, _ = _tables(kv, case["page"], g)
    mass = torch.rand(table.shape, generator=g, device="cuda") ** 6
    mass = torch.where(torch.rand(table.shape, generator=g, device="cuda") < 0.1, 0.0, mass)  # pages nobody looked at
    B, P = table.shape
    full = lambda n, t: torch.empty(n, dtype=t, device="cuda")  # noqa: E731
    return {"op": "select", "mass": mass, "table": table, "kv_lens": _int32(kv), "page": case["page"],
            "keep": case["keep"], "sink": case["sink"], "recent": case["recent"],
            "cold_blocks": full(B * P, torch.int32), "cold_index": full(B * P, torch.int32),
            "cold_starts": full(B + 1, torch.int32), "kept_tables": full((B, P), torch.int32),
            "kept_mass": full((B, P), torch.float32), "kept_lens": full(B, torch.int32)}


def prepare(case, seed):
    g = _gen(seed)
    s = {"attend": _prepare_attend, "mass": _prepare_attend, "append": _prepare_append,
         "select": _prepare_select}[case["op"]](case, g)
    if own:  # the handle that a serving loop keeps: arguments checked and packed once, contents read at every call
        s["call"] = _own_call(s)
    return s


# ---- the framework's calls --------------------------------------------------------------------------------------
def _own_call(s):
    import sys

    if "vlx-tee_b200" not in sys.path:
        sys.path.insert(0, "vlx-tee_b200")
    from ztcp_b200 import kvcache

    if s["op"] == "attend":
        return kvcache.prepare_attend(s["q"], s["k"], s["v"], s["table"], s["kv_lens"], s["out"], lse=s["lse"],
                                      q_starts=s["starts"], max_q_len=s["q_max"], rope_dim=s["rope"], scale=s["scale"])
    if s["op"] == "mass":
        return kvcache.prepare_page_mass(s["q"], s["k"], s["table"], s["kv_lens"], s["lse"], s["mass"], s["out"],
                                         decay=s["decay"], q_starts=s["starts"], max_q_len=s["q_max"],
                                         scale=s["scale"])
    if s["op"] == "append":
        return kvcache.prepare_append(s["q"], s["k"], s["v"], s["k_pool"], s["v_pool"], s["slots"], s["positions"],
                                      s["rope_table"], s["q_out"], q_weight=s["q_weight"], k_weight=s["k_weight"],
                                      norm_from=s["norm_from"], eps=s["eps"], interleaved=s["interleaved"])
    return kvcache.prepare_select(s["mass"], s["table"], s["kv_lens"], s["cold_blocks"], s["cold_index"],
                                  s["cold_starts"], s["kept_tables"], s["kept_mass"], s["kept_lens"],
                                  page_tokens=s["page"], keep=s["keep"], sink=s["sink"], recent=s["recent"])


# ---- plain forms ------------------------------------------------------------------------------------------------
def _scores(s):
    """Scores [B, H, G, Q, L] of the padded batch (-inf where masked), log-sum-exp of the packed rows, row index."""
    q, k, table, lens, starts = s["q"], s["k"], s["table"], s["kv_lens"], s["starts"]
    (_, T, H, D), (B, P), Q = k.shape, table.shape, s["q_max"]
    keys = k[table.clamp_min(0).long()].reshape(B, P * T, H, D).float()
    q_len = starts[1:] - starts[:-1]
    i = torch.arange(Q, device=q.device)
    rows = (starts[:-1, None] + i).clamp_max(q.shape[0] - 1).long()
    there = i < q_len[:, None]
    qs = q[rows].float().reshape(B, Q, H, -1, D)
    x = torch.matmul(qs.permute(0, 2, 3, 1, 4).reshape(B, H, -1, D), keys.permute(0, 2, 3, 1)) * s["scale"]
    x = x.reshape(B, H, -1, Q, P * T)
    last = (lens - q_len)[:, None] + i
    seen = (torch.arange(P * T, device=q.device) <= last[..., None]) & there[..., None]
    x = x.masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True).clamp_min(-3e38)
    lse = (x - top).exp_().sum(-1).log_() + top[..., 0]
    return x, lse.permute(0, 3, 1, 2)[there].reshape(q.shape[0], -1), there


def _plain_attend(s):
    x, lse, there = _scores(s)
    B, H, G, Q, L = x.shape
    values = (s["k"][..., s["rope"]:] if s["v"] is None else s["v"])
    values = values[s["table"].clamp_min(0).long()].reshape(B, L, H, -1).float()
    x -= x.amax(-1, keepdim=True).clamp_min(-3e38)
    p = x.exp_()
    o = torch.matmul(p.reshape(B, H, G * Q, L), values.permute(0, 2, 1, 3)).reshape(B, H, G, Q, -1)
    o /= p.sum(-1, keepdim=True).clamp_min(1e-38)
    out = o.permute(0, 3, 1, 2, 4)[there].reshape(s["q"].shape[0], H * G, -1).to(s["q"].dtype)
    return {"out": out, "lse": lse}


def _plain_mass(s):
    q, k, table, lens, starts = s["q"], s["k"], s["table"], s["kv_lens"], s["starts"]
    x, _, there = _scores(s)
    B, H, G, Q, L = x.shape
    T, P = k.shape[1], table.shape[1]
    i = torch.arange(Q, device=q.device)
    rows = (starts[:-1, None] + i).clamp_max(q.shape[0] - 1).long()
    lse = s["lse"][rows].reshape(B, Q, H, G).permute(0, 2, 3, 1)
    weight = (x - lse[..., None]).exp_().reshape(B, H * G * Q, P, T)
    return {"mass": s["mass"] * s["decay"] * (torch.arange(P, device=q.device) * T < lens[:, None])
            + weight.sum(-1).sum(1)}


def _norm_rotate(x, weight, s):
    x, f, R = x.float(), s["norm_from"], s["rope"]
    if weight is not None:
        y = x[..., f:]
        y = y * (y.square().mean(-1, keepdim=True) + s["eps"]).rsqrt() * weight
        x = torch.cat([x[..., :f], y], dim=-1)
    at = s["rope_table"][s["positions"].long()][:, None]
    cos, sin = at[..., :R // 2], at[..., R // 2:]
    if s["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., R:]], dim=-1).to(s["q"].dtype)


def _plain_append(s):
    q = _norm_rotate(s["q"], s["q_weight"], s)
    s["k_pool"].flatten(0, 1)[s["slots"]] = _norm_rotate(s["k"], s["k_weight"], s)
    if s["v"] is not None:
        s["v_pool"].flatten(0, 1)[s["slots"]] = s["v"]
    return {"q": q, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_select(s):
    mass, table, lens, T = s["mass"], s["table"], s["kv_lens"], s["page"]
    B, P = table.shape
    page = torch.arange(P, device=mass.device)
    pages = (lens + T - 1) // T
    count = torch.minimum(pages - s["keep"], pages - s["sink"] - s["recent"]).clamp_min(0)
    free = (page >= s["sink"]) & (page < (pages - s["recent"])[:, None])
    order = torch.where(free, mass, float("inf")).sort(dim=1, stable=True).indices
    rank = torch.empty_like(order).scatter_(1, order, page.expand(B, P))
    cold = (rank < count[:, None]) & free
    kept = ~cold & (page < pages[:, None])
    starts = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
    flat = torch.arange(B * P, device=mass.device)
    first = torch.where(cold.flatten(), flat, B * P).sort().values  # the cold pages, in order, then B * P
    there = first < B * P
    index = torch.where(there, first, -1).to(torch.int32)
    blocks = torch.where(there, table.flatten()[first.clamp_max(B * P - 1)], -1).to(torch.int32)
    order = torch.where(kept, page, P).sort(dim=1).values
    there, order = order < P, order.clamp_max(P - 1)
    return {"cold_blocks": blocks, "cold_index": index, "cold_starts": starts,
            "kept_tables": torch.where(there, table.gather(1, order), -1),
            "kept_mass": torch.where(there, mass.gather(1, order), 0.0), "kept_lens": lens - (count * T).to(torch.int32)}


def run(s):
    if own:
        s["call"]()
        if s["op"] == "attend":
            return {"out": s["out"], "lse": s["lse"]}
        if s["op"] == "mass":
            return {"mass": s["out"]}
        if s["op"] == "append":
            return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
        return {n: s[n] for n in ("cold_blocks", "cold_index", "cold_starts", "kept_tables", "kept_mass", "kept_lens")}
    return {"attend": _plain_attend, "mass": _plain_mass, "append": _plain_append, "select": _plain_select}[s["op"]](s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------
def work(case):
    if case["op"] == "select":
        kv, _ = _lens(case)
        pages = [-(-n // case["page"]) for n in kv]
        P = max(pages)
        return {"bytes": sum(pages) * 8 + 16 * len(pages) * P + 12 * len(pages), "flops": 0}
    if case["op"] == "append":
        n, D = case["tokens"], case["dim"]
        vectors = case["heads"] + case["kv_heads"] * (1 if case["norm_from"] else 2)
        return {"bytes": n * (vectors * D * 2 * 2 + case["rope"] * 4 + 12), "flops": 6 * n * vectors * D}
    kv, q_len = _lens(case)
    D, H, heads = case["dim"], case["kv_heads"], case["heads"]
    dv = D - case["rope"]
    pairs = sum(b * a - b * (b - 1) // 2 for a, b in zip(kv, q_len)) * heads
    rows = sum(q_len) * heads
    if case["op"] == "mass":
        pages = [-(-n // case["page"]) for n in kv]
        return {"bytes": sum(kv) * H * D * 2 + rows * (D * 2 + 4) + 4 * sum(pages) + 8 * len(kv) * max(pages),
                "flops": 2 * D * pairs}
    once = D if case["rope"] else 2 * D
    return {"bytes": sum(kv) * H * once * 2 + rows * ((D + dv) * 2 + 4), "flops": 2 * (D + dv) * pairs}


# ---- the operators' definitions in 64 bits ----------------------------------------------------------------------
def _exact_attend(s):
    q, k, table = s["q"].double(), s["k"], s["table"]
    T, H, D = k.shape[1:]
    G = q.shape[1] // H
    kv, starts = s["kv_lens"].tolist(), s["starts"].tolist()
    dv = D - s["rope"]
    out = torch.zeros((q.shape[0], H * G, dv), dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    sums = torch.zeros(table.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(kv):
        at = torch.arange(n, device=q.device)
        slot = table[b].long()[at // T] * T + at % T
        a, e = starts[b], starts[b + 1]
        hidden = at[None, :] > (torch.arange(e - a, device=q.device) + n - (e - a))[:, None]
        for h in range(H):
            keys = k.view(-1, H, D)[slot, h].double()
            values = keys[:, s["rope"]:] if s["v"] is None else s["v"].view(-1, H, D)[slot, h].double()
            for j in range(h * G, h * G + G):
                x = (q[a:e, j] @ keys.T) * s["scale"]
                x[hidden] = float("-inf")
                if s["op"] == "attend":
                    lse[a:e, j] = torch.logsumexp(x, 1)
                    out[a:e, j] = torch.exp(x - lse[a:e, j, None]) @ values
                else:
                    w = torch.exp(x - s["lse"][a:e, j, None].double()).sum(0)
                    sums[b].index_add_(0, at // T, w)
    if s["op"] == "attend":
        return {"out": out, "lse": lse}
    for b, n in enumerate(kv):
        p = -(-n // T)
        sums[b, :p] += s["decay"] * s["mass"][b, :p].double()
    return {"mass": sums}


def _exact_append(s, case):
    D, R, f = case["dim"], case["rope"], s["norm_from"]
    pos = s["positions"].cpu().double()
    w = s["rope_table"].double().cpu()[s["positions"].cpu().long()]

    def turn(x, weight):
        x = x.cpu().double().clone()
        if weight is not None:
            r = 1.0 / torch.sqrt((x[..., f:] ** 2).sum(-1, keepdim=True) / (D - f) + s["eps"])
            x[..., f:] *= r * weight.cpu().double()
        y = x.clone()
        for i in range(R // 2):
            a, b = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + R // 2)
            c, d = w[:, None, i], w[:, None, R // 2 + i]
            y[..., a] = x[..., a] * c - x[..., b] * d
            y[..., b] = x[..., a] * d + x[..., b] * c
        return y

    assert pos.numel() == case["tokens"]
    slots = s["slots"].cpu()
    pools = []
    for pool, new in ((s["k_pool"], turn(s["k"], s["k_weight"])), (s["v_pool"], None if s["v"] is None else s["v"].cpu().double())):
        if pool is None:
            pools.append(None)
            continue
        flat = torch.zeros(pool.shape, dtype=torch.float64)
        flat.view(-1, *pool.shape[2:])[slots] = new
        pools.append(flat)
    return {"q": turn(s["q"], s["q_weight"]), "k_pool": pools[0], "v_pool": pools[1]}


def _exact_select(s):
    mass, table, lens = s["mass"].double().cpu().tolist(), s["table"].cpu().tolist(), s["kv_lens"].cpu().tolist()
    B, P = len(table), len(table[0])
    blocks, index, starts, tables, kept_mass, kept_lens = [], [], [0], [], [], []
    for b, n in enumerate(lens):
        pages = -(-n // s["page"])
        count = max(0, min(pages - s["keep"], pages - s["sink"] - s["recent"]))
        free = sorted(range(s["sink"], pages - s["recent"]), key=lambda p: (mass[b][p], p))
        cold = set(free[:count])
        for p in sorted(cold):
            blocks.append(table[b][p])
            index.append(b * P + p)
        starts.append(len(blocks))
        keep = [p for p in range(pages) if p not in cold]
        tables.append([table[b][p] for p in keep] + [-1] * (P - len(keep)))
        kept_mass.append([mass[b][p] for p in keep] + [0.0] * (P - len(keep)))
        kept_lens.append(n - count * s["page"])
    tail = [-1] * (B * P - len(blocks))
    whole = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return {"cold_blocks": whole(blocks + tail), "cold_index": whole(index + tail), "cold_starts": whole(starts),
            "kept_tables": whole(tables), "kept_mass": torch.tensor(kept_mass, dtype=torch.float64),
            "kept_lens": whole(kept_lens)}


def exact(case, seed):
    s = {"attend": _prepare_attend, "mass": _prepare_attend, "append": _prepare_append,
         "select": _prepare_select}[case["op"]](case, _gen(seed))
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "select":
        return _exact_select(s)
    return _exact_attend(s)
