"""Operators on the paged K/V pool of 4 bits, as cases to be timed: rows are stored and loaded again, attention reads them
(decode steps, prompts behind a prefix, a few rows that look back), and rows with little attention weight are evicted.

A value of the pool is ``code * scale * head``: ``code`` one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign (4 bits), ``scale`` an
e4m3 number for 16 neighbouring channels, ``head`` an fp32 factor per key / value head. ``scale`` is the block's largest
magnitude over ``6 head``; rounding is to nearest, ties to the even code. The pool is ``[layers,] pages, heads, page / 16,
18 D`` bytes: 16 tokens of one head as the codes of their keys (8 D bytes), of their values (8 D), the scales of the keys (D)
and of the values (D), each in the order in which the lanes of a warp take them (``token_major`` undoes it). Beside it lies
an fp32 attention weight per token and head.

``own`` chooses between the package's kernels and the plain form.
"""
import math

import torch

own = False

DEVICE = "cuda"
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------ cases
def _attend(name, heads, kv_heads, dim, requests, cached, new, page=16, window=0, tracked=False, dtype="bf16"):
    """``cached``: tokens of a request before the step, from .. to; ``new``: rows of a request in the step, from .. to."""
    return dict(name=name, op="attend", heads=heads, kv_heads=kv_heads, dim=dim, requests=requests, cached_min=cached[0],
                cached_max=cached[1], new_min=new[0], new_max=new[1], page=page, window=window, tracked=tracked, dtype=dtype)


def _store(name, kv_heads, dim, rows, page=16, dtype="bf16"):
    return dict(name=name, op="store", kv_heads=kv_heads, dim=dim, rows=rows, page=page, dtype=dtype)


def _evict(name, kv_heads, dim, layers, requests, cached, budget, recent, sinks, page=16):
    return dict(name=name, op="evict", kv_heads=kv_heads, dim=dim, layers=layers, requests=requests, cached_min=cached[0],
                cached_max=cached[1], budget=budget, recent=recent, sinks=sinks, page=page, dtype="bf16")


def listed():
    return [
        # a chat with one user: every microsecond of the call is waited for
        _attend("one request", 32, 8, 128, 1, (700, 700), (1, 1)),
        # a server's running batch, lengths as they come (the benchmark's requests lie in this range)
        _attend("running batch", 32, 8, 128, 64, (511, 2303), (1, 1)),
        # few requests over long documents
        _attend("long documents", 64, 8, 128, 4, (70001, 120000), (1, 1)),
        # a batch whose attention weights are kept for eviction
        _attend("weighed batch", 32, 8, 128, 48, (900, 5000), (1, 1), tracked=True),
        # narrow heads in fp16, a window, larger pages
        _attend("windowed narrow heads", 24, 8, 64, 40, (1, 6000), (1, 1), page=64, window=1024, dtype="fp16"),
        # a prompt's last rows look back over it: the weights by which its rows are first evicted
        _attend("looking back", 32, 8, 128, 3, (5000, 9000), (17, 32), tracked=True),
        # the chunks of two prompts behind cached prefixes
        _attend("prompts behind prefixes", 32, 8, 128, 2, (3000, 6500), (1700, 2300)),
        # a decode step's new rows
        _store("store rows of a step", 8, 128, 64),
        # a prompt chunk's new rows
        _store("store a prompt chunk", 8, 128, 8192),
        # one long conversation is cut down, in the layers of a slice of the model
        _evict("evict one request", 8, 128, 4, 1, (9000, 9000), 2048, 512, 4),
        # a batch of long ones is cut down
        _evict("evict a batch", 8, 128, 4, 12, (12000, 40000), 2048, 256, 4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    dim = rng.choice([64, 128, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8])
    kind = rng.choice(["decode", "decode", "decode", "rows", "prompt", "store", "evict"])
    if kind == "store":
        c = _store("", kv_heads, dim, _log(rng, 1, 8192), page, dtype)
    elif kind == "evict":
        budget = _log(rng, 64, 2048)
        sinks = rng.choice([0, 1, 4])
        lo = _log(rng, 50, 30000)
        hi = min(40000, lo + _log(rng, 1, 10000))
        layers = rng.randint(1, 4)
        requests = max(1, min(_log(rng, 1, 12), 12 * 4 * 40000 // (layers * hi)))
        c = _evict("", kv_heads if dim < 256 else min(kv_heads, 4), dim, layers, requests, (lo, hi), budget,
                   rng.randint(1, max(1, budget // 2)), sinks, page)
    else:
        heads = kv_heads * rng.choice([1, 2, 4, 4, 5, 7, 8, 16])
        tracked = rng.random() < 0.3
        window = _log(rng, 100, 5000) if rng.random() < 0.2 else 0
        if kind == "prompt":
            heads, window = min(heads, max(1, 4096 // dim // kv_heads) * kv_heads), 0
            new = _log(rng, 200, 2000)
            c = _attend("", heads, kv_heads, dim, rng.randint(1, 2), (_log(rng, 1, 3000), 4000), (new, new + new // 8), page, 0,
                        False, dtype)
        elif kind == "rows":
            new = rng.randint(2, 24)
            lo = _log(rng, 1, 4000)
            c = _attend("", min(heads, 32 // kv_heads * kv_heads), kv_heads, dim, rng.randint(1, 6), (lo, 2 * lo + 10),
                        (1, new), page, window, tracked, dtype)
        else:
            requests = _log(rng, 1, 256)
            most = max(64, min(100000, 600000 // (requests * max(1, dim // 64))))
            lo = _log(rng, 1, most)
            c = _attend("", heads, kv_heads, dim, requests, (lo, min(most, 3 * lo) if lo < most else lo), (1, 1), page, window,
                        tracked, dtype)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------------ the pool's layout
def token_major(tiles, dim):
    """``[..., 18 D]`` bytes of 16 tokens -> codes of the keys ``[..., 16, D / 2]`` (two channels a byte, the lower one in the
    low bits), of the values, scales of the keys ``[..., 16, D / 16]``, of the values."""
    lead = tiles.shape[:-1]
    n = len(lead)
    k, v, ks, vs = tiles.split([8 * dim, 8 * dim, dim, dim], -1)

    def order(x, shape, places, last):
        return x.reshape(*lead, *shape).permute(*range(n), *[n + p for p in places]).reshape(*lead, 16, last)

    w, c = (2, 1) if dim == 64 else (1, dim // 128)
    k = order(k, (2 // w, c, 4, 2, 4, w, 16 // w), (2, 0, 5, 3, 4, 1, 6), dim // 2)
    w = 256 // dim
    v = order(v, (4 // w, 8, 4, w, dim // 16), (2, 0, 3, 1, 4), dim // 2)
    ks = order(ks, (4, 2, 4, 2, dim // 64), (0, 3, 1, 2, 4), dim // 16)
    vs = order(vs, (dim // 16, 4, 4), (1, 2, 0), dim // 16)
    return k, v, ks, vs


def lane_major(k, v, ks, vs):
    """The inverse of ``token_major``."""
    lead = k.shape[:-2]
    n = len(lead)
    dim = 2 * k.shape[-1]

    def order(x, shape, places):
        return x.reshape(*lead, *shape).permute(*range(n), *[n + p for p in places]).reshape(*lead, -1)

    w, c = (2, 1) if dim == 64 else (1, dim // 128)
    k = order(k, (4, 2 // w, w, 2, 4, c, 16 // w), (1, 5, 0, 3, 4, 2, 6))
    w = 256 // dim
    v = order(v, (4, 4 // w, w, 8, dim // 16), (1, 3, 0, 2, 4))
    ks = order(ks, (4, 2, 2, 4, dim // 64), (0, 2, 3, 1, 4))
    vs = order(vs, (4, 4, dim // 16), (2, 0, 1))
    return torch.cat([k, v, ks, vs], -1)


def quantise(x, head):
    """Rows ``[..., heads, D]`` -> codes (two a byte) and scales (bytes of e4m3)."""
    x = x.float().unflatten(-1, (-1, 16))
    head = head[:, None, None]
    scale = (x.abs().amax(-1, keepdim=True) / (6.0 * head)).clamp(max=448.0).to(torch.float8_e4m3fn)
    step = scale.float() * head
    y = torch.where(step > 0, x / torch.where(step > 0, step, 1.0), 0.0)
    a = y.abs()
    code = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    code = (code + (y < 0).to(torch.uint8) * 8).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], scale.view(torch.uint8)[..., 0]


def values(codes, scales, head):
    """The inverse: ``[..., tokens, D]`` in fp32; ``head`` broadcasts to it."""
    table = torch.tensor(CODES + tuple(-c for c in CODES), device=codes.device)
    x = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).flatten(-2)
    return (x.unflatten(-1, (-1, 16)) * scales.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2) * head


# ------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _rows(n, heads, dim, dtype, g):
    """Keys as a normed and rotated projection leaves them (a few strong channels), and values, smaller."""
    k = torch.randn((n, heads, dim), generator=g, device=DEVICE)
    k[..., 3::29] *= 4.0
    v = torch.randn((n, heads, dim), generator=g, device=DEVICE) * 0.25
    return k.to(dtype), v.to(dtype)


def _filled(pages, heads, page, dim, k_head, v_head, g):
    """A layer's pool with random rows in all pages."""
    parts = []
    for at in range(0, pages, 4096):
        n = min(4096, pages - at)
        k, v = _rows(n * page, heads, dim, torch.float32, g)
        kc, ks = quantise(k, k_head)
        vc, vs = quantise(v, v_head)
        parts.append(lane_major(*(x.view(n, page // 16, 16, heads, -1).permute(0, 3, 1, 2, 4) for x in (kc, vc, ks, vs))))
    return torch.cat(parts)


def _heads(n, g):
    """The factors of the heads' keys and values as a calibration over some text gives them."""
    return (0.03 + 0.02 * torch.rand(n, generator=g, device=DEVICE), 0.005 + 0.002 * torch.rand(n, generator=g, device=DEVICE))


def _lengths(lo, hi, n, start):
    """Lengths spread over lo .. hi, in no order. They go by the case alone: outputs of one case have one shape."""
    return torch.tensor([lo + int((hi - lo + 1) * ((start + i * 0.6180339887498949) % 1.0)) for i in range(n)])


def _cached(case):
    return _lengths(case["cached_min"], case["cached_max"], case["requests"], 0.37)


def _new(case):
    return _lengths(case["new_min"], case["new_max"], case["requests"], 0.71)


def prepare(case, seed):
    g = _generator(seed)
    heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    dtype = DTYPES[case["dtype"]]
    k_head, v_head = _heads(heads, g)
    s = dict(case=case, k_head=k_head, v_head=v_head)
    if case["op"] == "store":
        rows = case["rows"]
        pages = rows // page + 40
        s["k"], s["v"] = _rows(rows, heads, dim, dtype, g)
        s["cache"] = _filled(pages, heads, page, dim, k_head, v_head, g)
        # rows of a prompt lie page by page; pages come in any order
        order = torch.randperm(pages, generator=g, device=DEVICE)
        s["out_loc"] = (order[:, None] * page + torch.arange(page, device=DEVICE)).flatten()[5:5 + rows].int()
        return s
    requests = case["requests"]
    cached = _cached(case)
    if case["op"] == "attend":
        new = _new(case)
        lens = cached + new
        used = -(-lens // page)
        pages = int(used.sum()) + 3
        order = torch.randperm(pages - 1, generator=g, device=DEVICE).int()
        width = int(used.max())
        first = torch.cumsum(used, 0) - used
        at = first[:, None] + torch.arange(width)
        s["block_table"] = order[torch.where(torch.arange(width) < used[:, None], at, 0).to(DEVICE)]
        s["cache"] = _filled(pages, heads, page, dim, k_head, v_head, g)
        s["q"] = torch.randn((int(new.sum()), case["heads"], dim), generator=g, device=DEVICE).to(dtype)
        s["host"] = (torch.cat([torch.zeros(1, dtype=torch.long), torch.cumsum(new, 0)]).int().numpy(), lens.int().numpy())
        s["cu_q"], s["seq_lens"] = (torch.from_numpy(x).to(DEVICE) for x in s["host"])
        s["max_q"], s["max_kv"] = int(new.max()), int(lens.max())
        s["scale"] = 1.0 / math.sqrt(dim)
        s["weights"] = torch.rand((pages, heads, page), generator=g, device=DEVICE) if case["tracked"] else None
        return s
    used = -(-cached // page)
    width, slim = int(used.max()), -(-case["budget"] // page)
    pages = int(used.sum()) + requests * slim + 3
    order = torch.randperm(pages - 1, generator=g, device=DEVICE).int()
    first = torch.cumsum(used, 0) - used
    at = first[:, None] + torch.arange(width)
    s["block_table"] = order[torch.where(torch.arange(width) < used[:, None], at, 0).to(DEVICE)]
    s["new_table"] = order[int(used.sum()):int(used.sum()) + requests * slim].view(requests, slim).contiguous()
    s["cache"] = torch.stack([_filled(pages, heads, page, dim, k_head, v_head, g) for _ in range(case["layers"])])
    # a few tokens draw most of the attention, the later ones have been looked at less often; equal weights occur
    w = torch.rand((case["layers"], pages, heads, page), generator=g, device=DEVICE)
    s["weights"] = torch.round(w ** 6 * 4096) / 64
    s["seq_lens"] = cached.int().to(DEVICE)
    s["max_kv"] = int(cached.max())
    kept = torch.minimum(cached, torch.tensor(case["budget"]))
    # where the rows that stay will lie
    slots = (s["new_table"].cpu().long()[:, :, None] * page + torch.arange(page)).flatten(1)
    s["slots"] = torch.cat([slots[b, :int(kept[b])] for b in range(requests)]).int().to(DEVICE)
    return s


# ------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return _run_own(s)
    return {"attend": _attend_plain, "store": _store_plain, "evict": _evict_plain}[op](s)


def _run_own(s):
    from minisglang_rdna4_b200 import ops

    op, k_head, v_head = s["case"]["op"], s["k_head"], s["v_head"]
    if op == "store":
        ops.store_kv_fp4(s["k"], s["v"], s["cache"], s["out_loc"], k_head, v_head)
        return ops.load_kv_fp4(s["cache"], s["out_loc"], k_head, v_head, s["k"].dtype)
    if op == "evict":
        c = s["case"]
        kept, lens = ops.evict_kv_fp4(s["cache"], s["weights"], s["block_table"], s["seq_lens"], s["new_table"], c["budget"],
                                      c["recent"], c["sinks"], max_kv=s["max_kv"])
        return kept, lens, s["weights"], *ops.load_kv_fp4(s["cache"], s["slots"], k_head, v_head, DTYPES[c["dtype"]])
    plan = None
    if s["max_q"] > 1 and s["weights"] is None:
        plan = ops.prefill_plan_fp4(s["q"], s["cache"], *s["host"], window=s["case"]["window"])
    out = ops.paged_attention_fp4(s["q"], s["cache"], s["block_table"], s["cu_q"], s["seq_lens"], s["scale"], k_scale=k_head,
                                  v_scale=v_head, window=s["case"]["window"], max_q=s["max_q"], max_kv=s["max_kv"],
                                  weights=s["weights"], plan=plan)
    return out if s["weights"] is None else (out, s["weights"])


def _gathered(s, cache, table):
    """Keys and values ``[requests, heads, tokens, D]`` of the pages in ``table``."""
    dim = s["case"]["dim"]
    k, v, ks, vs = (x.transpose(1, 2).flatten(2, 4) for x in token_major(cache[table.long()], dim))
    return values(k, ks, s["k_head"][:, None, None]), values(v, vs, s["v_head"][:, None, None])


def _attend_plain(s):
    c, q, lens = s["case"], s["q"], s["seq_lens"].long()
    k, v = _gathered(s, s["cache"], s["block_table"])
    requests, kv_heads, tokens, dim = k.shape
    group = c["heads"] // kv_heads
    cu = s["cu_q"].long()
    row = torch.arange(s["max_q"], device=DEVICE)
    real = row < (cu[1:] - cu[:-1])[:, None]                                    # [requests, rows]
    at = torch.where(real, cu[:-1, None] + row, 0)
    x = q[at].float().view(requests, -1, kv_heads, group, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    pos = (lens - (cu[1:] - cu[:-1]))[:, None] + row
    key = torch.arange(tokens, device=DEVICE)
    seen = real[:, :, None] & (key <= pos[:, :, None])
    if c["window"]:
        seen &= key > pos[:, :, None] - c["window"]
    seen = seen[:, None, None].expand(-1, 1, group, -1, -1).flatten(2, 3)       # [requests, 1, group * rows, tokens]
    score = (x @ k.transpose(-1, -2) * s["scale"]).masked_fill_(~seen, -torch.inf)
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = score.sub_(top).exp_()
    p /= p.sum(-1, keepdim=True).clamp(min=1e-30)
    out = (p @ v).view(requests, kv_heads, group, -1, dim).permute(0, 3, 1, 2, 4).flatten(2, 3)
    out = out[real].to(q.dtype)
    if s["weights"] is None:
        return out
    page = c["page"]
    here = key < lens[:, None]
    where = (s["block_table"].long()[:, key // page] * page + key % page)[here]
    flat = s["weights"].transpose(0, 1).flatten(1).clone()                      # [heads, slots]
    flat.index_add_(1, where, p.sum(2).transpose(0, 1)[:, here])
    s["weights"].copy_(flat.view(kv_heads, -1, page).transpose(0, 1))
    return out, s["weights"]


def _put(cache, loc, k, v, ks, vs, page, dim):
    """Writes token rows ``[rows, heads, ...]`` at the slots ``loc`` of one layer."""
    where = (loc // page, slice(None), loc % page // 16, loc % 16)
    rows = token_major(cache, dim)
    for x, y in zip(rows, (k, v, ks, vs)):
        x[where] = y
    cache.copy_(lane_major(*rows))


def _take(cache, loc, s, page, dim):
    where = (loc // page, slice(None), loc % page // 16, loc % 16)
    k, v, ks, vs = (x[where] for x in token_major(cache, dim))
    return values(k, ks, s["k_head"][:, None]), values(v, vs, s["v_head"][:, None])


def _store_plain(s):
    page, dim, loc = s["case"]["page"], s["case"]["dim"], s["out_loc"].long()
    kc, ks = quantise(s["k"], s["k_head"])
    vc, vs = quantise(s["v"], s["v_head"])
    _put(s["cache"], loc, kc, vc, ks, vs, page, dim)
    k, v = _take(s["cache"], loc, s, page, dim)
    return k.to(s["k"].dtype), v.to(s["v"].dtype)


def _chosen(w, n, budget, recent, sinks):
    """Which tokens stay: ``w [..., requests, heads, tokens]``, ``n [requests]`` -> ``[..., budget]`` ascending, -1 behind."""
    i = torch.arange(w.shape[-1], device=w.device)
    n = n[:, None, None]
    sure = (i < n) & ((i < sinks) | (i >= n - recent))
    w = w.masked_fill(sure, torch.inf).masked_fill(i >= n, -1.0)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :budget]
    if order.shape[-1] < budget:
        order = torch.nn.functional.pad(order, (0, budget - order.shape[-1]), value=w.shape[-1])
    order = torch.where(order < n, order, 1 << 40).sort(-1).values
    return torch.where(order < n, order, -1)


def _evict_plain(s):
    c = s["case"]
    page, dim, budget = c["page"], c["dim"], c["budget"]
    table, n = s["block_table"].long(), s["seq_lens"].long()
    layers, requests = c["layers"], c["requests"]
    w = s["weights"][:, table].transpose(2, 3).flatten(3)                         # [layers, requests, heads, tokens]
    kept = _chosen(w, n, budget, c["recent"], c["sinks"])
    at = kept.clamp(min=0)
    there = kept >= 0
    old = [x.transpose(2, 3).flatten(3, 5) for x in token_major(s["cache"][:, table], dim)]
    slim = s["new_table"].shape[1] * page - budget
    new = s["new_table"].long()
    rows = [torch.gather(x, 3, at[..., None].expand(*at.shape, x.shape[-1])) for x in old]
    fresh = []
    for x, now in zip(rows, token_major(s["cache"][:, new], dim)):                # what no row comes to stays
        now = now.transpose(2, 3).flatten(3, 5)
        x = torch.cat([torch.where(there[..., None], x, now[..., :budget, :]), now[..., budget:, :]], 3)
        fresh.append(x.unflatten(3, (-1, page // 16, 16)).transpose(2, 3))
    s["cache"][:, new] = lane_major(*fresh)
    now = s["weights"][:, new].transpose(2, 3).flatten(3)
    moved = torch.cat([torch.where(there, torch.gather(w, 3, at), now[..., :budget]), now[..., budget:]], 3)
    s["weights"][:, new] = moved.unflatten(3, (-1, page)).transpose(2, 3)
    loc = s["slots"].long()
    where = (slice(None), loc // page, slice(None), loc % page // 16, loc % 16)
    k, v, ks, vs = (x[where].transpose(0, 1) for x in token_major(s["cache"], dim))
    k, v = (values(a, b, h[:, None]).to(DTYPES[c["dtype"]])
            for a, b, h in ((k, ks, s["k_head"]), (v, vs, s["v_head"])))
    return kept.int(), torch.minimum(n, torch.tensor(budget, device=DEVICE)).int(), s["weights"], k, v


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    heads, dim = case["kv_heads"], case["dim"]
    row = heads * dim * 9 // 8                  # bytes of a token's key and value in the pool
    if case["op"] == "store":
        n = case["rows"]
        return {"bytes": n * (2 * row + 8 * heads * dim + 8), "flops": n * heads * dim * 8}
    cached = _cached(case)
    if case["op"] == "evict":
        # of a request's tokens: every weight is read; of those that stay the row and the weight are moved, the row is loaded
        kept = int(torch.minimum(cached, torch.tensor(case["budget"])).sum())
        tokens = int(cached.sum())
        moved = tokens * heads * 4 + kept * (3 * row + heads * (4 + 4 + 4) + 4 * heads * dim)
        return {"bytes": case["layers"] * moved, "flops": case["layers"] * tokens * heads}
    new = _new(case)
    window = case["window"] or 1 << 30
    seen = int(torch.minimum(cached + new, window + new - 1).sum())
    pairs = sum(int(torch.arange(c + 1, c + n + 1).clamp(max=window).sum()) for c, n in zip(cached.tolist(), new.tolist()))
    moved = seen * (row + (8 * heads if case["tracked"] else 0)) + 4 * int(new.sum()) * case["heads"] * dim
    return {"bytes": moved, "flops": pairs * case["heads"] * dim * 4}


# ------------------------------------------------------------------------------------------ the definition, in 64 bits
_E4M3 = [m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127]


def _nearest(x, grid):
    """Index of the grid value (ascending, from 0) next to x >= 0; of two that are as near, the even index."""
    grid = torch.tensor(grid, dtype=torch.float64, device=x.device)
    hi = torch.searchsorted(grid, x).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    a, b = x - grid[lo], grid[hi] - x
    return torch.where((a < b) | ((a == b) & (lo % 2 == 0)), lo, hi)


def _rounded(x, head):
    """Rows as the pool holds them."""
    x = x.double().unflatten(-1, (-1, 16))
    head = head.double()[:, None, None]
    scale = torch.tensor(_E4M3, dtype=torch.float64, device=x.device)[_nearest(x.abs().amax(-1, keepdim=True) / (6 * head), _E4M3)]
    step = scale * head
    code = _nearest(torch.where(step > 0, x.abs() / torch.where(step > 0, step, 1.0), 0.0), CODES)
    return (torch.tensor(CODES, dtype=torch.float64, device=x.device)[code] * x.sign() * step).flatten(-2)


def _token(tile, t, dim):
    """Key and value of token ``t`` of tiles ``[..., 18 D]`` without their heads' factors, byte by byte from the lanes that
    hold them."""
    table = torch.tensor(CODES + tuple(-c for c in CODES), dtype=torch.float64, device=tile.device)
    sf = torch.tensor(_E4M3 + [math.nan] + [-x for x in _E4M3] + [math.nan], dtype=torch.float64, device=tile.device)
    d = torch.arange(dim, device=tile.device)
    r, g = (t >> 1) & 1, 2 * (t >> 2) + (t & 1)             # the key's row of the lane and the lane's group of four
    j, i = d // (dim // 4), d % (dim // 4)
    at = r * (dim // 8) + i // 2                              # of the lane's D / 4 bytes
    k = tile[..., at // 16 * 512 + (4 * g + j) * 16 + at % 16].long() >> (i % 2 * 4) & 15
    ks = tile[..., 16 * dim + (4 * g + j) * (dim // 32) + r * (dim // 64) + i // 16].long()
    g, i, j, e = d // (dim // 8), d % (dim // 8), t >> 2, t & 3
    at = e * (dim // 16) + i // 2
    v = tile[..., 8 * dim + at // 16 * 512 + (4 * g + j) * 16 + at % 16].long() >> (i % 2 * 4) & 15
    vs = tile[..., 17 * dim + (d // 16 * 4 + j) * 4 + e].long()
    return table[k] * sf[ks], table[v] * sf[vs]


def _request(cache, pages, dim, k_head, v_head, n):
    """Keys and values ``[heads, n, D]`` of one request."""
    tiles = cache[pages.long()].transpose(0, 1).flatten(1, 2)                     # [heads, tiles, 18 D]
    both = [_token(tiles, t, dim) for t in range(16)]
    k, v = (torch.stack([x[w] for x in both], 2).flatten(1, 2)[:, :n] for w in (0, 1))
    return k * k_head.double()[:, None, None], v * v_head.double()[:, None, None]


def exact(case, seed):
    s = prepare(case, seed)
    dim, page = case["dim"], case["page"]
    if case["op"] == "store":
        return _rounded(s["k"], s["k_head"]), _rounded(s["v"], s["v_head"])
    lens = s["seq_lens"].tolist()
    if case["op"] == "attend":
        cu, group = s["cu_q"].tolist(), case["heads"] // case["kv_heads"]
        w = None if s["weights"] is None else s["weights"].double()
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
        for b, n in enumerate(lens):
            pages = s["block_table"][b, :-(-n // page)]
            k, v = _request(s["cache"], pages, dim, s["k_head"], s["v_head"], n)
            i = torch.arange(n, device=DEVICE)
            summed = torch.zeros((case["kv_heads"], n), dtype=torch.float64, device=DEVICE)
            for at in range(cu[b], cu[b + 1], 256):
                end = min(at + 256, cu[b + 1])
                p = n - cu[b + 1] + torch.arange(at, end, device=DEVICE)[:, None]
                hidden = i > p
                if case["window"]:
                    hidden |= i <= p - case["window"]
                for h in range(case["heads"]):
                    score = (s["q"][at:end, h].double() @ k[h // group].T) / math.sqrt(dim)
                    prob = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                    out[at:end, h] = prob @ v[h // group]
                    summed[h // group] += prob.sum(0)
            if w is not None:
                for h in range(case["kv_heads"]):
                    w[pages.long()[i // page], h, i % page] += summed[h]
        return out if w is None else (out, w)
    w = s["weights"].double()
    keys, vals = [], []
    for layer in range(case["layers"]):
        rows = []
        for b, n in enumerate(lens):
            pages = s["block_table"][b, :-(-n // page)].long()
            i = torch.arange(n, device=DEVICE)
            m = min(n, case["budget"])
            k, v = _request(s["cache"][layer], pages, dim, s["k_head"], s["v_head"], n)
            new = s["new_table"][b].long()
            j = torch.arange(m, device=DEVICE)
            stay = []
            for h in range(case["kv_heads"]):
                mine = s["weights"][layer][pages[i // page], h, i % page]
                if n > case["budget"]:
                    rank = mine.double()
                    rank[:case["sinks"]] = math.inf
                    rank[n - case["recent"]:] = math.inf
                    # by weight, then by place
                    at = torch.sort(torch.argsort(-rank, stable=True)[:m]).values
                else:
                    at = i
                w[layer][new[j // page], h, j % page] = mine[at].double()
                stay.append(at)
            rows.append((torch.stack([k[h, a] for h, a in enumerate(stay)], 1), torch.stack([v[h, a] for h, a in enumerate(stay)], 1)))
        keys.append(torch.cat([r[0] for r in rows]))
        vals.append(torch.cat([r[1] for r in rows]))
    return None, None, w, torch.stack(keys), torch.stack(vals)
