"""Plain restatements of the operators on the paged K/V pool of 4 bits (``csrc/kv_fp4.cuh`` has the format)."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import ref
from .ref import E2M1_VALUES


def _order(dim: int):
    """How the bytes of a tile lie: for keys, values and their scales the shape as stored, the axes that make a token, and
    those that make its row."""
    w, c = (2, 1) if dim == 64 else (1, dim // 128)      # tokens in 16 bytes of a lane; 16-byte chunks of a token and lane
    u = 256 // dim
    return (((2 // w, c, 4, 2, 4, w, 16 // w), (2, 0, 5, 3), (4, 1, 6)),
            ((4 // u, 8, 4, u, dim // 16), (2, 0, 3), (1, 4)),
            ((4, 2, 4, 2, dim // 64), (0, 3, 1), (2, 4)),
            ((dim // 16, 4, 4), (1, 2), (0,)))


def unpack_tiles(cache: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``[..., 18 D]`` bytes -> codes of keys and of values ``[..., 16, D / 2]``, scales of both ``[..., 16, D / 16]``."""
    dim = cache.shape[-1] // 18
    lead, n = cache.shape[:-1], cache.dim() - 1
    return tuple(x.reshape(*lead, *shape).permute(*range(n), *(n + i for i in tok + row)).reshape(*lead, 16, x.shape[-1] // 16)
                 for x, (shape, tok, row) in zip(cache.split([8 * dim, 8 * dim, dim, dim], -1), _order(dim)))


def pack_tiles(*parts: torch.Tensor) -> torch.Tensor:
    """The inverse of ``unpack_tiles``."""
    lead, dim = parts[0].shape[:-2], 2 * parts[0].shape[-1]
    n = len(lead)
    flat = []
    for x, (shape, tok, row) in zip(parts, _order(dim)):
        places = tok + row
        back = sorted(range(len(places)), key=places.__getitem__)
        flat.append(x.reshape(*lead, *(shape[i] for i in places)).permute(*range(n), *(n + i for i in back)).reshape(*lead, 16 * x.shape[-1]))
    return torch.cat(flat, -1)


def quantise(x: torch.Tensor, head: Optional[torch.Tensor]) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows ``[T, heads, D]`` -> two codes a byte ``[T, heads, D / 2]`` and e4m3 scales ``[T, heads, D / 16]`` (bytes)."""
    x = x.float().unflatten(-1, (-1, 16))
    head = torch.ones(x.shape[1]) if head is None else head.float()
    head = head.to(x.device)[:, None, None]
    sf = (x.abs().amax(-1, keepdim=True) / (6.0 * head)).clamp(max=ref.FP8_MAX).to(torch.float8_e4m3fn)
    step = sf.float() * head
    y = torch.where(step > 0, x / step, torch.zeros_like(x))
    bounds = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=x.device)
    a = y.abs()[..., None]
    even = torch.arange(7, device=x.device) % 2 == 0        # a tie goes to the even code: down at the even bounds
    code = torch.where(even, a > bounds, a >= bounds).sum(-1).to(torch.uint8)
    code = (code + 8 * torch.signbit(y).to(torch.uint8)).flatten(-2)
    return code[..., 0::2] | code[..., 1::2] << 4, sf.view(torch.uint8)[..., 0]


def dequantise(codes: torch.Tensor, sf: torch.Tensor, head: Optional[torch.Tensor]) -> torch.Tensor:
    """The inverse: fp32 ``[..., heads, D]``."""
    table = torch.tensor(E2M1_VALUES, device=codes.device)
    x = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)
    x = (x.unflatten(-1, (-1, 16)) * sf.contiguous().view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)
    return x if head is None else x * head.float()[:, None]


def _place(loc: torch.Tensor, page: int):
    return loc // page, slice(None), loc % page // 16, loc % 16


def store_kv_fp4(k, v, cache, out_loc, k_scale=None, v_scale=None, weights=None) -> None:
    dim, page, hk = cache.shape[-1] // 18, cache.shape[-2] * 16, cache.shape[-3]
    loc = out_loc.long()
    inside = (loc >= 0) & (loc < cache.shape[0] * page)
    loc, k, v = loc[inside], k.reshape(-1, hk, dim)[inside], v.reshape(-1, hk, dim)[inside]
    pages, back = torch.unique(loc // page, return_inverse=True)
    parts = unpack_tiles(cache[pages])
    (kc, ks), (vc, vs) = quantise(k, k_scale), quantise(v, v_scale)
    where = (back, slice(None), loc % page // 16, loc % 16)
    for part, rows in zip(parts, (kc, vc, ks, vs)):
        part[where] = rows
    cache[pages] = pack_tiles(*parts)
    if weights is not None:
        weights[loc // page, :, loc % page] = 0.0


def load_kv_fp4(cache, slots, k_scale, v_scale, dtype):
    if cache.dim() == 5:
        both = [load_kv_fp4(c, slots, k_scale, v_scale, dtype) for c in cache]
        return tuple(torch.stack([x[w] for x in both]) for w in (0, 1))
    page = cache.shape[-2] * 16
    loc = slots.long()
    inside = (loc >= 0) & (loc < cache.shape[0] * page)
    loc = torch.where(inside, loc, 0)
    pages, back = torch.unique(loc // page, return_inverse=True)
    parts = unpack_tiles(cache[pages])
    kc, vc, ks, vs = (x[back, :, loc % page // 16, loc % 16] for x in parts)
    outside = ~inside[:, None, None]                # (slot 0 is read for them, which may hold a NaN)
    return tuple(dequantise(c, s, h).masked_fill(outside, 0.0).to(dtype) for c, s, h in ((kc, ks, k_scale), (vc, vs, v_scale)))


def paged_attention_fp4(q, cache, block_table, cu_q, seq_lens, scale, k_scale=None, v_scale=None, window=0, weights=None):
    t, hq, dim = q.shape
    hk, page = cache.shape[1], cache.shape[2] * 16
    group = hq // hk
    out = torch.zeros(q.shape, dtype=torch.float32, device=q.device)
    cu = cu_q.tolist()
    for b, n in enumerate(seq_lens.tolist()):
        q_len = cu[b + 1] - cu[b]
        n = min(n, block_table.shape[1] * page)
        if q_len <= 0 or n <= 0:
            continue
        i = torch.arange(n, device=q.device)
        pages = block_table[b].long().clamp(0, cache.shape[0] - 1)
        kc, vc, ks, vs = (x.permute(0, 2, 3, 1, 4).flatten(0, 2)[:n] for x in unpack_tiles(cache[pages]))
        kk, vv = dequantise(kc, ks, k_scale), dequantise(vc, vs, v_scale)            # [n, hk, D]
        qq = q[cu[b]:cu[b + 1]].float().view(q_len, hk, group, dim)
        s = torch.einsum("qhgd,nhd->hgqn", qq, kk) * scale
        pos = torch.arange(n - q_len, n, device=q.device)[:, None]
        hidden = i > pos
        if window > 0:
            hidden = hidden | (i <= pos - window)
        s = s.masked_fill(hidden, float("-inf"))
        p = torch.softmax(s, -1).masked_fill(hidden, 0.0)
        none = vv.isnan()
        o = torch.einsum("hgqn,nhd->qhgd", p, vv.masked_fill(none, 0.0))
        if none.any():                                        # a NaN reaches the rows that see it, no others
            o = o.masked_fill(torch.einsum("qn,nhd->qhd", (~hidden).float(), none.float())[:, :, None] > 0, float("nan"))
        out[cu[b]:cu[b + 1]] = o.reshape(q_len, hq, dim)
        if weights is not None:
            weights[pages[i // page], :, i % page] += p.sum((1, 2)).T
    return out.to(q.dtype)


def evict_kv_fp4(cache, weights, block_table, seq_lens, new_table, budget, recent, sinks):
    if cache.dim() == 5:
        both = [evict_kv_fp4(c, w, block_table, seq_lens, new_table, budget, recent, sinks) for c, w in zip(cache, weights)]
        return torch.stack([x[0] for x in both]), both[0][1]
    hk, page = cache.shape[1], cache.shape[2] * 16
    kept = torch.full((seq_lens.numel(), hk, budget), -1, dtype=torch.int32, device=cache.device)
    lens = seq_lens.clamp(0, block_table.shape[1] * page)
    for b, n in enumerate(lens.tolist()):
        m = min(n, budget)
        if m == 0:
            continue
        old, new = block_table[b].long().clamp(0, cache.shape[0] - 1), new_table[b, :-(-m // page)].long()
        i = torch.arange(n, device=cache.device)
        w = weights[old[i // page], :, i % page].T                                       # [hk, n]
        if n > budget:
            sure = ((i < sinks) | (i >= n - recent)).expand_as(w)
            order = torch.sort(w, dim=-1, descending=True, stable=True).indices           # a NaN first
            order = order.gather(1, torch.sort(sure.gather(1, order).int(), dim=-1, descending=True, stable=True).indices)
            stay = order[:, :budget].sort(-1).values
        else:
            stay = i.expand(hk, n)
        kept[b, :, :m] = stay.int()
        parts = [x.transpose(0, 1).flatten(1, 3) for x in unpack_tiles(cache[old])]     # [hk, tokens, bytes]
        fresh = [x.transpose(0, 1).flatten(1, 3) for x in unpack_tiles(cache[new.clamp(0, cache.shape[0] - 1)])]
        for x, y in zip(parts, fresh):
            y[:, :m] = x.gather(1, stay[..., None].expand(*stay.shape, x.shape[-1]))
        there = (new >= 0) & (new < cache.shape[0])                                      # what would go to any other page is dropped
        cache[new[there]] = pack_tiles(*(y.unflatten(1, (-1, page // 16, 16)).transpose(0, 1) for y in fresh))[there]
        j = torch.arange(m, device=cache.device)
        j = j[there[j // page]]
        weights[new[j // page], :, j % page] = w.gather(1, stay).T[j]
    return kept, torch.clamp(lens, max=budget).int()
