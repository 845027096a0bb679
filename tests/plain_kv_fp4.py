"""The paged K/V pool of 4 bits in 64 bits and plain loops, from the format's definition alone: bytes of a tile by token and
channel, quantisation by distance to the table's values, attention request by request."""
import math

import torch

CODES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127]


def places(dim):
    """Byte of the tile and low / high half of it for every token and channel, of keys and of values; bytes of the scales."""
    k, v, half = (torch.zeros(16, dim, dtype=torch.long) for _ in range(3))
    ks, vs = (torch.zeros(16, dim // 16, dtype=torch.long) for _ in range(2))
    for lane in range(32):
        g, j = lane // 4, lane % 4
        for r in range(2):
            t = 4 * (g // 2) + 2 * r + g % 2
            for i in range(dim // 4):
                at = r * dim // 8 + i // 2
                k[t, j * dim // 4 + i] = at // 16 * 512 + lane * 16 + at % 16
                half[:, j * dim // 4 + i] = i % 2
            for i in range(dim // 64):
                ks[t, j * dim // 64 + i] = 16 * dim + lane * dim // 32 + r * dim // 64 + i
        for e in range(4):
            for i in range(dim // 8):
                at = e * dim // 16 + i // 2
                v[4 * j + e, g * dim // 8 + i] = 8 * dim + at // 16 * 512 + lane * 16 + at % 16
    for b in range(dim // 16):
        for t in range(16):
            vs[t, b] = 17 * dim + b * 16 + t
    return k, v, half, ks, vs


def values(cache, k_head=None, v_head=None):
    """All keys and values ``[pages, heads, page, D]`` in 64 bits, on the CPU."""
    cache = cache.cpu()
    dim = cache.shape[-1] // 18
    k, v, half, ks, vs = places(dim)
    code = torch.tensor(CODES + [-c for c in CODES], dtype=torch.float64)
    sf = torch.tensor(E4M3 + [math.nan] + [-c for c in E4M3] + [math.nan], dtype=torch.float64)
    out = []
    for at, scale, head in ((k, ks, k_head), (v, vs, v_head)):
        x = code[(cache[..., at] >> (4 * half).to(torch.uint8) & 15).long()] * sf[cache[..., scale].long()].repeat_interleave(16, -1)
        x = x.flatten(2, 3)
        out.append(x if head is None else x * head.cpu().double()[:, None, None])
    return out


def nearest(x, grid):
    """Nearest value of the grid to each x >= 0, of two the one with the even index."""
    grid = torch.tensor(grid, dtype=torch.float64)
    far = (x[..., None] - grid).abs()
    best = far.amin(-1, keepdim=True)
    index = torch.arange(len(grid))
    cost = torch.where(far == best, index % 2, 2)
    return grid[cost.argmin(-1)]


def rounded(x, head):
    """Rows ``[T, heads, D]`` as the pool holds them, in 64 bits."""
    x = x.cpu().double().unflatten(-1, (-1, 16))
    head = torch.ones(x.shape[1], dtype=torch.float64) if head is None else head.cpu().double()
    head = head[:, None, None]
    step = nearest((x.abs().amax(-1, keepdim=True) / (6 * head)).clamp(max=448.0), E4M3) * head
    y = torch.where(step > 0, (x.abs() / step).clamp(max=6.0), 0.0)
    return (nearest(y, CODES) * x.sign() * step).flatten(-2)


def attention(q, k, v, table, cu_q, lens, scale, window=0):
    """``(out, tolerance of out for one rounding of the probabilities to 11 bits and of out to q's type, weights of each token
    [request: [heads, tokens]], their tolerance)``. The tolerances follow the arithmetic: products of 4-bit keys and 16-bit
    queries are exact, D of them are summed in 32 bits (each addition off by at most 2^-23 of the sum of magnitudes), a score
    that is off by d changes its weight by a share of 2 d, the exponential and the sums of weights add 2^-19. Probabilities are
    held in f16 after a factor of 2^7: those below 2^-14 / 2^7 of the largest are subnormal, in steps of 2^-24, so off by up to
    2^-25 / 2^7 = 2^-32 of a sum of weights that is at least 1 (the largest is): 2^-32 times the magnitudes in sight."""
    t, hq, dim = q.shape
    hk, page = k.shape[1], k.shape[2]
    q = q.cpu()
    half_step = torch.finfo(q.dtype).eps / 2
    q = q.double()
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    weights, weights_tol = [], []
    cu = cu_q.tolist()
    for b, n in enumerate(lens.tolist()):
        n = max(0, min(n, table.shape[1] * page))
        pages = table[b].long().cpu()
        kk, vv = (x[pages].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(hq // hk, 0) for x in (k, v))
        qq = q[cu[b]:cu[b + 1]].transpose(0, 1)
        m = qq.shape[1]
        i, p = torch.arange(n), n - m + torch.arange(m)[:, None]
        hidden = i > p
        if window:
            hidden = hidden | (i <= p - window)
        s = (qq @ kk.nan_to_num().transpose(1, 2) * scale).masked_fill(hidden, -math.inf)
        size = (qq.abs() @ kk.nan_to_num().abs().transpose(1, 2) * abs(scale)).masked_fill(hidden, 0.0)
        off = dim * 2.0 ** -23 * (size.amax(-1, keepdim=True) if n else torch.zeros(hq, m, 1))
        w = torch.softmax(s, -1).masked_fill(hidden, 0.0)
        share = 2 * off + 2.0 ** -19
        o = w @ vv.nan_to_num()
        out[cu[b]:cu[b + 1]] = o.transpose(0, 1)
        tol[cu[b]:cu[b + 1]] = (o.abs() * half_step + (share + 2.0 ** -11) * (w @ vv.nan_to_num().abs())
                                + 2.0 ** -32 * ((~hidden).double() @ vv.nan_to_num().abs())
                                + torch.finfo(torch.float16).tiny * (q.dtype == torch.float16)).transpose(0, 1) + 1e-12
        weights.append(w.unflatten(0, (hk, -1)).sum((1, 2)))
        weights_tol.append((w * share).unflatten(0, (hk, -1)).sum((1, 2)))
    return out, tol, weights, weights_tol


def chosen(w, n, budget, recent, sinks):
    """Token indices that stay, of one head's weights ``w`` (a list of numbers)."""
    if n <= budget:
        return list(range(n))
    sure = [i for i in range(n) if i < sinks or i >= n - recent]
    rest = [i for i in range(sinks, n - recent)]
    rest.sort(key=lambda i: (0 if math.isnan(w[i]) else 1, -w[i] if not math.isnan(w[i]) else 0.0, i))
    return sorted(sure + rest[:budget - len(sure)])
