"""Kernels of the paged K/V pool of 4 bits against loops in 64 bits (``plain_kv_fp4``)."""
import math

import pytest
import torch

import plain_kv_fp4 as plain
from minisglang_rdna4_b200 import ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(pages, hk, page, dim, seed=0, powers=True):
    """A pool that the store filled with random rows, and the factors of its heads."""
    g = torch.Generator("cuda").manual_seed(seed)
    cache = torch.zeros(pages, hk, page // 16, 18 * dim, dtype=torch.uint8, device="cuda")
    if powers:
        ks, vs = (2.0 ** torch.randint(lo, lo + 3, (hk,), generator=g, device="cuda") for lo in (-6, -8))
    else:
        ks, vs = (0.02 + 0.01 * torch.rand(hk, generator=g, device="cuda") for _ in range(2))
    k, v = (torch.randn(pages * page, hk, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    k[..., 5::31] *= 5
    ops.store_kv_fp4(k, v, cache, torch.arange(pages * page, dtype=torch.int32, device="cuda"), ks, vs)
    return cache, ks, vs, k, v


def tables(lens, page, spare=2, seed=0, width=None):
    """Pages in a random order; unused entries name the last page."""
    need = [-(-n // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    width = width or max(need + [1])
    rows, at = [], 0
    for n in need:
        rows.append(order[at:at + n] + [order[-1]] * (width - n))
        at += n
    return ints(rows), total


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hk,page", [(1, 16), (3, 48), (8, 64)])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
def test_store_and_load(dim, hk, page, dtype):
    torch.manual_seed(dim + hk)
    pages, rows = 5, 2 * page + 5
    cache = torch.full((pages, hk, page // 16, 18 * dim), 0x11, dtype=torch.uint8, device="cuda")
    before = plain.values(cache)
    ks, vs = 2.0 ** torch.randint(-6, -2, (hk,), device="cuda"), 2.0 ** torch.randint(-9, -5, (hk,), device="cuda")
    # rows of a projection: keys and values lie in wider rows
    wide = torch.randn(rows, 2 * hk * dim + 24, device="cuda").to(dtype)
    k, v = wide[:, 8:8 + hk * dim], wide[:, 8 + hk * dim:8 + 2 * hk * dim]
    loc = torch.randperm(pages * page, device="cuda")[:rows].int()
    loc[3], loc[7] = -1, pages * page
    weights = torch.ones(pages, hk, page, device="cuda")
    ops.store_kv_fp4(k, v, cache, loc, ks, vs, weights)
    inside = (loc >= 0) & (loc < pages * page)
    at = loc[inside].long().cpu()
    got = plain.values(cache, ks, vs)
    for x, y, old, head in zip(got, (k, v), before, (ks, vs)):
        want = (old * head.cpu().double()[:, None, None]).transpose(1, 2).flatten(0, 1)
        want[at] = plain.rounded(y.reshape(rows, hk, dim)[inside], head)
        assert torch.equal(x.transpose(1, 2).flatten(0, 1), want)
    assert torch.equal(weights.transpose(1, 2).flatten(0, 1).cpu()[at], torch.zeros(len(at), hk))
    assert int(weights.sum()) == (pages * page - len(at)) * hk
    back = ops.load_kv_fp4(cache, loc, ks, vs, dtype)
    for x, y in zip(back, got):
        want = torch.zeros(rows, hk, dim, dtype=torch.float64)
        want[inside.cpu()] = y.transpose(1, 2).flatten(0, 1)[at]
        assert torch.equal(x.cpu().double(), want.to(dtype).double())
    # rows that do not lie on 16 bytes, and a copy's
    odd = torch.randn(rows, hk * dim + 3, device="cuda").to(dtype)[:, 3:]
    ops.store_kv_fp4(odd, odd, cache, loc, ks, vs)
    first = cache.clone()
    ops.store_kv_fp4(odd.contiguous().view(rows, hk, dim), odd.contiguous().view(rows, hk, dim), cache, loc, ks, vs)
    assert torch.equal(first, cache)
    # a bounds-checking build names the slot behind the pool, nothing else (rows without a slot, -1, are ordinary)
    from minisglang_rdna4_b200.ops import cuda as K

    assert all(line.endswith(f"value {pages * page} limit {pages * page}") for line in K.bounds_report())


@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
def test_codes_are_those_of_a_division(dtype):
    """Every finite magnitude of the type over scales of heads that are no powers of two: the code of x / (scale * head) as fp32
    divides, which the store's quotients have to round to."""
    bits = torch.arange(1, 0x7F80 if dtype == torch.bfloat16 else 0x7C00, dtype=torch.int32, device="cuda").to(torch.int16)
    x = bits.view(dtype)
    x = torch.cat([x, -x])
    x = x[(x.abs() < 60000.0) & (x.abs() > 1e-4)]
    x = x[torch.randperm(x.numel(), generator=torch.Generator("cuda").manual_seed(2), device="cuda")]
    x = torch.cat([x, x[:(-x.numel()) % 128]]).view(-1, 1, 128)
    rows = x.shape[0]
    for head in (0.0137, 0.77, 3.1, 29.0, 33.3):
        cache = torch.zeros(-(-rows // 16), 1, 1, 18 * 128, dtype=torch.uint8, device="cuda")
        h = torch.tensor([head], device="cuda")
        ops.store_kv_fp4(x, x, cache, torch.arange(rows, dtype=torch.int32, device="cuda"), h, h)
        from minisglang_rdna4_b200.ops import ref_fp4

        code, sf = ref_fp4.quantise(x, h)
        got = ref_fp4.unpack_tiles(cache)
        for c, s in ((got[0], got[2]), (got[1], got[3])):
            assert torch.equal(s.reshape(-1, 8)[:rows], sf.reshape(-1, 8))
            assert torch.equal(c.reshape(-1, 64)[:rows], code.reshape(-1, 64))


def test_store_of_special_rows():
    # (2 alone in its block: 2 / 6 lies between the scales 0.3125 and 0.34375, nearer to the second, 6 times which is held)
    cache = torch.full((1, 1, 1, 18 * 64), 0x55, dtype=torch.uint8, device="cuda")
    k = torch.zeros(4, 1, 64, device="cuda")
    k[1, 0, :3] = torch.tensor([1e30, -1e30, 1.0])
    k[2, 0, 20], k[2, 0, 40], k[3, 0] = math.nan, 2.0, 1e-30
    k = k.bfloat16()
    ops.store_kv_fp4(k, k, cache, ints([0, 1, 2, 3]))
    for x in plain.values(cache):
        x = x[0, 0]
        assert (x[0] == 0).all() and (x[3] == 0).all() and x[1, :3].tolist() == [2688.0, -2688.0, 0.0]
        assert x[2, 16:32].isnan().all() and x[2, 40] == 6 * 0.34375 and not x[2, 32:].isnan().any()
    k[0, 0, 0] = math.inf
    ops.store_kv_fp4(k[:1], k[:1], cache, ints([0]))
    assert plain.values(cache)[0][0, 0, 0, 0] == 2688.0


def attend(lens, news, hq, hk, dim, dtype=torch.bfloat16, page=16, window=0, weighed=False, seed=0, powers=True, scale=None, **kw):
    table, pages = tables(lens, page, seed=seed)
    cache, ks, vs, _, _ = make(pages, hk, page, dim, seed, powers)
    g = torch.Generator("cuda").manual_seed(seed + 1)
    cu = ints([0] + torch.tensor(news).cumsum(0).tolist())
    q = torch.randn(sum(news), hq, dim, generator=g, device="cuda").to(dtype)
    weights = torch.rand(pages, hk, page, generator=g, device="cuda") if weighed else None
    before = weights.clone() if weighed else None
    scale = scale or dim ** -0.5
    lens = ints(lens)
    out = ops.paged_attention_fp4(q, cache, table, cu, lens, scale, k_scale=ks, v_scale=vs, window=window, weights=weights,
                                  **{"max_q": max(news), "max_kv": int(lens.max()), **kw})
    want, tol, w, w_tol = plain.attention(q, *plain.values(cache, ks, vs), table, cu, lens, scale, window)
    assert torch.isfinite(out).all()
    assert ((out.cpu().double() - want).abs() <= tol).all(), float(((out.cpu().double() - want).abs() / tol).max())
    if weighed:
        expect, room = before.cpu().double(), torch.zeros(before.shape, dtype=torch.float64)
        for b, n in enumerate(lens.tolist()):
            i = torch.arange(n)
            at = (table[b].cpu().long()[i // page], slice(None), i % page)
            expect[at] += w[b].T
            room[at] += w_tol[b].T
        room = room + expect * 2.0 ** -22                     # sums over the heads and with what was there
        off = (weights.cpu().double() - expect).abs()
        assert (off <= room).all(), float((off / room).max())
        assert torch.equal(weights.cpu()[room == 0], before.cpu()[room == 0])
    return out


DECODE = {
    "one": [1], "tile": [16], "over": [17], "edges": [15, 16, 17, 31, 32, 33, 63, 64, 65], "none": [0, 5, 0], "alone": [700],
    "ragged": [90, 3500, 64, 1, 1200, 65, 2500, 0, 333], "many": [(37 * i) % 300 + 1 for i in range(200)], "long": [20011],
}


@pytest.mark.parametrize("lens", DECODE.values(), ids=DECODE.keys())
@pytest.mark.parametrize("weighed", [False, True], ids=["", "weighed"])
def test_decode(lens, weighed):
    attend(lens, [1] * len(lens), 8, 2, 128, weighed=weighed)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(1, 1), (2, 2), (5, 1), (14, 2), (32, 4), (16, 1), (24, 8), (40, 2)])
@pytest.mark.parametrize("dtype", TYPES, ids=["bf16", "fp16"])
def test_decode_heads(dim, hq, hk, dtype):
    attend([333, 50, 1], [1, 1, 1], hq, hk, dim, dtype, page=32, weighed=hq % 2 == 0, powers=False)


@pytest.mark.parametrize("window", [1, 15, 16, 100, 5000])
def test_windows(window):
    attend([1, 200, 17, 1000], [1] * 4, 8, 2, 64, window=window, weighed=True, page=64)
    attend([1, 200, 17, 1000], [1, 30, 17, 9], 8, 2, 128, window=window, weighed=True)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("hq,hk", [(4, 4), (7, 1), (8, 2), (16, 1)])
@pytest.mark.parametrize("weighed", [False, True], ids=["", "weighed"])
def test_rows(dim, hq, hk, weighed):
    """Requests that bring 0, 1 or many rows, up to all of their tokens."""
    attend([30, 100, 513, 40, 77], [30, 0, 5, 1, 70], hq, hk, dim, weighed=weighed, powers=False)


PROMPTS = [(8, 2, 128, torch.bfloat16, 0), (8, 2, 128, torch.float16, 0), (7, 1, 128, torch.bfloat16, 0), (6, 6, 64, torch.bfloat16, 0),
           (8, 4, 64, torch.bfloat16, 0), (8, 2, 128, torch.bfloat16, 100), (5, 1, 64, torch.bfloat16, 300),
           (7, 1, 128, torch.float16, 0), (6, 6, 64, torch.float16, 0), (8, 4, 64, torch.float16, 40), (8, 2, 128, torch.float16, 100)]


@pytest.mark.parametrize("hq,hk,dim,dtype,window", PROMPTS, ids=["-".join(map(str, p)) for p in PROMPTS])
def test_prompts(hq, hk, dim, dtype, window):
    """With a plan: the tensor-core form. Its probabilities go into the second product in q's type."""
    lens, news, page = [300, 129, 128, 700, 5], [300, 128, 5, 200, 5], 32
    table, pages = tables(lens, page)
    cache, ks, vs, _, _ = make(pages, hk, page, dim, powers=False)
    # what lies behind the requests and in no page may be anything
    cache[int(table[4, -1])] = 0x7F
    cu = ints([0] + torch.tensor(news).cumsum(0).tolist())
    q = torch.randn(sum(news), hq, dim, device="cuda").to(dtype)
    plan = ops.prefill_plan_fp4(q, cache, cu.cpu().numpy(), ints(lens).cpu().numpy(), window)
    assert plan is not None
    out = ops.paged_attention_fp4(q, cache, table, cu, ints(lens), 0.1, k_scale=ks, v_scale=vs, window=window, max_q=300, max_kv=700,
                                  plan=plan)
    values = plain.values(cache, ks, vs)
    want, tol, _, _ = plain.attention(q, *values, table, cu, ints(lens), 0.1, window)
    if dtype == torch.bfloat16:
        # 8 bits in place of 11 for the probabilities: the sum of weighted magnitudes times 2^-8 more. That sum is the attention
        # over the magnitudes of the values
        size = torch.zeros_like(want)
        weight = lambda v: plain.attention(q, values[0], v, table, cu, ints(lens), 0.1, window)[0]  # noqa: E731
        size = weight(values[1].abs())
        tol = tol + size * 2.0 ** -8
    assert torch.isfinite(out).all()
    assert ((out.cpu().double() - want).abs() <= tol).all(), float(((out.cpu().double() - want).abs() / tol).max())
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(q, cache, table, cu, ints(lens), 0.1, window=window + 1, max_q=300, plan=plan)
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(q, cache, table, cu, ints(lens), -0.1, window=window, max_q=300, plan=plan)


def test_plan_of_another_step():
    """A plan whose rows, requests or tokens the step does not have is refused on the host."""
    n = lambda *x: torch.tensor(x, dtype=torch.int32).numpy()  # noqa: E731
    cache = torch.zeros(40, 2, 2, 18 * 128, dtype=torch.uint8, device="cuda")
    q = torch.zeros(300, 4, 128, device="cuda", dtype=torch.bfloat16)
    table, cu, lens = torch.arange(20, dtype=torch.int32, device="cuda").view(2, 10), ints([0, 100, 300]), ints([150, 310])
    plan = ops.prefill_plan_fp4(q, cache, n(0, 100, 300), n(150, 310))
    ops.paged_attention_fp4(q, cache, table, cu, lens, 0.1, max_q=200, plan=plan)
    for fewer_rows, fewer_requests, fewer_pages in ((q[:299], table, table), (q, table[:1], table), (q, table, table[:, :9])):
        b = 1 if fewer_requests.shape[0] == 1 else 2
        t = fewer_pages[:b]
        with pytest.raises(ValueError, match="made for 2 requests"):
            ops.paged_attention_fp4(fewer_rows, cache, t, cu[:b + 1], lens[:b], 0.1, max_q=200, plan=plan)


def test_longest_request_is_not_read_in_a_capture():
    cache = torch.zeros(4, 2, 1, 18 * 64, dtype=torch.uint8, device="cuda")
    q = torch.zeros(1, 4, 64, device="cuda", dtype=torch.bfloat16)
    args = (q, cache, ints([[0]]), ints([0, 1]), ints([5]), 0.1)
    ops.paged_attention_fp4(*args, max_q=1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="max_q of 0"):
            ops.paged_attention_fp4(*args)
        out = ops.paged_attention_fp4(*args, max_q=1)
    graph.replay()
    assert torch.isfinite(out).all()


def test_steps_that_take_no_prompt_form():
    cache = torch.zeros(4, 2, 1, 18 * 128, dtype=torch.uint8, device="cuda")
    n = lambda *x: torch.tensor(x, dtype=torch.int32).numpy()  # noqa: E731
    q = torch.zeros(200, 4, 128, device="cuda", dtype=torch.bfloat16)
    assert ops.prefill_plan_fp4(q, cache, n(0, 200), n(200)) is not None
    assert ops.prefill_plan_fp4(q, cache, n(0, 200), n(100)) is None              # more rows than tokens
    assert ops.prefill_plan_fp4(q[:20], cache, n(0, 20), n(50000)) is None        # few rows for the keys
    assert ops.prefill_plan_fp4(q[:0], cache, n(0), n()) is None
    with pytest.raises(ValueError):
        ops.prefill_plan_fp4(q, cache, n(0, 200), n(200, 200))
    wide = torch.zeros(4, 2, 1, 18 * 256, dtype=torch.uint8, device="cuda")
    assert ops.prefill_plan_fp4(torch.zeros(200, 4, 256, device="cuda").half(), wide, n(0, 200), n(200)) is None


def test_more_rows_than_tokens():
    """Rows in front of the text see nothing."""
    attend([3, 0, 20], [5, 2, 20], 4, 2, 64, weighed=True)


def test_bounds_may_be_loose_or_read_from_the_device():
    for kw in (dict(max_q=9, max_kv=4096), dict(max_q=0, max_kv=0)):
        attend([70, 200], [1, 4], 8, 2, 128, weighed=True, **kw)
    attend([70, 200], [1, 1], 8, 2, 128, weighed=True, max_q=0, max_kv=1 << 20)


def test_more_rows_than_said_and_windows_without_an_end():
    attend([70, 200, 33], [3, 9, 33], 8, 2, 128, weighed=True, max_q=1)
    attend([70, 200], [1, 4], 8, 2, 64, weighed=True, window=(1 << 40) + 1)


def test_more_requests_than_a_launch_takes():
    lens = [(29 * i) % 70 for i in range(700)]
    attend(lens, [1] * 700, 4, 2, 64, weighed=True)
    attend([n + 3 for n in lens], [(7 * i) % 4 for i in range(700)], 4, 2, 64, weighed=True)


def test_a_scale_below_zero():
    attend([70, 200], [1, 4], 8, 2, 128, weighed=True, scale=-0.1)


def test_large_scores():
    """Scores of some hundreds: one token takes all."""
    attend([300, 1000], [1, 3], 8, 2, 128, scale=6.0)


def test_what_lies_behind_a_request_does_not_matter():
    lens, page = [21, 90], 16
    table, pages = tables(lens, page)
    cache, ks, vs, _, _ = make(pages, 2, page, 128)
    q = torch.randn(2, 8, 128, device="cuda").bfloat16()
    run = lambda: ops.paged_attention_fp4(q, cache, table, ints([0, 1, 2]), ints(lens), 0.1, k_scale=ks, v_scale=vs, max_q=1,  # noqa: E731
                                          max_kv=90)
    first = run()
    bad = torch.full((1, 2, 128), math.nan, device="cuda").bfloat16()
    for i in range(21, 32):
        ops.store_kv_fp4(bad, bad, cache, ints([int(table[0, 1]) * page + i % page]), ks, vs)
    for i in range(90, 96):
        ops.store_kv_fp4(bad, bad, cache, ints([int(table[1, 5]) * page + i % page]), ks, vs)
    assert torch.equal(first, run())
    # a NaN that is seen shows
    ops.store_kv_fp4(bad, bad, cache, ints([int(table[0, 1]) * page + 20 % page]), ks, vs)
    assert run()[0].isnan().all() and torch.equal(run()[1], first[1])


def test_same_results_every_time():
    kw = dict(lens=[3000, 17, 900, 0, 20000], news=[1] * 5, hq=8, hk=2, dim=128)
    assert torch.equal(attend(**kw, weighed=True), attend(**kw, weighed=True))


def test_a_table_of_any_stride_and_queries_of_any_stride():
    lens, page = [40, 60], 16
    table, pages = tables(lens, page)
    cache, ks, vs, _, _ = make(pages, 2, page, 64)
    q = torch.randn(2, 4, 64, device="cuda").bfloat16()
    run = lambda q, t: ops.paged_attention_fp4(q, cache, t, ints([0, 1, 2]), ints(lens), 0.1, k_scale=ks, v_scale=vs)  # noqa: E731
    want = run(q, table)
    wide = torch.zeros(2, 11, dtype=torch.int32, device="cuda")
    wide[:, 3:7] = table
    assert torch.equal(run(torch.stack([q, q], 2).flatten(1, 2)[:, ::2], wide[:, 3:7]), want)
    assert torch.equal(run(q, table.t().contiguous().t()), want)


def test_pool_beyond_32_bits():
    page, hk, dim = 64, 8, 128
    pages = (1 << 32) // (hk * 4 * 18 * dim) + 40
    cache = torch.zeros(pages, hk, page // 16, 18 * dim, dtype=torch.uint8, device="cuda")
    n = 150
    k, v = (torch.randn(n, hk, dim, device="cuda").bfloat16() for _ in range(2))
    table = ints([[pages - 1, 3, pages - 7]])
    loc = torch.cat([torch.arange(page, device="cuda") + p * page for p in table[0].tolist()])[:n].int()
    weights = torch.zeros(pages, hk, page, device="cuda")
    ops.store_kv_fp4(k, v, cache, loc)
    q = torch.randn(1, 16, dim, device="cuda").bfloat16()
    out = ops.paged_attention_fp4(q, cache, table, ints([0, 1]), ints([n]), 0.1, max_q=1, max_kv=n, weights=weights)
    small = cache[table[0].long()]
    want, tol, w, _ = plain.attention(q, *plain.values(small), ints([[0, 1, 2]]), ints([0, 1]), ints([n]), 0.1)
    assert ((out.cpu().double() - want).abs() <= tol).all()
    got = weights[table[0].long()].transpose(0, 1).flatten(1)[:, :n].cpu().double()
    assert (got - w[0]).abs().max() < 1e-5
    back = ops.load_kv_fp4(cache, loc)
    assert all(torch.equal(x.cpu().double(), plain.rounded(y, None)) for x, y in zip(back, (k, v)))
    kept, _ = ops.evict_kv_fp4(cache, weights, table, ints([n]), ints([[pages - 3]]), 50, 5)
    rows = kept[0, 0].long()
    slots = (torch.arange(50, device="cuda") + (pages - 3) * page).int()
    assert all(torch.equal(x[:, 0], y[rows, 0]) for x, y in zip(ops.load_kv_fp4(cache, slots), back))


# ------------------------------------------------------------------------------------------ eviction
EVICT = [([50, 21, 5, 0, 64, 22], 21, 6, 2), ([100, 3000, 900], 64, 64, 0), ([100, 3000, 900], 64, 0, 64), ([70, 2000], 33, 0, 0),
         ([9000, 8193, 12000], 2048, 100, 4), ([40], 1, 0, 0), ([60000], 1000, 10, 1)]


@pytest.mark.parametrize("lens,budget,recent,sinks", EVICT, ids=[str(e[0][0]) + "_to_" + str(e[1]) for e in EVICT])
@pytest.mark.parametrize("dim,page,layers", [(64, 16, 0), (128, 32, 2), (256, 16, 1)])
def test_evict(lens, budget, recent, sinks, dim, page, layers):
    hk = 2
    slim = -(-budget // page)
    table, pages = tables(lens, page, spare=len(lens) * slim + 1)
    new = torch.tensor([p for p in range(pages) if p not in set(table.flatten().tolist())][:len(lens) * slim],
                       dtype=torch.int32, device="cuda").view(len(lens), slim)
    g = torch.Generator("cuda").manual_seed(1)
    cache = torch.randint(0, 256, (max(layers, 1), pages, hk, page // 16, 18 * dim), generator=g, device="cuda", dtype=torch.uint8)
    weights = torch.rand(max(layers, 1), pages, hk, page, generator=g, device="cuda")
    weights = torch.round(weights ** 4 * 256)                # many equal ones
    weights[0, table[0, 0], 0, 3], weights[0, table[0, 0], 1, 9] = math.nan, math.inf
    weights[0, table[0, 0], 1, 5], weights[0, table[0, 0], 1, 6] = -0.0, -3.0
    if not layers:
        cache, weights = cache[0], weights[0]
    old, old_w = cache.clone(), weights.clone()
    kept, now = ops.evict_kv_fp4(cache, weights, table, ints(lens), new, budget, recent, sinks,
                                 **({"max_kv": max(lens)} if dim == 128 else {}))
    assert now.tolist() == [min(n, budget) for n in lens]
    from minisglang_rdna4_b200.ops import ref_fp4

    for a, w, a0, w0, kept in zip(*((x if layers else x[None]) for x in (cache, weights, old, old_w, kept))):
        want, want_w = a0.clone(), w0.clone()
        stay, _ = ref_fp4.evict_kv_fp4(want, want_w, table, ints(lens), new, budget, recent, sinks)
        if max(lens) <= 9000:
            for b, n in enumerate(lens):
                i = torch.arange(n)
                for h in range(hk):
                    mine = w0[table[b].long()[i.cuda() // page], h, i.cuda() % page].tolist()
                    s = plain.chosen(mine, n, budget, recent, sinks)
                    assert kept[b, h].tolist() == s + [-1] * (budget - len(s))
        assert torch.equal(kept, stay)
        assert torch.equal(a, want) and torch.equal(w.nan_to_num(-7.0), want_w.nan_to_num(-7.0))


@pytest.mark.parametrize("requests", [13, 32, 33])
def test_evict_more_than_runs_at_once(requests):
    """(layer, request, head) units in several waves: requests in the order of their lengths, equal, empty and short ones among them."""
    hk, page, dim, layers, budget = 4, 16, 64, 5, 40
    lens = [(i * 37) % 200 if i % 4 else 120 for i in range(requests)]
    table, pages = tables(lens, page, spare=3 * requests + 1)
    new = torch.tensor([p for p in range(pages) if p not in set(table.flatten().tolist())][:3 * requests],
                       dtype=torch.int32, device="cuda").view(requests, 3)
    g = torch.Generator("cuda").manual_seed(3)
    cache = torch.randint(0, 256, (layers, pages, hk, 1, 18 * dim), generator=g, device="cuda", dtype=torch.uint8)
    weights = torch.round(torch.rand(layers, pages, hk, page, generator=g, device="cuda") * 50)
    want, want_w = cache.clone(), weights.clone()
    from minisglang_rdna4_b200.ops import ref_fp4

    kept, now = ops.evict_kv_fp4(cache, weights, table, ints(lens), new, budget, 5, 2)
    stay, want_now = ref_fp4.evict_kv_fp4(want, want_w, table, ints(lens), new, budget, 5, 2)
    assert torch.equal(now, want_now.to(now)) and torch.equal(kept, stay)
    assert torch.equal(cache, want) and torch.equal(weights, want_w)


@pytest.mark.parametrize("lens,budget,recent,sinks", [([131, 997, 4099], 65, 7, 3), ([50021], 1025, 3, 13), ([18, 19, 20, 21, 22], 17, 1, 15)],
                         ids=["short", "beyond_shared_memory", "one_candidate"])
@pytest.mark.parametrize("offset", [0, 1], ids=["aligned", "on_4_bytes"])
def test_evict_weights_anywhere(lens, budget, recent, sinks, offset):
    """Ends of the candidates inside groups of four tokens; weights that begin on 4 bytes, their layers an odd distance apart."""
    hk, page, dim, layers, slim = 2, 32, 64, 2, -(-budget // 32)
    table, pages = tables(lens, page, spare=len(lens) * slim + 1)
    new = torch.tensor([p for p in range(pages) if p not in set(table.flatten().tolist())][:len(lens) * slim],
                       dtype=torch.int32, device="cuda").view(len(lens), slim)
    g = torch.Generator("cuda").manual_seed(2)
    cache = torch.randint(0, 256, (layers, pages, hk, page // 16, 18 * dim), generator=g, device="cuda", dtype=torch.uint8)
    stride = pages * hk * page + 3 * offset
    weights = torch.zeros(layers * stride + 8, device="cuda")[offset:].as_strided((layers, pages, hk, page), (stride, hk * page, page, 1))
    weights.copy_(torch.round(torch.rand(weights.shape, generator=g, device="cuda") ** 3 * 40))
    want, want_w = cache.clone(), weights.clone()
    from minisglang_rdna4_b200.ops import ref_fp4

    kept, _ = ops.evict_kv_fp4(cache, weights, table, ints(lens), new, budget, recent, sinks)
    stay, _ = ref_fp4.evict_kv_fp4(want, want_w, table, ints(lens), new, budget, recent, sinks)
    assert torch.equal(kept, stay) and torch.equal(cache, want) and torch.equal(weights, want_w)


def test_a_conversation_is_stored_weighed_and_cut():
    """Store, weighed attention, eviction, new tokens, attention again, in a captured graph and eagerly."""
    page, hk, hq, dim, lens, budget = 16, 2, 8, 128, [700, 90, 1500], 128
    slim = budget // page + 1
    torch.manual_seed(5)
    pages = 44 + 6 + 94 + 3 * slim              # of the requests, and those that they are cut down into
    ks, vs = torch.full((hk,), 1 / 64, device="cuda"), torch.full((hk,), 1 / 128, device="cuda")
    order = torch.randperm(pages).int().cuda()
    table = torch.zeros(3, 94, dtype=torch.int32, device="cuda")
    table[0, :44], table[1, :6], table[2] = order[:44], order[44:50], order[50:144]
    new = order[144:].view(3, slim)
    cache = torch.zeros(pages, hk, 1, 18 * dim, dtype=torch.uint8, device="cuda")
    weights = torch.full((pages, hk, page), 9.0, device="cuda")
    total = sum(lens)
    k, v = (torch.randn(total + 3, hk, dim, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(total + 3, hq, dim, device="cuda").bfloat16()
    loc = torch.cat([(table[b].long()[i // page] * page + i % page) for b, n in enumerate(lens)
                     for i in [torch.arange(n, device="cuda")]]).int()
    cu, n = ints([0, 700, 790, 2290]), ints(lens)

    def turn():
        ops.store_kv_fp4(k[:total], v[:total], cache, loc, ks, vs, weights)
        first = ops.paged_attention_fp4(q[:total], cache, table, cu, n, 0.1, k_scale=ks, v_scale=vs, max_q=1500, max_kv=1500,
                                        weights=weights)
        kept, now = ops.evict_kv_fp4(cache, weights, table, n, new, budget, 20, 4)
        at = torch.gather(new, 1, (now // page)[:, None].long())[:, 0] * page + now % page
        ops.store_kv_fp4(k[total:], v[total:], cache, at, ks, vs, weights)
        last = ops.paged_attention_fp4(q[total:], cache, new, steps, now + 1, 0.1, k_scale=ks, v_scale=vs, max_q=1, max_kv=budget + 1, weights=weights)
        return first, kept, now, last, weights.clone()

    steps = ints([0, 1, 2, 3])
    eager = [x.clone() for x in turn()]
    kk, vv = plain.rounded(k, ks), plain.rounded(v, vs)
    for b in range(3):
        for h in range(hq):
            at = eager[1][b, h // 4].cpu().long()
            at = torch.cat([at[at >= 0] + int(cu[b]), torch.tensor([total + b])])
            w = torch.softmax(q[total + b, h].cpu().double() @ kk[at, h // 4].T * 0.1, -1)
            assert (eager[3][b, h].cpu().double() - w @ vv[at, h // 4]).abs().max() < 2.0 ** -7
    assert torch.isfinite(eager[4]).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        turn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = turn()
    cache.zero_()
    weights.fill_(1.0)
    graph.replay()
    weights_then = captured[4].clone()
    graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(captured[:4], eager[:4]))
    for b, m in enumerate(eager[2].tolist()):            # slots behind the rows keep what was there: 9 before, 1 now
        mine = [w[new[b].long()].transpose(0, 1).flatten(1) for w in (captured[4], eager[4])]
        assert torch.equal(mine[0][:, :m + 1], mine[1][:, :m + 1])
        assert (mine[0][:, m + 1:] == 1.0).all() and (mine[1][:, m + 1:] == 9.0).all()
    assert torch.equal(weights_then, captured[4])


def test_two_streams_at_once():
    lens = [5000, 300, 9000]
    table, pages = tables(lens, 16)
    cache, ks, vs, _, _ = make(pages, 2, 16, 128)
    qs = [torch.randn(3, 8, 128, device="cuda").bfloat16() for _ in range(2)]
    cu, n = ints([0, 1, 2, 3]), ints(lens)
    run = lambda q: ops.paged_attention_fp4(q, cache, table, cu, n, 0.1, k_scale=ks, v_scale=vs, max_q=1, max_kv=9000)  # noqa: E731
    want = [run(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(qs[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in (0, 1) for x in got[i])


def test_refusals():
    cache, ks, vs, k, v = make(4, 2, 16, 64)
    loc = ints([1, 2])
    with pytest.raises(ValueError):
        ops.store_kv_fp4(k[:2], v[:2], cache, loc.cpu(), ks, vs)
    with pytest.raises(ValueError):
        ops.store_kv_fp4(k[:2].cpu(), v[:2], cache, loc, ks, vs)
    with pytest.raises(ValueError):
        ops.load_kv_fp4(cache, loc, ks.cpu())
    q = torch.randn(2, 4, 64, device="cuda").half()
    with pytest.raises(ValueError):
        ops.paged_attention_fp4(q, cache, ints([[0], [1]]), ints([0, 1, 2]), ints([5, 6]).cpu(), 1.0)
    assert ops.load_kv_fp4(cache, ints([]), ks, vs)[0].shape == (0, 2, 64)
    none = ops.paged_attention_fp4(q[:0], cache, ints([[0], [1]]), ints([0, 0, 0]), ints([5, 6]), 1.0)
    assert none.shape == (0, 4, 64)
    ops.store_kv_fp4(k[:0], v[:0], cache, ints([]), ks, vs)
