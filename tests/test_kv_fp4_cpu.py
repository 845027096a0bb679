"""The paged K/V pool of 4 bits on the CPU: the plain path against loops in 64 bits, and what is refused."""
import math

import pytest
import torch

import plain_kv_fp4 as plain
from minisglang_rdna4_b200 import ops

DIMS = [64, 128, 256]


def make(pages, hk, page, dim, seed=0):
    """A pool with random rows in all slots (written by the store), and the factors of its heads (powers of two)."""
    g = torch.Generator().manual_seed(seed)
    cache = torch.zeros(pages, hk, page // 16, 18 * dim, dtype=torch.uint8)
    ks, vs = 2.0 ** torch.randint(-6, -3, (hk,), generator=g), 2.0 ** torch.randint(-8, -5, (hk,), generator=g)
    k, v = (torch.randn(pages * page, hk, dim, generator=g).bfloat16() for _ in range(2))
    ops.store_kv_fp4(k, v, cache, torch.arange(pages * page, dtype=torch.int32), ks, vs)
    return cache, ks, vs, k, v


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("page", [16, 48])
def test_store_gives_the_nearest_values(dim, page):
    cache, ks, vs, k, v = make(3, 2, page, dim)
    got = plain.values(cache, ks, vs)
    for x, y, head in zip(got, (k, v), (ks, vs)):
        assert torch.equal(x.transpose(1, 2).flatten(0, 1), plain.rounded(y, head))
    loc = torch.randperm(3 * page)[:20].int()
    for x, y in zip(ops.load_kv_fp4(cache, loc, ks, vs, torch.float16), got):
        assert torch.equal(x.double(), y.transpose(1, 2).flatten(0, 1)[loc.long()].half().double())


def test_store_of_special_rows():
    # (2 alone in its block: 2 / 6 lies between the scales 0.3125 and 0.34375, nearer to the second, 6 times which is held)
    cache = torch.full((1, 1, 1, 18 * 64), 0x55, dtype=torch.uint8)
    k = torch.zeros(4, 1, 64)
    k[1, 0, :3] = torch.tensor([1e30, -1e30, 1.0])         # saturates
    k[2, 0, 20] = math.nan                                  # its block only
    k[2, 0, 40] = 2.0
    k[3, 0] = 1e-30                                         # too small for any scale
    k = k.bfloat16()
    weights = torch.ones(1, 1, 16)
    ops.store_kv_fp4(k, k, cache, ints([0, 1, 2, -1]), None, None, weights)
    ops.store_kv_fp4(k[3:], k[3:], cache, ints([16]))       # behind the pool
    ops.store_kv_fp4(k[3:], k[3:], cache, ints([3]))
    x = plain.values(cache)[0][0, 0]
    assert (x[0] == 0).all() and (x[3] == 0).all()
    assert x[1, :3].tolist() == [6 * 448.0, -6 * 448.0, 0.0]
    assert x[2, 16:32].isnan().all() and x[2, 40] == 6 * 0.34375 and not x[2, 32:].isnan().any()
    assert weights[0, 0].tolist() == [0.0] * 3 + [1.0] * 13
    same = ops.load_kv_fp4(cache, ints([2, 16, -5]))[0]
    assert same[0, 0, 16:32].isnan().all() and (same[1:] == 0).all()


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("window", [0, 1, 20])
def test_attention(dim, window):
    cache, ks, vs, _, _ = make(9, 2, 16, dim)
    lens, news = [40, 0, 1, 33], [3, 0, 1, 1]
    table = ints([[4, 1, 7], [0, 0, 0], [2, 0, 0], [8, 3, 5]])
    cu = ints([0, 3, 3, 4, 5])
    q = torch.randn(5, 6, dim).half()
    weights = torch.rand(9, 2, 16)
    before = weights.clone()
    out = ops.paged_attention_fp4(q, cache, table, cu, ints(lens), 0.2, k_scale=ks, v_scale=vs, window=window, weights=weights)
    want, tol, w, w_tol = plain.attention(q, *plain.values(cache, ks, vs), table, cu, ints(lens), 0.2, window)
    assert ((out.double() - want).abs() <= tol).all()
    for b, n in enumerate(lens):
        for i in range(n):
            page = int(table[b, i // 16])
            got = weights[page, :, i % 16].double() - before[page, :, i % 16].double()
            assert ((got - w[b][:, i]).abs() <= w_tol[b][:, i] + 2.0 ** -22).all(), news


@pytest.mark.parametrize("layered", [False, True])
def test_evict(layered):
    page, budget, recent, sinks = 16, 21, 6, 2
    cache, ks, vs, _, _ = make(30, 2, page, 64)
    lens = [50, 21, 5, 0, 64]
    table = ints([[0, 1, 2, 3], [4, 5, 5, 5], [6, 6, 6, 6], [7, 7, 7, 7], [8, 9, 10, 11]])
    new = ints([[12, 13], [14, 15], [16, 17], [18, 19], [20, 21]])
    weights = torch.randint(0, 4, (30, 2, page)).float()
    weights[1, 0, 3] = math.nan
    weights[2, 1, 1], weights[0, 1, 7] = math.inf, -math.inf
    if layered:
        cache, weights = torch.stack([cache, cache.flip(0)]), torch.stack([weights, weights.flip(1)])
    old, old_w = cache.clone(), weights.clone()
    kept, now = ops.evict_kv_fp4(cache, weights, table, ints(lens), new, budget, recent, sinks)
    assert now.tolist() == [min(n, budget) for n in lens]
    fresh = torch.unique(new)
    for a, w, a0, w0, kept in zip(*((x if layered else x[None]) for x in (cache, weights, old, old_w, kept))):
        rest = [p for p in range(30) if p not in fresh]
        assert torch.equal(a[rest], a0[rest]) and torch.equal(w[rest].nan_to_num(9.5), w0[rest].nan_to_num(9.5))
        for b, n in enumerate(lens):
            for h in range(2):
                i = torch.arange(n)
                mine = w0[table[b].long()[i // page], h, i % page]
                stay = plain.chosen(mine.tolist(), n, budget, recent, sinks)
                assert kept[b, h].tolist() == stay + [-1] * (budget - len(stay))
                for j, s in enumerate(stay):
                    p, p0 = int(new[b, j // page]), int(table[b, s // page])
                    x, y = (plain.values(z[at:at + 1, h:h + 1])[w] for z, at, w in ((a, p, 0), (a0, p0, 0)))
                    assert torch.equal(x[0, 0, j % page], y[0, 0, s % page])
                    assert torch.equal(w[p, h, j % page].nan_to_num(9.5), w0[p0, h, s % page].nan_to_num(9.5))
        # behind the rows that stay
        last = int(new[4, 1])
        x, y = plain.values(a[last:last + 1]), plain.values(a0[last:last + 1])
        assert all(torch.equal(s[:, :, 5:], t[:, :, 5:]) for s, t in zip(x, y)) and torch.equal(w[last, :, 5:], w0[last, :, 5:])


def test_refusals():
    cache, ks, vs, k, v = make(4, 2, 16, 64)
    loc, q = ints([1, 2]), torch.randn(2, 4, 64).half()
    k, v = k[:2], v[:2]
    weights = torch.zeros(4, 2, 16)
    table, cu, lens = ints([[0, 1], [2, 3]]), ints([0, 1, 2]), ints([5, 20])
    for bad in (cache.int(), cache[0], cache[..., :500], cache.transpose(0, 1), cache[:, :, :, ::2]):
        with pytest.raises(ValueError):
            ops.store_kv_fp4(k, v, bad, loc, ks, vs)
        with pytest.raises(ValueError):
            ops.load_kv_fp4(bad, loc, ks, vs)
        with pytest.raises(ValueError):
            ops.paged_attention_fp4(q, bad, table, cu, lens, 1.0)
        with pytest.raises(ValueError):
            ops.evict_kv_fp4(bad, weights, table, lens, table, 8, 2)
    for kw in (dict(k=k.float()), dict(v=v[:1]), dict(k=k[..., :32]), dict(out_loc=loc.long()), dict(k_scale=ks.double()),
               dict(v_scale=vs[:1]), dict(weights=weights.half()), dict(weights=weights[:3]), dict(v=v.half())):
        with pytest.raises((TypeError, ValueError)):
            ops.store_kv_fp4(**{**dict(k=k, v=v, cache=cache, out_loc=loc, k_scale=ks, v_scale=vs), **kw})
    for kw in (dict(slots=loc.long()), dict(dtype=torch.float32), dict(k_scale=vs[:1])):
        with pytest.raises((TypeError, ValueError)):
            ops.load_kv_fp4(**{**dict(cache=cache, slots=loc), **kw})
    good = dict(q=q, cache=cache, block_table=table, cu_q=cu, seq_lens=lens, scale=1.0)
    for kw in (dict(q=q.double()), dict(q=q[:, :3]), dict(q=q[..., :32]), dict(q=q[:, :0]), dict(block_table=table.long()),
               dict(block_table=table[:1]), dict(cu_q=cu[:2]), dict(seq_lens=lens.long()), dict(window=-1), dict(max_q=-1),
               dict(weights=weights[:, :1]), dict(weights=weights, plan=object()), dict(k_scale=ks[:1]), dict(v_scale=vs.half())):
        with pytest.raises((TypeError, ValueError)):
            ops.paged_attention_fp4(**{**good, **kw})
    good = dict(cache=cache, weights=weights, block_table=table, seq_lens=lens, new_table=ints([[2], [3]]), budget=10, recent=4)
    for kw in (dict(weights=weights[:2]), dict(weights=weights.double()), dict(budget=0), dict(recent=-1), dict(sinks=7),
               dict(sinks=-1), dict(budget=17), dict(new_table=ints([[1]])), dict(new_table=ints([[1], [2]]).long()), dict(max_kv=-1),
               dict(block_table=table[:, :0]), dict(seq_lens=lens[:1])):
        with pytest.raises(ValueError):
            ops.evict_kv_fp4(**{**good, **kw})
    assert ops.prefill_plan_fp4(q, cache, cu.numpy(), lens.numpy()) is None


def test_a_conversation_is_stored_weighed_and_cut():
    """Store, attention with weights, eviction, a new token, attention again: as a server would go on."""
    page, hk, dim, n, budget = 16, 2, 64, 45, 20
    torch.manual_seed(3)
    cache, weights = torch.zeros(8, hk, 1, 18 * dim, dtype=torch.uint8), torch.full((8, hk, page), 7.0)
    k, v = (torch.randn(n + 1, hk, dim).bfloat16() for _ in range(2))
    q = torch.randn(n + 1, 4, dim).bfloat16()
    table, new = ints([[0, 1, 2]]), ints([[3, 4]])
    ops.store_kv_fp4(k[:n], v[:n], cache, torch.arange(n, dtype=torch.int32), weights=weights)
    ops.paged_attention_fp4(q[:n], cache, table, ints([0, n]), ints([n]), 0.125, weights=weights)
    assert abs(float(weights[:3].transpose(0, 1).flatten(1)[:, :n].sum()) - n * 4) < 1e-3      # every row gives 1 in all
    kept, lens = ops.evict_kv_fp4(cache, weights, table, ints([n]), new, budget, 4, 1)
    loc = ints([int(new[0, budget // page]) * page + budget % page])
    ops.store_kv_fp4(k[n:], v[n:], cache, loc, weights=weights)
    out = ops.paged_attention_fp4(q[n:], cache, new, ints([0, 1]), lens + 1, 0.125, weights=weights)
    kk, vv = plain.rounded(k, None), plain.rounded(v, None)
    for h in range(4):
        at = kept[0, h // 2].long().tolist() + [n]
        w = torch.softmax(q[n, h].double() @ kk[at, h // 2].T * 0.125, -1)
        assert (out[0, h].double() - w @ vv[at, h // 2]).abs().max() < 2.0 ** -7


def _config(**kw):
    from minisglang_rdna4_b200.models.config import ModelConfig

    d = dict(model_type="qwen3", hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
             intermediate_size=256, vocab_size=512, max_position_embeddings=1024, rms_norm_eps=1e-6, rope_theta=10000.0,
             tie_word_embeddings=True, architectures=["Qwen3ForCausalLM"])
    return ModelConfig.from_hf({**d, **kw})


def _engine(**kw):
    from minisglang_rdna4_b200.llm import LLM

    return LLM(**{**dict(model_config=_config(), use_dummy_weight=True, kv_cache_dtype="nvfp4", device="cpu", page_size=16,
                         max_running_req=4, num_page_override=64, seed=0), **kw})


def test_engine_serves_from_a_pool_of_4_bits():
    from minisglang_rdna4_b200 import SamplingParams
    from minisglang_rdna4_b200.kvcache import FP4KVCache

    llm = _engine()
    pool = llm.engine.kv_cache
    assert isinstance(pool, FP4KVCache) and pool.bytes_per_token == 2 * 2 * 72
    sp = SamplingParams(temperature=0.0, max_tokens=5, ignore_eos=True)
    prompts = [list(range(3, 60)), [7, 8, 9]]
    first = [o.token_ids for o in llm.generate(prompts, sp)]
    again = [o.token_ids for o in llm.generate(prompts, sp)]          # from the prefix cache
    assert first == again and all(len(t) == 5 for t in first)
    assert (pool._buf[:, :-1] != 0).any()
    llm.cache.check_integrity()
    llm.shutdown()


@pytest.mark.parametrize("kw", [dict(page_size=8), dict(spec_algorithm="ngram"), dict(model_config="wide")])
def test_engine_names_what_the_pool_does_not_go_with(kw):
    if kw.get("model_config"):
        kw = dict(model_config=_config(head_dim=32))
    with pytest.raises(ValueError, match="nvfp4"):
        _engine(**kw)


def test_pool():
    from minisglang_rdna4_b200.kvcache import FP4KVCache

    pool = FP4KVCache(3, 6, 16, 2, 64, torch.bfloat16, "cpu", weights=True)
    k, v = (torch.randn(20, 2, 64).bfloat16() for _ in range(2))
    loc = torch.arange(3, 23, dtype=torch.int32)
    pool.store_kv(k, v, loc, 1)
    for which, x in ((0, k), (1, v)):
        want = plain.rounded(x, pool.k_scale[1])
        assert torch.equal(pool.gather(1, loc, which).double(), want.bfloat16().double())
        assert (pool.gather(0, loc, which) == 0).all()
    pool.weights[:, :, :, :] = torch.rand(pool.weights.shape)
    kept, lens = pool.evict(ints([[0, 1]]), ints([23]), ints([[4]]), 10, 3, 1)
    assert kept.shape == (3, 1, 2, 10) and lens.tolist() == [10]
    assert torch.equal(pool.gather(1, ints([64 + 9]), 0), pool.gather(1, ints([22]), 0))
    for bad in (dict(head_dim=96), dict(page_size=24)):
        with pytest.raises(ValueError):
            FP4KVCache(**{**dict(num_layers=1, num_pages=2, page_size=16, num_kv_heads=1, head_dim=64, dtype=torch.bfloat16,
                                 device="cpu"), **bad})
    with pytest.raises(ValueError):
        FP4KVCache(1, 2, 16, 1, 64, torch.bfloat16, "cpu").evict(ints([[0]]), ints([5]), ints([[1]]), 4, 1)
    with pytest.raises(NotImplementedError):
        pool.k_cache(0)


REFUSED = {"speculative decoding": dict(spec_algorithm="ngram"), "cache of": dict(latent_layers=[1]), "block diffusion": dict(canvas_length=8),
           "images": dict(vision=object()), "heads differ": dict(global_head_dim=512), "96 channels": dict(head_dim=96),
           "pages of 8": dict(page_size=8)}


@pytest.mark.parametrize("why", [""] + list(REFUSED))
def test_what_the_engine_refuses(why):
    from types import SimpleNamespace

    from minisglang_rdna4_b200.engine.engine import Engine

    fields = dict(spec_algorithm="none", page_size=16, latent_layers=[], layered=False, has_fp32_kernels=False, is_mla=False,
                  canvas_length=0, vision=None, image_bidirectional=True, swa_layers=[], global_head_dim=0, num_kv_layers=2, head_dim=128,
                  model_type="some", attn_geometry=lambda i: (i, i))
    fields.update(REFUSED.get(why, {}))
    both = SimpleNamespace(**fields)
    engine = SimpleNamespace(config=both, model_config=both)
    if why:
        with pytest.raises(ValueError, match=f"nvfp4 does not go with .*{why}"):
            Engine._refuse_fp4_pool(engine)
    else:
        Engine._refuse_fp4_pool(engine)


@pytest.mark.parametrize("window,tile", [(0, 128), (0, 256), (1, 128), (100, 256), (128, 128), (5000, 128)])
def test_prompt_tables(window, tile):
    """The tables that the host library builds are those that NumPy does; a step of many requests has larger ones."""
    import numpy as np

    from minisglang_rdna4_b200.ops import host
    from minisglang_rdna4_b200.ops.cuda import PrefillPlan

    rng = np.random.default_rng(0)
    for b in (1, 2, 7, 400):
        rows = rng.integers(0, 700, b)
        lens = rows + np.where(rng.random(b) < 0.3, 0, rng.integers(0, 3000 // min(b, 20), b))
        cu = np.concatenate([[0], np.cumsum(rows)])
        want = PrefillPlan(cu, lens, "cpu", window, tile=tile)
        tables, t_pad, items, total, longest = host.prompt_tables(cu, lens, window, tile)
        assert (t_pad, items, total, longest) == (want.t_pad, want.n_items, rows.sum(), lens.max())
        assert (8 * items, 8 * items + t_pad // 128) == (want.off_blk, want.off_req)
        assert np.array_equal(tables, want.tables.numpy())
    with pytest.raises(ValueError):
        host.prompt_tables(np.array([0, 5]), np.array([4]), window, tile)
    with pytest.raises(ValueError):
        host.prompt_tables(np.array([5, 0]), np.array([4]), window, tile)
    with pytest.raises(ValueError):
        host.prompt_tables(np.array([-1, 3]), np.array([4]), window, tile)
    with pytest.raises(ValueError):
        host.prompt_tables(np.array([0, 3]), np.array([4, 4]), window, tile)
