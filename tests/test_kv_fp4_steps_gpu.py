"""The engine's steps over the 4-bit K/V pool on a GPU: what graphs, streams and layers share."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _config(heads=8, kv_heads=2, dim=128, positions=4096):
    from minisglang_rdna4_b200.models.config import ModelConfig

    d = dict(model_type="qwen3", hidden_size=512, num_hidden_layers=2, num_attention_heads=heads, num_key_value_heads=kv_heads,
             head_dim=dim, intermediate_size=1024, vocab_size=2048, max_position_embeddings=positions, rms_norm_eps=1e-6,
             rope_theta=10000.0, tie_word_embeddings=True, architectures=["Qwen3ForCausalLM"])
    return ModelConfig.from_hf(d)


def _prompts(lens, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 2048, (n,), generator=g).tolist() for n in lens]


def test_a_captured_graph_after_a_longer_step(monkeypatch):
    """The slots that a graph has captured hold their numbers after a step of more rows, whatever is allocated then."""
    from minisglang_rdna4_b200.layers import attention

    monkeypatch.setattr(attention, "_COUNTING", {})
    device = torch.device("cuda", torch.cuda.current_device())
    attention._counting(8, device)                                # as the warm-up ahead of a capture does
    got = torch.zeros(1000, dtype=torch.int32, device=device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got.copy_(attention._counting(1000, device))
    assert torch.equal(attention._counting(50000, device).cpu(), torch.arange(50000, dtype=torch.int32))
    junk = [torch.full((16384,), -7, dtype=torch.int32, device=device) for _ in range(64)]
    graph.replay()
    assert torch.equal(got.cpu(), torch.arange(1000, dtype=torch.int32)) and len(junk) == 64


def test_graphs_match_eager_steps_after_a_long_prompt():
    """Decode graphs, then a prompt of more rows than any step before in one go, then decode graphs again: as without graphs. (Four
    requests of one length: no padded rows.)"""
    from minisglang_rdna4_b200 import SamplingParams
    from minisglang_rdna4_b200.llm import LLM

    def run(**kw):
        llm = LLM(model_config=_config(positions=20480), use_dummy_weight=True, kv_cache_dtype="nvfp4", device="cuda", page_size=16,
                  max_running_req=4, num_page_override=2048, max_extend_tokens=20000, seed=0, **kw)
        out = []
        for i, lens in enumerate([[200] * 4, [17001], [211] * 4]):
            sp = SamplingParams(temperature=0.0, max_tokens=9 if len(lens) > 1 else 1, ignore_eos=True)
            out.append([o.token_ids for o in llm.generate(_prompts(lens, i), sp)])
        llm.shutdown()
        return out

    assert run() == run(cuda_graph_max_bs=-1)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _step(pages, hk, dim, lens, news, seed):
    """A prompt step over a pool of its own, as a call without arguments."""
    from minisglang_rdna4_b200 import ops

    g = torch.Generator("cuda").manual_seed(seed)
    cache = torch.zeros(pages, hk, 1, 18 * dim, dtype=torch.uint8, device="cuda")
    k, v = (torch.randn(pages * 16, hk, dim, generator=g, device="cuda").bfloat16() for _ in range(2))
    ops.store_kv_fp4(k, v, cache, torch.arange(pages * 16, dtype=torch.int32, device="cuda"))
    width = -(-max(lens) // 16)
    table = torch.randint(0, pages, (len(lens), width), generator=g, device="cuda", dtype=torch.int32)
    cu = _ints([0] + torch.tensor(news).cumsum(0).tolist())
    q = torch.randn(sum(news), 4 * hk, dim, generator=g, device="cuda").bfloat16()
    plan = ops.prefill_plan_fp4(q, cache, cu.cpu().numpy(), _ints(lens).cpu().numpy())
    assert plan is not None
    n = _ints(lens)
    return lambda: ops.paged_attention_fp4(q, cache, table, cu, n, 0.1, max_q=max(news), plan=plan)


def test_prompts_on_two_streams_at_once():
    """Steps of different lengths and contents, one of which needs the larger scratch, side by side: as one after the other."""
    steps = [_step(300, 2, 128, [1500, 3000], [700, 900], 0), _step(300, 2, 128, [9000, 700, 2000], [1500, 700, 100], 1)]
    want = [run() for run in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(12):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(steps[i]())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in (0, 1) for x in got[i])


@pytest.mark.parametrize("max_q", [1 << 31, 1 << 32, (1 << 32) + 1, 1 << 40])
def test_bounds_beyond_32_bits(max_q):
    """``max_q`` and ``max_kv`` may be larger than what the step has, by any amount."""
    from minisglang_rdna4_b200 import ops

    g = torch.Generator("cuda").manual_seed(0)
    cache = torch.zeros(20, 2, 1, 18 * 128, dtype=torch.uint8, device="cuda")
    k, v = (torch.randn(320, 2, 128, generator=g, device="cuda").bfloat16() for _ in range(2))
    ops.store_kv_fp4(k, v, cache, torch.arange(320, dtype=torch.int32, device="cuda"))
    table, cu, lens = torch.arange(20, dtype=torch.int32, device="cuda").view(2, 10), _ints([0, 5, 6]), _ints([150, 20])
    q = torch.randn(6, 8, 128, generator=g, device="cuda").bfloat16()
    got = [ops.paged_attention_fp4(q, cache, table, cu, lens, 0.1, max_q=n, max_kv=n) for n in (6, max_q)]
    assert torch.equal(*got) and torch.isfinite(got[0]).all()


@pytest.mark.parametrize("heads,kv_heads,dim,quant", [(8, 2, 128, None), (7, 1, 128, None), (8, 4, 64, None), (4, 2, 256, None), (8, 2, 128, "mxfp4")])
def test_served_steps_against_loops_in_64_bits(monkeypatch, heads, kv_heads, dim, quant):
    """Every layer of every step that the engine runs eagerly (chunked prompts, cached prefixes, decode steps), checked where it calls the
    operators: rows go to the slots of their positions, quantised with the layer's own factors; what attention reads is what was stored;
    its output is that of a plain form over these values."""
    import plain_kv_fp4 as plain
    from minisglang_rdna4_b200 import SamplingParams, ops
    from minisglang_rdna4_b200.kvcache import fp8_scales
    from minisglang_rdna4_b200.llm import LLM

    g = torch.Generator().manual_seed(4)
    factors = [2.0 ** torch.randint(lo, lo + 3, (2, kv_heads), generator=g) for lo in (-8, -10)]
    monkeypatch.setattr(fp8_scales, "resolve_kv_scales", lambda *a, **k: (6 * factors[0], 6 * factors[1], "test"))
    llm = LLM(model_config=_config(heads, kv_heads, dim), use_dummy_weight=True, quantization=quant, kv_cache_dtype="nvfp4", device="cuda",
              page_size=16, max_running_req=8, num_page_override=512, max_extend_tokens=256, cuda_graph_max_bs=-1, seed=0)
    pool = llm.engine.kv_cache
    layer_of = {pool.plane(i).data_ptr(): i for i in range(2)}
    held = [torch.full((2, 513 * 16, kv_heads, dim), float("nan"), dtype=torch.float64) for _ in range(2)]     # keys, values
    store, attend, slots, seen = ops.store_kv_fp4, ops.paged_attention_fp4, {}, dict(plan=0, none=0, decode=0, prefix=0)

    def checked_store(k, v, cache, out_loc, *args):
        store(k, v, cache, out_loc, *args)
        layer = layer_of[cache.data_ptr()]
        slots[layer] = out_loc.cpu().long()
        for x, y, head in zip(held, (k, v), factors):
            x[layer, slots[layer]] = plain.rounded(y, head[layer])

    def checked_attend(q, cache, table, cu_q, lens, scale, **kw):
        out = attend(q, cache, table, cu_q, lens, scale, **kw)
        layer, cu, rows = layer_of[cache.data_ptr()], cu_q.tolist(), table.cpu().long()
        for b, n in enumerate(lens.tolist()):
            at = (rows[b, :-(-n // 16), None] * 16 + torch.arange(16)).flatten()[:n]
            assert torch.equal(slots[layer][cu[b]:cu[b + 1]], at[n - (cu[b + 1] - cu[b]):])
            assert not held[0][layer, at].isnan().any()
        pages = [x[layer].view(513, 16, kv_heads, dim).transpose(1, 2) for x in held]
        read = [x.cpu() for x in plain.values(cache, factors[0][layer], factors[1][layer])]
        for x, y in zip(pages, read):
            assert torch.equal(x[~x.isnan()], y[~x.isnan()])
        assert window_free(kw)
        want, tol, _, _ = plain.attention(q, *read, rows, cu_q, lens, scale)
        if kw.get("plan") is not None:
            # probabilities of 8 bits in place of 11: 2^-8 of the sum of weighted magnitudes more, the attention over the magnitudes
            tol = tol + 2.0 ** -8 * plain.attention(q, read[0], read[1].abs(), rows, cu_q, lens, scale)[0]
        off = (out.cpu().double() - want).abs()
        assert (off <= tol).all(), float((off / tol).max())
        kind = "decode" if kw["max_q"] == 1 else "plan" if kw.get("plan") is not None else "none"
        seen[kind] += 1
        seen["prefix"] += kw["max_q"] > 1 and int((lens - (cu_q[1:] - cu_q[:-1])).max()) > 0
        return out

    def window_free(kw):
        return kw.get("window", 0) == 0 and kw.get("weights") is None

    monkeypatch.setattr(ops, "store_kv_fp4", checked_store)
    monkeypatch.setattr(ops, "paged_attention_fp4", checked_attend)
    sp = SamplingParams(temperature=0.0, max_tokens=5, ignore_eos=True)
    for _ in range(2):
        assert all(len(o.token_ids) == 5 for o in llm.generate(_prompts([1, 16, 17, 300, 5, 700]), sp))
    llm.shutdown()
    assert seen["decode"] and seen["prefix"] and (seen["plan"] if dim < 256 else seen["none"])


@pytest.mark.parametrize("hq,hk,dim", [(8, 2, 128), (7, 1, 64)])
def test_replays_with_padded_requests(hq, hk, dim):
    """A captured step of eight requests (store, attention), replayed with 8, 5, 1 and 0 real ones: the others are padding (one token of a
    spare page), as the engine pads. Real rows against the plain form; nothing but their slots and the spare page changes."""
    import plain_kv_fp4 as plain
    from minisglang_rdna4_b200 import ops

    g = torch.Generator("cuda").manual_seed(dim)
    pages, spare, width = 120, 119, 14
    cache = torch.zeros(pages, hk, 1, 18 * dim, dtype=torch.uint8, device="cuda")
    ks, vs = (2.0 ** torch.randint(-7, -4, (hk,), generator=g, device="cuda") for _ in range(2))
    fill = [torch.randn(pages * 16, hk, dim, generator=g, device="cuda").bfloat16() for _ in range(2)]
    ops.store_kv_fp4(*fill, cache, torch.arange(pages * 16, dtype=torch.int32, device="cuda"), ks, vs)
    k, v = (torch.zeros(8, hk, dim, device="cuda").bfloat16() for _ in range(2))
    q = torch.zeros(8, hq, dim, device="cuda").bfloat16()
    loc, lens, cu = torch.full((8,), spare * 16, dtype=torch.int32, device="cuda"), _ints([1] * 8), _ints(list(range(9)))
    table = torch.full((8, width), spare, dtype=torch.int32, device="cuda")

    def step():
        ops.store_kv_fp4(k, v, cache, loc, ks, vs)
        return ops.paged_attention_fp4(q, cache, table, cu, lens, 0.1, k_scale=ks, v_scale=vs, max_q=1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    order = torch.randperm(119, generator=g, device="cuda").int()
    for real in (8, 5, 1, 0, 8):
        n = torch.randint(1, 16 * width, (8,), generator=g, device="cuda").int()
        n[real:] = 1
        table.fill_(spare)
        loc.fill_(spare * 16)
        at = 0
        for b in range(real):
            need = -(-int(n[b]) // 16)
            table[b, :need] = order[at:at + need]
            at += need
            loc[b] = int(table[b, need - 1]) * 16 + (int(n[b]) - 1) % 16
        lens.copy_(n)
        for x in (k, v, q):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))
        before = plain.values(cache, ks, vs)
        graph.replay()
        after = plain.values(cache, ks, vs)
        slots = loc[:real].cpu().long()
        for x, y, rows, head in zip(before, after, (k, v), (ks, vs)):
            x, y = (z[:spare].transpose(1, 2).flatten(0, 1) for z in (x, y))
            x[slots] = plain.rounded(rows[:real], head)
            assert torch.equal(x, y)
        want, tol, _, _ = plain.attention(q, *after, table, cu, lens, 0.1)
        assert ((out.cpu().double() - want).abs() <= tol)[:real].all() and torch.isfinite(out).all()


def test_layers_that_differ_in_query_heads_serve_prompts(monkeypatch):
    """Layers of one window with 4 and with 8 query heads a key head: each takes the form for prompts with a plan of its own, and the
    output of every call is that of a plain form."""
    import plain_kv_fp4 as plain
    from minisglang_rdna4_b200 import SamplingParams, ops
    from minisglang_rdna4_b200.llm import LLM
    from minisglang_rdna4_b200.models.config import ModelConfig

    rope = {kind: {"rope_type": "default", "rope_theta": 10000.0} for kind in ("full_attention", "sliding_attention")}
    config = ModelConfig.from_hf(dict(
        model_type="laguna", architectures=["LagunaForCausalLM"], hidden_size=512, num_attention_heads=8,
        num_attention_heads_per_layer=[8, 16, 16, 8], num_key_value_heads=2, head_dim=64, intermediate_size=512,
        moe_intermediate_size=256, shared_expert_intermediate_size=256, num_experts=8, num_experts_per_tok=2, norm_topk_prob=True,
        routed_scaling_factor=1.0, first_k_dense_replace=1, vocab_size=2048, num_hidden_layers=4,
        layer_types=["full_attention", "full_attention", "sliding_attention", "sliding_attention"], sliding_window=100,
        rms_norm_eps=1e-6, rope_parameters=rope, max_position_embeddings=2048, tie_word_embeddings=False, hidden_act="silu"))
    llm = LLM(model_config=config, use_dummy_weight=True, kv_cache_dtype="nvfp4", device="cuda", page_size=16, max_running_req=4,
              num_page_override=256, max_extend_tokens=512, cuda_graph_max_bs=-1, seed=0)
    attend, seen = ops.paged_attention_fp4, set()

    def checked(q, cache, table, cu_q, lens, scale, **kw):
        out = attend(q, cache, table, cu_q, lens, scale, **kw)
        read = plain.values(cache, kw["k_scale"], kw["v_scale"])
        rows = table.cpu().long()
        want, tol, _, _ = plain.attention(q, *read, rows, cu_q, lens, scale, kw["window"])
        if kw["plan"] is not None:
            seen.add((q.shape[1], kw["window"]))
            # probabilities of 8 bits in place of 11: 2^-8 of the sum of weighted magnitudes more, the attention over the magnitudes
            tol = tol + 2.0 ** -8 * plain.attention(q, read[0], read[1].abs(), rows, cu_q, lens, scale, kw["window"])[0]
        assert ((out.cpu().double() - want).abs() <= tol).all()
        return out

    monkeypatch.setattr(ops, "paged_attention_fp4", checked)
    out = llm.generate(_prompts([300, 700, 40]), SamplingParams(temperature=0.0, max_tokens=4, ignore_eos=True))
    llm.shutdown()
    assert all(len(o.token_ids) == 4 for o in out)
    assert seen == {(8, 0), (16, 0), (16, 100), (8, 100)}


def test_a_captured_prompt_keeps_its_scratch():
    """A prompt over the 16-bit pool in a graph gathers into memory of the graph: longer prompts behind the capture neither free nor
    overwrite it."""
    import numpy as np

    from minisglang_rdna4_b200.ops import cuda as K

    g = torch.Generator("cuda").manual_seed(0)
    pool = [torch.randn(700, 2, 16, 128, generator=g, device="cuda").bfloat16() for _ in range(2)]

    def prompt(n):
        q = torch.randn(n, 8, 128, generator=torch.Generator("cuda").manual_seed(n), device="cuda").bfloat16()
        table = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda")[None]
        plan = K.PrefillPlan(np.array([0, n]), np.array([n]), q.device)
        return lambda: K.paged_attention(q, *pool, table, None, None, 0.1, max_q=n, max_kv=n, plan=plan)

    short, long = prompt(900), prompt(11000)
    want = short()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = short()
    first = long().clone()
    junk = [torch.full((1 << 22,), float("nan"), device="cuda") for _ in range(8)]
    for _ in range(2):
        graph.replay()
        assert torch.equal(got, want) and torch.equal(long(), first)
    assert len(junk) == 8
