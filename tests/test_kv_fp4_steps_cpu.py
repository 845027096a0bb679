"""What the engine's steps over the 4-bit K/V pool keep and share, on the CPU."""
import pytest
import torch


def test_slots_of_a_step_stay_where_a_captured_graph_has_them(monkeypatch):
    """A longer step neither moves nor frees what shorter ones were given."""
    from minisglang_rdna4_b200.layers import attention

    monkeypatch.setattr(attention, "_COUNTING", {})
    device = torch.device("cpu")
    first = attention._counting(8, device).data_ptr()
    for n in (16384, 16385, 40000, 10, 200000):
        assert torch.equal(attention._counting(n, device), torch.arange(n, dtype=torch.int32))
        assert attention._counting(8, device).data_ptr() == first
    middle = attention._counting(17000, device).data_ptr()
    attention._counting(300000, device)
    assert attention._counting(17000, device).data_ptr() == middle != first


def test_prompts_on_two_streams_share_no_scratch(monkeypatch):
    """The rows that a prompt gathers lie in memory of its stream: another stream's prompt neither overwrites nor frees them, and a
    graph's are its own."""
    from minisglang_rdna4_b200.ops import cuda as K

    at = [11, 0]                     # stream, capture
    monkeypatch.setattr(K, "_TC_SCRATCH", {})
    monkeypatch.setattr(K, "_stream", lambda: at[0])
    monkeypatch.setattr(K, "_capture_id", lambda stream: at[1])
    get = lambda rows: K._tc_scratch(torch.device("cpu"), torch.float16, 1, rows)  # noqa: E731
    spans = lambda hit: [(x.data_ptr(), x.data_ptr() + 2 * x.numel()) for x in hit[:2]]  # noqa: E731
    first = get(100)
    assert get(8192)[0] is first[0] and first[2] == 8192 and first[0].numel() == 8192 * 128
    at[0] = 12
    second, grown = get(100), get(9000)
    assert second[0] is not first[0] and grown[2] == 16384
    for x in spans(first):
        for y in spans(second) + spans(grown):
            assert x[1] <= y[0] or y[1] <= x[0]
    at[0] = 11
    assert get(1)[0] is first[0]
    at[1] = 5
    captured = get(1)
    assert captured[0] is not first[0] and not captured[0].any()
    at[1] = 0
    assert get(1)[0] is first[0]
    for at[0] in range(20, 40):      # a stream in use keeps its own, the others do not pile up
        get(1)
        at[0], keep = 11, at[0]
        assert get(1)[0] is first[0]
        at[0] = keep
    assert len(K._TC_SCRATCH) == K.TC_SCRATCH_SETS


def test_new_pages_outside_the_pool_are_written_nowhere():
    from minisglang_rdna4_b200 import ops

    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    g = torch.Generator().manual_seed(0)
    cache = torch.randint(0, 256, (9, 2, 1, 18 * 64), generator=g, dtype=torch.uint8)
    weights = torch.rand(9, 2, 16, generator=g)
    table, lens = ints([[1, 2, 3], [4, 4, 4]]), ints([48, 7])
    good, good_w = cache.clone(), weights.clone()
    stay, _ = ops.evict_kv_fp4(good, good_w, table, lens, ints([[5, 6], [7, 7]]), 20, 4)
    want, want_w = cache.clone(), weights.clone()
    want[6], want_w[6] = good[6], good_w[6]
    kept, now = ops.evict_kv_fp4(cache, weights, table, lens, ints([[-1, 6], [9, 7]]), 20, 4)
    assert torch.equal(kept, stay) and now.tolist() == [20, 7]
    assert torch.equal(cache, want) and torch.equal(weights, want_w)


def _nan_pool(dim=64, hk=2, pages=4):
    from minisglang_rdna4_b200 import ops

    g = torch.Generator().manual_seed(1)
    cache = torch.zeros(pages, hk, 1, 18 * dim, dtype=torch.uint8)
    k, v = (torch.randn(pages * 16, hk, dim, generator=g).bfloat16() for _ in range(2))
    return cache, k, v, lambda: ops.store_kv_fp4(k, v, cache, torch.arange(pages * 16, dtype=torch.int32))


def test_slots_outside_the_pool_are_zeros_beside_a_nan():
    from minisglang_rdna4_b200 import ops

    cache, k, v, store = _nan_pool()
    k[0, 0, 3] = v[0, 1, 40] = float("nan")
    store()
    slots = torch.tensor([-1, 0, 64, -(1 << 31), 1 << 30], dtype=torch.int32)
    for x in (ops.load_kv_fp4(cache, slots), [y[0] for y in ops.load_kv_fp4(torch.stack([cache, cache]), slots)]):
        for y in x:
            assert (y[[0, 2, 3, 4]] == 0).all() and int(y[1].isnan().sum()) == 16


def _with_and_without_a_nan(where, window):
    """A request of 50 tokens with 30 rows over a pool with and without a NaN in channels 16 .. 31 of key head 1 of token 35's key or
    value: ``(outputs, weights, rows that see it)``."""
    from minisglang_rdna4_b200 import ops

    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    got = []
    for value in (0.0, float("nan")):
        cache, k, v, store = _nan_pool()
        (k if where == "key" else v)[35, 1, 16:32] = value
        store()
        q = torch.randn(30, 4, 64, generator=torch.Generator().manual_seed(2)).half()
        weights = torch.zeros(4, 2, 16)
        out = ops.paged_attention_fp4(q, cache, ints([[0, 1, 2, 3]]), ints([0, 30]), ints([50]), 0.1, window=window, weights=weights)
        got.append((out, weights.transpose(0, 1).flatten(1)))
    pos = torch.arange(20, 50)
    return got, (pos >= 35) & ((pos < 35 + window) if window else pos >= 0)


@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("where", ["key", "value"])
def test_a_nan_reaches_the_rows_that_see_it_alone(where, window):
    ((clean, clean_w), (out, weights)), sees = _with_and_without_a_nan(where, window)
    bad = torch.zeros(30, 4, 64, dtype=torch.bool)
    bad[sees, 2:, slice(16, 32) if where == "value" else slice(64)] = True
    assert torch.equal(out.isnan(), bad) and torch.equal(out[~bad], clean[~bad])
    given = torch.zeros(2, 64, dtype=torch.bool)
    if where == "key":                   # the weights that its rows give are none either
        first = 35 - window + 1 if window else 0
        given[1, first:35 + window if window else 50] = True
        given[1, 50:] = False
    assert torch.equal(weights.isnan(), given) and torch.equal(weights[~given], clean_w[~given])


def test_layers_that_differ_in_query_heads_have_plans_of_their_own(monkeypatch):
    from minisglang_rdna4_b200.attention import paged

    made = []
    monkeypatch.setattr(paged.ops, "prefill_plan_fp4", lambda q, cache, cu, n, window: made.append((window, q.shape[1])) or made[-1])
    cache = torch.zeros(1, 2, 1, 18 * 64, dtype=torch.uint8)
    plans = paged.Fp4Plans(None, None)
    for _ in range(2):                   # layers of a model with 8 and 12 query heads, with and without a window
        for window, heads in ((0, 8), (0, 12), (64, 12), (64, 8)):
            assert plans.of(torch.zeros(5, heads, 64), cache, window) == (window, heads)
    assert len(made) == 4


def _engine(**model):
    """As much of an engine as its boot has when the pool is sized, on a GPU of 64 GiB."""
    from types import SimpleNamespace as Some

    mc = Some(**{**dict(latent_layers=[], layered=False, has_fp32_kernels=False, is_mla=False, canvas_length=0, vision=None,
                        image_bidirectional=True, swa_layers=[], global_head_dim=0, num_kv_layers=3, num_kv_heads=2, head_dim=128,
                        model_type="some", is_recurrent=False, intermediate_size=512, q_size=1024, kv_size=256, hidden_size=512,
                        attn_geometry=lambda i: (2, 128)), **model})
    config = Some(spec_algorithm="none", page_size=16, num_page_override=None, tp_size=1, memory_ratio=0.9, max_running_req=4,
                  max_extend_tokens=1024)
    return Some(config=config, model_config=mc, kv_fp8=False, kv_fp4=True, dtype=torch.bfloat16, kv_layers=3, kv_heads_local=2,
                page_size=16, _main_geometry=None, mla_latent=False, _head_geometry=None, device=torch.device("cuda"), _swa_layers=0,
                cpu_group=None)


def test_a_pool_whose_layers_all_have_another_geometry_is_refused():
    from minisglang_rdna4_b200.engine.engine import Engine

    Engine._refuse_fp4_pool(_engine())
    Engine._refuse_fp4_pool(_engine(global_head_dim=128))
    for heads, width in ((2, 256), (1, 128)):
        with pytest.raises(ValueError, match=f"nvfp4 does not go with layers of {heads} key heads of {width} channels"):
            Engine._refuse_fp4_pool(_engine(global_head_dim=width, attn_geometry=lambda i: (heads, width)))


def test_pages_are_counted_in_4_bits_whatever_names_the_geometry(monkeypatch):
    from minisglang_rdna4_b200.engine.engine import Engine

    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (60 << 30, 64 << 30))
    plain, named, wide = _engine(), _engine(global_head_dim=128), _engine(global_head_dim=128)
    named._main_geometry = wide._main_geometry = [(2, 128)] * 3
    wide.kv_fp4 = False
    pages = [Engine._determine_num_pages(e) for e in (plain, named, wide)]
    assert pages[0] == pages[1] and 3.5 < pages[0] / pages[2] < 3.6          # 16 bits against 4.5


def test_factors_that_are_no_positive_numbers_are_refused():
    from minisglang_rdna4_b200.kvcache import FP4KVCache

    pool = FP4KVCache(2, 4, 16, 2, 64, torch.bfloat16, "cpu")
    good = torch.full((2, 2), 0.25)
    for value in (0.0, -1.0, float("nan"), float("inf")):
        bad = good.clone()
        bad[1, 0] = value
        for pair in ((bad, good), (good, bad)):
            with pytest.raises(ValueError, match="positive"):
                pool.set_scales(*pair)
    pool.set_scales(good, 2 * good)
    assert torch.equal(pool.k_scale, good) and torch.equal(pool.v_scale, 2 * good)


def test_a_wait_that_ran_out_over_the_4_bit_pool_is_a_status_of_attention(monkeypatch):
    from types import SimpleNamespace

    from minisglang_rdna4_b200.ops import _lib, cuda

    state = dict.fromkeys(("msgl_attn_status", "msgl_attn_tc_status", "msgl_talk_status", "msgl_attention_fp4_status"), 0)

    def reader(name):
        def read(reset):
            got = state[name]
            state[name] = 0 if reset else got
            return got
        return read

    monkeypatch.setattr(cuda, "lib", lambda: SimpleNamespace(**{name: reader(name) for name in state}))
    monkeypatch.setattr(_lib, "bind", lambda *args: None)
    assert cuda.attn_status() == 0
    for name in state:
        state[name] = 401
        assert cuda.attn_status(reset=False) == 401 and cuda.attn_status() == 401 and cuda.attn_status() == 0, name
    state.update(dict.fromkeys(state, 5))
    assert cuda.attn_status() == 5 and cuda.attn_status() == 0      # all are reset by one call


def test_eviction_refuses_layers_that_overlap():
    from minisglang_rdna4_b200 import ops

    ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    cache, weights = torch.zeros(2, 4, 1, 1, 18 * 64, dtype=torch.uint8), torch.zeros(2, 4, 1, 16)
    half = torch.zeros(6, 1, 1, 18 * 64, dtype=torch.uint8).as_strided((2, 4, 1, 1, 18 * 64), (2 * 18 * 64, 18 * 64, 18 * 64, 18 * 64, 1))
    args = (ints([[0, 1]]), ints([20]), ints([[2]]), 8, 2)
    for c, w in ((cache[:1].expand(2, -1, -1, -1, -1), weights), (half, weights), (cache, weights[:1].expand(2, -1, -1, -1))):
        with pytest.raises(ValueError, match="overlap"):
            ops.evict_kv_fp4(c, w, *args)
    assert ops.evict_kv_fp4(cache, weights, *args)[1].tolist() == [8]
    assert ops.evict_kv_fp4(cache[:1].expand(1, -1, -1, -1, -1), weights[:1], *args)[1].tolist() == [8]
