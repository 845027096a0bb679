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
