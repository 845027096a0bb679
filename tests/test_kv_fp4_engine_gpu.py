"""The engine over a K/V pool of 4 bits: prompts, chunks, a cached prefix, decode steps in graphs and without."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu


def _config(layers=2, heads=8, kv_heads=2, dim=128):
    from minisglang_rdna4_b200.models.config import ModelConfig

    d = dict(model_type="qwen3", hidden_size=512, num_hidden_layers=layers, num_attention_heads=heads, num_key_value_heads=kv_heads,
             head_dim=dim, intermediate_size=1024, vocab_size=2048, max_position_embeddings=4096, rms_norm_eps=1e-6, rope_theta=10000.0,
             tie_word_embeddings=True, architectures=["Qwen3ForCausalLM"])
    return ModelConfig.from_hf(d)


def _tokens(prompts, runs=1, max_tokens=9, **kw):
    from minisglang_rdna4_b200 import SamplingParams
    from minisglang_rdna4_b200.llm import LLM
    from minisglang_rdna4_b200.ops import cuda as K
    from minisglang_rdna4_b200.ops import kv_fp4

    llm = LLM(**{**dict(model_config=_config(), use_dummy_weight=True, kv_cache_dtype="nvfp4", device="cuda", page_size=16,
                        max_running_req=8, num_page_override=512, seed=0), **kw})
    sp = SamplingParams(temperature=0.0, max_tokens=max_tokens, ignore_eos=True)
    out = [[o.token_ids for o in llm.generate(prompts, sp)] for _ in range(runs)]
    assert K.attn_status() == 0 and K.gemm_status() == 0 and kv_fp4.attention_fp4_status() == 0
    assert "fp4_attention_kernel" in K.LEDGER.get("paged_attention_fp4", "")
    llm.cache.check_integrity()
    llm.shutdown()
    return out


def _prompts(lens, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 2048, (n,), generator=g).tolist() for n in lens]


@pytest.mark.parametrize("quant", [None, "mxfp4"])
def test_graphs_match_eager_steps(quant):
    """Four requests of one length and one bucket of a graph: no padded rows, so the same sums in the same order."""
    prompts = _prompts([200] * 4)
    graph = _tokens(prompts, quantization=quant)
    eager = _tokens(prompts, quantization=quant, cuda_graph_max_bs=-1)
    assert graph == eager and all(len(t) == 9 for t in graph[0])


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (7, 1, 128), (8, 4, 64), (4, 2, 256)])
def test_lengths_and_shapes_of_all_kinds(heads, kv_heads, dim):
    """Padded graphs, chunked prompts and cached prefixes run, and requests give as many tokens as asked for."""
    out = _tokens(_prompts([1, 16, 17, 300, 5, 700]), runs=2, model_config=_config(heads=heads, kv_heads=kv_heads, dim=dim),
                  max_extend_tokens=256)
    assert all(len(t) == 9 for run in out for t in run)


def test_fills_what_memory_a_pool_of_8_bits_leaves():
    """A token takes 9 / 16 of the bytes that it takes in 8 bits, so more pages fit."""
    from minisglang_rdna4_b200.llm import LLM

    pages = {}
    for kv in ("fp8", "nvfp4"):
        llm = LLM(model_config=_config(), use_dummy_weight=True, kv_cache_dtype=kv, device="cuda", page_size=16, max_running_req=8,
                  seed=0, memory_ratio=0.06)
        pages[kv] = llm.engine.num_pages
        llm.shutdown()
        del llm
        gc.collect()
        torch.cuda.empty_cache()
    assert 1.7 < pages["nvfp4"] / pages["fp8"] < 1.85
