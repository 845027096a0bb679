"""Python side of the paged K/V pool of 4 bits: checks of arguments, and the kernels of ``csrc/kv_fp4.cu`` and
``csrc/attention_fp4.cu``. The checks hold on the CPU path too (``ops.ref_fp4``)."""
from __future__ import annotations

import ctypes
from typing import Dict, Optional, Tuple

import numpy as np
import torch

from . import _lib
from . import cuda as K
from ._lib import c_f, c_i, c_ll, c_p, check, lib
from .host import prompt_tables

_lib.bind("msgl_store_fp4", c_i, [c_p, c_p, c_ll, c_ll] + [c_p] * 5 + [c_i] * 4 + [c_ll, c_i, c_p])
_lib.bind("msgl_load_fp4", c_i, [c_p, c_ll, c_i] + [c_p] * 5 + [c_i] * 4 + [c_ll, c_i, c_p])
_lib.bind("msgl_evict_fp4", c_i, [c_p, c_ll, c_p, c_ll, c_i, c_p, c_i, c_p, c_i, c_p, c_p, c_p] + [c_i] * 9 + [c_p])
_lib.bind("msgl_attention_fp4", c_i, [c_p] * 4 + [c_ll, c_i] + [c_p] * 7 + [c_i] * 9 + [c_f, c_i, c_p])
_lib.bind("msgl_attention_fp4_workspace", c_ll, [c_i] * 6 + [c_p])
_lib.bind("msgl_prompt_fp4", c_i, [c_p] * 4 + [c_ll, c_i, c_p, c_p, c_ll, c_i, c_p, c_i] + [c_p] * 4 + [c_i] * 8 + [c_f, c_i, c_p])
_lib.bind("msgl_attention_fp4_status", c_i, [c_i])

TILE = 16                       # tokens of a tile
WIDTHS = (64, 128, 256)
_ROWS = (torch.bfloat16, torch.float16)


def tile_bytes(dim: int) -> int:
    """Bytes of 16 tokens of one head: codes of keys and values (8 D each) and their scales (D each)."""
    return 18 * dim


_SHAPES: Dict[torch.Size, Tuple[int, int, int, int, int]] = {}


def _shape_of(shape: torch.Size) -> Tuple[int, int, int, int, int]:
    if len(shape) not in (4, 5):
        raise ValueError("a 4-bit K/V pool is uint8 [pages, heads, page / 16, 18 D] (layers in front where they are taken)")
    pages, hk, tiles, width = shape[-4:]
    dim = width // 18
    if dim not in WIDTHS or width % 18 or tiles < 1 or hk < 1 or pages < 1:
        raise ValueError(f"a 4-bit K/V pool has heads of 64, 128 or 256 channels (tiles of 18 D bytes), not {tuple(shape)}")
    if len(_SHAPES) > 256:
        _SHAPES.clear()
    _SHAPES[shape] = hit = (shape[0] if len(shape) == 5 else 1, pages, hk, tiles * TILE, dim)
    return hit


def pool_shape(cache: torch.Tensor, layered: bool = False) -> Tuple[int, int, int, int, int]:
    """``(layers, pages, heads, page size, D)`` of ``[pages, heads, page / 16, 18 D]`` bytes (``layered``: with or without
    layers in front)."""
    shape = cache.shape
    hit = _SHAPES.get(shape) or _shape_of(shape)
    if cache.dtype is not torch.uint8 or (len(shape) == 5 and not layered):
        raise ValueError("a 4-bit K/V pool is uint8 [pages, heads, page / 16, 18 D]" + (", layers in front" if layered else ""))
    if cache.data_ptr() % 16 or not cache.is_contiguous():
        if cache.data_ptr() % 16 or len(shape) == 4 or cache.stride(0) % 16 or not cache[0].is_contiguous():
            raise ValueError("the layers of a 4-bit K/V pool are contiguous, on 16-byte boundaries")
    return hit


def check_here(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    """All on one device, on a GPU the current one: the kernels go to its current stream."""
    here = first.get_device()
    for t in others:
        if t is not None and t.get_device() != here:
            raise ValueError(f"tensors on {first.device} and {t.device}")
    if here >= 0 and here != torch._C._cuda_getDevice():
        raise ValueError(f"tensors on {first.device}, but the current device is cuda:{torch._C._cuda_getDevice()}")


def check_ints(name: str, t: torch.Tensor, rows: Optional[int] = None, dims: int = 1) -> None:
    if t.dtype is not torch.int32 or t.dim() != dims or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name} is int32 with {dims} dimension(s) and {'any number of' if rows is None else rows} rows, not {t.dtype} "
                         f"{tuple(t.shape)}")


def check_heads(k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor], hk: int) -> None:
    for t in (k_scale, v_scale):
        if t is not None and (t.dtype is not torch.float32 or t.dim() != 1 or t.shape[0] != hk or not t.is_contiguous()):
            raise ValueError(f"k_scale and v_scale are fp32 [{hk}], one factor per key / value head")


def check_weights(weights: torch.Tensor, cache: torch.Tensor, pages: int, hk: int, page: int) -> None:
    want = (cache.shape[0],) * (cache.dim() == 5) + (pages, hk, page)
    if (weights.dtype is not torch.float32 or weights.shape != want
            or not (weights.is_contiguous() or (weights.dim() == 4 and weights[0].is_contiguous()))):
        raise ValueError(f"attention weights are contiguous fp32 {want}, not {weights.dtype} {tuple(weights.shape)}")


def check_apart(name: str, t: torch.Tensor, dims: int) -> None:
    """Layers in front of ``dims`` dimensions lie in memory of their own."""
    if t.dim() > dims and t.shape[0] > 1 and t.stride(0) < t.numel() // t.shape[0]:
        raise ValueError(f"the layers of {name} overlap")


def check_rows(k: torch.Tensor, v: torch.Tensor, rows: int, hk: int, dim: int) -> None:
    if k.dtype is not v.dtype or (k.dtype not in _ROWS and (k.is_cuda or k.dtype is not torch.float32)):
        raise TypeError(f"rows of bf16 or fp16, keys and values alike, not {k.dtype} and {v.dtype}")
    for x in (k, v):
        shape = x.shape
        if len(shape) not in (2, 3) or shape[0] != rows or (shape[1] != hk * dim if len(shape) == 2 else shape[1:] != (hk, dim)):
            raise ValueError(f"keys and values are [{rows}, {hk}, {dim}], not {tuple(shape)}")


def _rows(x: torch.Tensor, hk: int, dim: int) -> Tuple[torch.Tensor, int]:
    """The rows as the kernel can read them and how far they lie apart: where they are if they start on 16 bytes, else a
    copy."""
    ld, inner = x.stride(0), x.stride()[1:]
    if (inner == (dim, 1) or inner == (1,)) and ld % 8 == 0 and x.data_ptr() % 16 == 0:
        return x, ld
    x = x.reshape(x.shape[0], hk * dim)
    return (x.clone() if x.is_contiguous() else x.contiguous()), hk * dim


def _packed(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def store_kv_fp4(k, v, cache, out_loc, k_scale, v_scale, weights, shape):
    _, pages, hk, page, dim = shape
    (k, ldk), (v, ldv), out_loc = _rows(k, hk, dim), _rows(v, hk, dim), _packed(out_loc)
    check(lib().msgl_store_fp4(
        k.data_ptr(), v.data_ptr(), ldk, ldv, cache.data_ptr(), out_loc.data_ptr(), K._p(k_scale), K._p(v_scale), K._p(weights),
        out_loc.shape[0], hk, dim, page, pages, K._dt(k), K._stream()), "store_kv_fp4")
    K._count("store_kv_fp4", "store_fp4_kernel")


def load_kv_fp4(cache, slots, k_scale, v_scale, dtype, shape):
    layers, pages, hk, page, dim = shape
    slots, n, layered = _packed(slots), slots.shape[0], cache.dim() == 5
    both = torch.empty((2, layers, n, hk, dim) if layered else (2, n, hk, dim), dtype=dtype, device=cache.device)
    k, v = both.unbind(0)
    check(lib().msgl_load_fp4(cache.data_ptr(), cache.stride(0) if layered else 0, layers, slots.data_ptr(), K._p(k_scale),
                              K._p(v_scale), k.data_ptr(), v.data_ptr(), n, hk, dim, page, pages, K._DT[dtype], K._stream()),
          "load_kv_fp4")
    K._count("load_kv_fp4", "load_fp4_kernel")
    return k, v


def evict_kv_fp4(cache, weights, block_table, seq_lens, new_table, budget, recent, sinks, max_kv, shape):
    layers, pages, hk, page, dim = shape
    lead = (layers,) if cache.dim() == 5 else ()
    b = seq_lens.numel()
    block_table, seq_lens, new_table = _packed(block_table), _packed(seq_lens), _packed(new_table)
    kept = torch.empty(*lead, b, hk, budget, dtype=torch.int32, device=cache.device)
    lens = torch.empty(b, dtype=torch.int32, device=cache.device)
    check(lib().msgl_evict_fp4(
        cache.data_ptr(), cache.stride(0) if lead else 0, weights.data_ptr(), weights.stride(0) if lead else 0, layers,
        block_table.data_ptr(), block_table.shape[1], new_table.data_ptr(), new_table.shape[1], seq_lens.data_ptr(),
        kept.data_ptr(), lens.data_ptr(), b, hk, dim, page, pages, budget, recent, sinks, min(max_kv, block_table.shape[1] * page),
        K._stream()), "evict_kv_fp4")
    K._count("evict_kv_fp4", "evict_select_kernel + evict_move_kernel", 2)
    return kept, lens


_NEED: Dict[Tuple, Tuple[int, int]] = {}


def attention_fp4_workspace(rows: int, heads: int, kv_heads: int, dim: int, max_q: int, weighed: bool) -> Tuple[int, int]:
    """fp32 words that a call of ``paged_attention_fp4`` takes as its workspace, and its counters."""
    key = (rows if weighed else 0, heads, kv_heads, dim, max_q, weighed, torch._C._cuda_getDevice())
    hit = _NEED.get(key)
    if hit is None:
        if len(_NEED) > 4096:
            _NEED.clear()
        workers = ctypes.c_int()
        words = int(lib().msgl_attention_fp4_workspace(rows, heads, kv_heads, dim, max_q, int(weighed), ctypes.addressof(workers)))
        _NEED[key] = hit = (words, workers.value)
    return hit


def paged_attention_fp4(q, cache, block_table, cu_q, seq_lens, scale, k_scale, v_scale, window, max_q, weights, plan, workspace, shape):
    _, pages, hk, page, dim = shape
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    out = torch.empty_like(q)
    if block_table.stride(1) != 1:
        block_table = block_table.contiguous()
    if plan is not None:
        return _prefill(q, cache, out, block_table, plan, scale, k_scale, v_scale, window, shape)
    cu_q, seq_lens = _packed(cu_q), _packed(seq_lens)
    t, hq, _ = q.shape
    b = seq_lens.shape[0]
    if max_q == 0 and t and b:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("max_q of 0 is read from the device, outside of a graph's capture")
        max_q = int((cu_q[1:] - cu_q[:-1]).max())
    max_q = min(max_q, t)                # however large a bound the caller has
    if max_q == 0:
        return out
    need, workers = attention_fp4_workspace(t, hq, hk, dim, max_q, weights is not None)
    if workspace is None or workspace.numel() < need or workspace.data_ptr() % 16:
        workspace = torch.empty(need, dtype=torch.float32, device=q.device)
    check(lib().msgl_attention_fp4(
        q.data_ptr(), out.data_ptr(), cache.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
        cu_q.data_ptr(), seq_lens.data_ptr(), K._p(k_scale), K._p(v_scale), K._p(weights), workspace.data_ptr(),
        K._stream_counters(q.device, workers).data_ptr(), t, b, hq, hk, dim, page, pages, max_q, window, scale, K._dt(q),
        K._stream()), "paged_attention_fp4")
    K._count("paged_attention_fp4", "fp4_attention_kernel", 1 + (weights is not None))
    return out


def attention_fp4_status(reset=True) -> int:
    """Nonzero: a wait in the kernel ran out."""
    return int(lib().msgl_attention_fp4_status(int(reset)))


class PromptPlan(K.PrefillPlan):
    """The tables, and what they are for: window, heads, rows, tokens of the longest request."""

    __slots__ = ("window", "group", "dim", "rows", "longest")

    def __init__(self, cu_q, seq_lens, device, window, tile, tables) -> None:
        """``tables``: ``host.prompt_tables``; ``None``: they are built here."""
        if tables is None:
            super().__init__(cu_q, seq_lens, device, window, tile=tile)
            return
        host, self.t_pad, self.n_items = tables[:3]
        self.n_req, self.tile = seq_lens.size, tile
        self.off_blk = 8 * self.n_items
        self.off_req = self.off_blk + self.t_pad // 128
        self.tables = K._upload_tables(host, device)


def prefill_plan_fp4(q, cache, cu_q, seq_lens, window):
    """The tcgen05 form of prompts: heads of 64 or 128 channels."""
    hk, dim = cache.shape[1], cache.shape[3] // 18
    group = q.shape[1] // hk
    if dim == 256:
        return None
    cu_q, seq_lens = (np.ascontiguousarray(x, dtype=np.int64) for x in (cu_q, seq_lens))
    b, tile = seq_lens.size, 256 if group % 2 else 128
    if b == 0:
        return None
    if seq_lens.ndim != 1 or cu_q.shape != (b + 1,):
        raise ValueError(f"cu_q and seq_lens are the lengths of one step, not {cu_q.shape} and {seq_lens.shape}")
    try:
        tables = prompt_tables(cu_q, seq_lens, window, tile)
    except ValueError:                                        # rows in front of their text
        return None
    if tables is None:
        cu_q, seq_lens = np.minimum(cu_q, 1 << 30), np.minimum(seq_lens, 1 << 30)
        if (np.diff(cu_q) > seq_lens).any():
            return None
    rows, reach = (tables[3], tables[1]) if tables else (int(cu_q[b]), K.PrefillPlan.rows_in_reach(cu_q, seq_lens, window))
    if not K.tc_prefill_pays(rows, reach):
        return None
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("a prefill plan is made of lengths on the host, outside of a graph's capture")
    plan = PromptPlan(cu_q, seq_lens, q.device, window, tile, tables)
    plan.window, plan.group, plan.dim, plan.rows, plan.longest = window, group, dim, rows, tables[4] if tables else int(seq_lens.max())
    return plan


def _prefill(q, cache, out, block_table, plan, scale, k_scale, v_scale, window, shape):
    _, pages, hk, page, dim = shape
    if not isinstance(plan, PromptPlan) or (plan.window, plan.group, plan.dim) != (window, q.shape[1] // hk, dim):
        raise ValueError("the prefill plan was made for another window or other heads")
    if (plan.tables.device != q.device or plan.rows > q.shape[0] or plan.n_req > block_table.shape[0]
            or plan.longest > block_table.shape[1] * page):
        raise ValueError(f"the prefill plan was made for {plan.n_req} requests of up to {plan.longest} tokens, {plan.rows} rows, on "
                         f"{plan.tables.device}")
    if scale <= 0:
        raise ValueError("the form for prompts takes a scale above 0")
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError("the form for prompts, whose rows in 16 bits lie in memory that a stream's layers and steps share, is not captured in a graph")
    kc, vt, cap = K._tc_scratch(q.device, q.dtype, hk, plan.t_pad)
    base = plan.tables.data_ptr()
    check(lib().msgl_prompt_fp4(
        q.data_ptr(), out.data_ptr(), cache.data_ptr(), block_table.data_ptr(), block_table.stride(0), block_table.shape[1], kc.data_ptr(),
        vt.data_ptr(), cap, plan.t_pad, base, plan.n_items, base + 4 * plan.off_blk, base + 4 * plan.off_req, K._p(k_scale), K._p(v_scale),
        q.shape[0], q.shape[1], hk, dim, page, pages, int(window), int(plan.tile == 256), float(scale), K._dt(q), K._stream()),
        "paged_attention_fp4 (prompts)")
    K._count("paged_attention_fp4 (prompts)", "fp4_gather_kernel + attn_prefill_tc_kernel + fp4_prompt_nans_kernel", 3)
    return out
