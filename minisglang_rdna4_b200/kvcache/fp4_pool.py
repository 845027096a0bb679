"""Paged K/V pool of 4 bits.

One buffer ``[layers, pages + 1, kv_heads, page / 16, 18 * head_dim]`` of bytes: 16 tokens of a head lie together as e2m1 codes
of their keys and values and e4m3 scales of 16 channels each, in the order in which the attention kernel's lanes take them
(``csrc/kv_fp4.cuh``); 9/16 of a byte for a value. A value is ``code * scale * head`` with an fp32 factor per (layer, kv
head) for K and for V. Page ``num_pages`` is a scratch page for padded requests of a captured graph.

With ``weights=True`` an fp32 attention weight per (layer, token, kv head) lies beside it, which a caller of
``ops.paged_attention_fp4`` may let accumulate, and :meth:`evict` cuts requests down by.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .base import BaseKVCachePool

#: Factor of a head that nothing is known of: values up to 168 (2688 / 16) keep their block's scale, and blocks down to 0.006 have
#: a normal one (6 * 2^-6 / 16). Its cost: what is larger saturates, where an 8-bit pool holds 448 (a factor of 1 / 6, with
#: which blocks below 0.016 would lose bits of their scale). Heads that pass 168 need a calibrated factor.
DEFAULT_SCALE = 1.0 / 16


class FP4KVCache(BaseKVCachePool):
    fp8 = False
    fp4 = True

    def __init__(self, num_layers: int, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, dtype: torch.dtype,
                 device, weights: bool = False) -> None:
        if head_dim not in (64, 128, 256) or page_size % 16 or page_size <= 0:
            raise ValueError(f"a 4-bit K/V pool has heads of 64, 128 or 256 channels and pages of whole tiles of 16 tokens, not "
                             f"{head_dim} and {page_size}")
        if dtype not in (torch.bfloat16, torch.float16) and torch.device(device).type == "cuda":
            raise ValueError(f"a 4-bit K/V pool takes rows of bf16 or fp16, not {dtype}")
        self.num_layers, self.num_pages, self.page_size = num_layers, num_pages, page_size
        self.num_kv_heads, self.head_dim, self.compute_dtype = num_kv_heads, head_dim, dtype
        self._buf = torch.zeros((num_layers, num_pages + 1, num_kv_heads, page_size // 16, 18 * head_dim), dtype=torch.uint8,
                                device=device)
        self.k_scale, self.v_scale = (torch.full((num_layers, num_kv_heads), DEFAULT_SCALE, dtype=torch.float32, device=device)
                                      for _ in (0, 1))
        self.weights: Optional[torch.Tensor] = None
        if weights:
            self.weights = torch.zeros((num_layers, num_pages + 1, num_kv_heads, page_size), dtype=torch.float32, device=device)
        self._planes = self._buf.unbind(0)
        self._weights = self.weights.unbind(0) if weights else (None,) * num_layers

    # ---- accessors ----
    @property
    def dummy_page(self) -> int:
        return self.num_pages

    @property
    def device(self) -> torch.device:
        return self._buf.device

    @property
    def dtype(self) -> torch.dtype:
        return self._buf.dtype

    @staticmethod
    def token_bytes(num_layers: int, kv_heads: int, head_dim: int) -> int:
        return num_layers * kv_heads * head_dim * 18 // 16

    @property
    def bytes_per_token(self) -> int:
        return self.token_bytes(self.num_layers, self.num_kv_heads, self.head_dim)

    def plane(self, layer: int) -> torch.Tensor:
        """A layer's bytes ``[pages + 1, kv_heads, page / 16, 18 * head_dim]``: the ``cache`` of the operators."""
        return self._planes[layer]

    def layer_weights(self, layer: int) -> Optional[torch.Tensor]:
        return self._weights[layer]

    def k_cache(self, layer: int) -> torch.Tensor:
        raise NotImplementedError("a 4-bit pool holds keys and values together: plane(layer), or gather for 16-bit rows")

    v_cache = k_cache

    def set_scales(self, k_scale: torch.Tensor, v_scale: torch.Tensor) -> None:
        """Install the factors per (layer, head), above 0: the largest magnitude over 2688 (6 times the largest scale)."""
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if not bool(((t > 0) & torch.isfinite(t.float())).all()):      # a head's zeros would come back as NaN
                raise ValueError(f"factors of 4-bit K/V heads are positive numbers; {name} holds others")
        self.k_scale.copy_(k_scale.to(self.k_scale))
        self.v_scale.copy_(v_scale.to(self.v_scale))

    # ---- rows ----
    def store_kv(self, k: torch.Tensor, v: torch.Tensor, out_loc: torch.Tensor, layer: int) -> None:
        """Quantise rows ``[T, kv_heads, head_dim]`` into the token slots ``out_loc``; their attention weights start at zero."""
        from ..ops import store_kv_fp4

        store_kv_fp4(k, v, self._planes[layer], out_loc, self.k_scale[layer], self.v_scale[layer], self._weights[layer])

    def gather(self, layer: int, slots: torch.Tensor, which: int) -> torch.Tensor:
        """Keys (``which`` 0) or values of token slots ``[len(slots), kv_heads, head_dim]`` in 16 bits."""
        from ..ops import load_kv_fp4

        dtype = self.compute_dtype if self.compute_dtype == torch.float16 else torch.bfloat16
        return load_kv_fp4(self._planes[layer], slots.to(torch.int32), self.k_scale[layer], self.v_scale[layer], dtype)[which]

    def evict(self, block_table: torch.Tensor, seq_lens: torch.Tensor, new_table: torch.Tensor, budget: int, recent: int,
              sinks: int = 0, max_kv: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
        """Cut requests down to ``budget`` tokens in all layers at once (``ops.evict_kv_fp4``)."""
        from ..ops import evict_kv_fp4

        if self.weights is None:
            raise ValueError("the pool keeps no attention weights (weights=True)")
        return evict_kv_fp4(self._buf, self.weights, block_table, seq_lens, new_table, budget, recent, sinks, max_kv)
