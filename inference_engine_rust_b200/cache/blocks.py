"""Keys and values of a layer group in 8 bits, and the eviction of what attention has weighed least.

A block is 16 consecutive positions of one key/value head; its keys share one fp32 scale, its values another, and a number is kept
as a level (int8, or e4m3) that stands for level * scale.  A sequence's newest positions, fewer than 16, stand in `tail` in the run's
own type until their block is full: then it is turned into levels, once, from the numbers as they came.  A page of 64 positions of
a head takes 2 x 64 x (D + 1/4) bytes, 0.502 of bfloat16's.

With an `EvictionPolicy` each block also has the attention weight that it has received from the one-token steps (summed over the query
heads of its key head), and a sequence that has grown past the policy's bound goes back to `keep` positions: of its finished
blocks every layer and head keeps the last `recent` positions' and those with the largest weight.  Keys carry their rotation, so
where a block lies does not matter; the positions a sequence has lost are counted in `shift`, by which later rotations turn further.

Reference: the whole-sequence cache of src/layers/attention.rs:16-74 keeps every position in fp32; neither the levels nor the
eviction has a counterpart there.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

BLOCK_TOKENS = 16

CACHE_DTYPES = {"int8": torch.int8, "float8_e4m3": torch.float8_e4m3fn, "fp8": torch.float8_e4m3fn}


def parse_cache_dtype(name) -> Optional[torch.dtype]:
    """None: the run's own type.  "int8", "float8_e4m3" (or "fp8"): 8-bit levels with a scale per 16 positions and head."""
    if name is None:
        return None
    if isinstance(name, torch.dtype):
        if name in (torch.int8, torch.float8_e4m3fn):
            return name
    elif str(name) in CACHE_DTYPES:
        return CACHE_DTYPES[str(name)]
    raise ValueError(f"cache_dtype must be one of {sorted(CACHE_DTYPES)} or None, got {name!r}")


@dataclass(frozen=True)
class EvictionPolicy:
    """keep     positions (of finished blocks) that a sequence goes back to; a multiple of 16
    recent   how many of them are its newest, whatever their weight (a multiple of 16; default: a quarter of `keep`)
    every    one-token steps between two evictions of a sequence, which are also what the weights are gathered from at least
    """
    keep: int
    recent: Optional[int] = None
    every: int = 64

    def __post_init__(self):
        if self.recent is None:
            object.__setattr__(self, "recent", self.keep // 4 // BLOCK_TOKENS * BLOCK_TOKENS if isinstance(self.keep, int) else 0)
        for name in ("keep", "recent", "every"):
            v = getattr(self, name)
            if isinstance(v, bool) or not isinstance(v, int):
                raise ValueError(f"eviction: {name} must be a whole number, got {v!r}")
        if self.keep <= 0 or self.keep % BLOCK_TOKENS:
            raise ValueError(f"eviction: keep must be a positive multiple of {BLOCK_TOKENS}, got {self.keep}")
        if self.recent % BLOCK_TOKENS or not 0 <= self.recent <= self.keep:
            raise ValueError(f"eviction: recent must be a multiple of {BLOCK_TOKENS} between 0 and keep ({self.keep}), got {self.recent}")
        if self.every <= 0:
            raise ValueError(f"eviction: every must be positive, got {self.every}")

    def due(self, held: int, steps: int) -> bool:
        """Does a sequence that holds `held` positions go back now, `steps` one-token steps after it last did (or began)?"""
        return steps >= self.every and held >= self.keep + self.every

    def most_held(self, prompt: int) -> int:
        """The most positions that a sequence with a prompt of this length comes to hold."""
        return max(prompt, self.keep + BLOCK_TOKENS - 1) + self.every


class BlockStore:
    """The pools of a key/value group in 8 bits: what `KVGroup` keeps when the cache is made with `levels`."""

    def __init__(self, layers: int, n_pages: int, n_slots: int, kv_heads: int, head_dim: int, page_tokens: int, levels: torch.dtype,
                 dtype: torch.dtype, device, weights: bool):
        if page_tokens % BLOCK_TOKENS:
            raise ValueError(f"an 8-bit cache needs pages of a multiple of {BLOCK_TOKENS} positions, got {page_tokens}")
        shape = (layers, n_pages, kv_heads, page_tokens, head_dim)
        scales = (layers, n_pages, kv_heads, page_tokens // BLOCK_TOKENS)
        self.levels, self.page_tokens = levels, page_tokens
        self.k, self.v = (torch.empty(shape, dtype=levels, device=device) for _ in range(2))
        self.k_scale, self.v_scale = (torch.empty(scales, dtype=torch.float32, device=device) for _ in range(2))
        self.weight = torch.zeros(scales, dtype=torch.float32, device=device) if weights else None
        tail = (layers, n_slots, kv_heads, BLOCK_TOKENS, head_dim)
        self.tail_k, self.tail_v = (torch.empty(tail, dtype=dtype, device=device) for _ in range(2))
        self.shift = torch.zeros(n_slots, dtype=torch.int32, device=device) if weights else None

    def poison(self, pages=None) -> None:
        """NaN scales (of some pages, or of everything and the tails): whoever reads what was never written sees it."""
        at = slice(None) if pages is None else pages
        self.k_scale[:, at] = float("nan")
        self.v_scale[:, at] = float("nan")
        if pages is None:
            self.tail_k.fill_(float("nan"))
            self.tail_v.fill_(float("nan"))

    def view(self, layer: int, table: torch.Tensor, window: int, ring_pages: int):
        """What the block kernels receive for a layer."""
        from ..csrc import bindings as B
        return B.block_view(self.k[layer], self.v[layer], self.k_scale[layer], self.v_scale[layer], self.tail_k[layer], self.tail_v[layer], table,
                            window=window, ring_pages=ring_pages, weight=None if self.weight is None else self.weight[layer], shift=self.shift)

    def evict(self, table: torch.Tensor, slots: Sequence[int], held: Sequence[int], new_pages: np.ndarray, keep: int, recent: int, err) -> torch.Tensor:
        """Launch the eviction of these sequences (all layers); returns the numbers of the kept blocks [layers, sequences, kv_heads, keep]
        on the device.  `keep`, `recent` in blocks."""
        from ..csrc import bindings as B
        device = self.k.device
        # one copy for all the numbers, out of page-locked memory: the host does not wait for the device
        n, w = new_pages.shape
        host = torch.empty(n * (2 + w), dtype=torch.int32, pin_memory=True)
        host[:n] = torch.tensor(list(slots), dtype=torch.int32)
        host[n:2 * n] = torch.tensor(list(held), dtype=torch.int32)
        host[2 * n:] = torch.from_numpy(np.ascontiguousarray(new_pages, dtype=np.int32).reshape(-1))
        dev = host.to(device, non_blocking=True)
        kept = torch.empty((self.k.shape[0], n, self.k.shape[2], keep), dtype=torch.int32, device=device)
        B.block_evict(self.k, self.v, self.k_scale, self.v_scale, self.weight, table, dev[n:2 * n], dev[2 * n:].view(n, w), keep, recent, kept, err,
                      B.stream_ptr(), slots=dev[:n], shift=self.shift)
        return kept

    def bytes_per_token(self) -> float:
        layers, _, kv_heads, _, head_dim = self.k.shape
        per_block = 4 * (2 if self.weight is None else 3)
        return layers * kv_heads * (2 * head_dim + per_block / BLOCK_TOKENS)


__all__ = ["BLOCK_TOKENS", "BlockStore", "EvictionPolicy", "parse_cache_dtype"]
