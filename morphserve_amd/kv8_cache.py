"""The paged KV cache in 8 bits.

The reference's cache is fp16 (MorphServe/worker/model.py:180-190).  This one holds the codes of K and V in 8 bits --
``torch.float8_e4m3fn`` or ``torch.int8`` -- and one power-of-two scale for each (block, layer, kv head), K and V
apart: half the memory, and half the bytes a decode step has to read.  Block ids, block tables and the
``BlockManager`` are the fp16 cache's.

A code stands for ``code * 2 ** (scale - 127)``.  e4m3 keeps four significant bits of every value whatever the other
values of its block are; int8 keeps eight bits of the block's largest, which is closer for values of like size and
coarser for a block with a few large ones.
"""
from __future__ import annotations

import dataclasses
from typing import Sequence

import torch

from . import _capi

KINDS = (torch.float8_e4m3fn, torch.int8)


@dataclasses.dataclass
class KV8Cache:
    """``k`` [num_blocks, L, Hkv, 16, D], ``v`` [num_blocks, L, Hkv, D, 16] (a head dim's tokens innermost), both
    contiguous and of one code type; ``scales`` [L, Hkv, num_blocks, 2] uint8, the biased exponents of K and V."""
    k: torch.Tensor
    v: torch.Tensor
    scales: torch.Tensor

    @property
    def num_blocks(self) -> int:
        return self.k.shape[0]

    def descriptor(self) -> _capi.MkvPool8:
        """The cache as the C entries of include/morphkv.h take it; ``ValueError`` if the tensors do not make one."""
        return _capi.MkvPool8(*_capi.binding().pool_fields(self.k, self.v, self.scales))


def allocate_kv8_cache(num_blocks: int, shape_tail: Sequence[int], dtype: torch.dtype = torch.float8_e4m3fn,
                       device: str = "cuda") -> KV8Cache:
    """An empty cache of ``num_blocks`` blocks; ``shape_tail`` is ``(L, Hkv, block_size, D)`` as for
    ``allocate_kv_caches``.  Zero codes, scales of 1."""
    layers, heads, block, dim = (int(x) for x in shape_tail)
    if dtype not in KINDS:
        raise ValueError(f"an 8-bit cache holds float8_e4m3fn or int8 codes, got {dtype}")
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype)  # noqa: E731
    return KV8Cache(zeros(num_blocks, layers, heads, block, dim), zeros(num_blocks, layers, heads, dim, block),
                    torch.full((layers, heads, num_blocks, 2), 127, dtype=torch.uint8, device=device))
