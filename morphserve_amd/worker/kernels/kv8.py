"""The operators of the paged path over the 8-bit cache (``kv8_cache.KV8Cache``).

``store_kvcache_8bit``, ``paged_attention_8bit`` and ``chunked_prefill_attention_8bit`` are ``store_kvcache``
(MorphServe/worker/kernels/kvcache_mgmt.py:298-414), ``paged_attention``
(MorphServe/worker/kernels/paged_attn.py:700-1015) and ``chunked_prefill_attention`` with a ``KV8Cache`` in place of
the four cache arguments; ``rotary_embedding_and_store_kvcache_8bit`` is the pair of rotary embedding and append that
a layer runs back to back (MorphServe/worker/layers/transformer_layer.py:93-126) in one launch.  q, k, v and o are fp16
or bf16, rows of any stride whose head dims are contiguous (slices of a fused projection as they are).  A cache is
read with the type it was written with.

All calls launch on the current stream of the tensors' device, allocate nothing but the split partials (from torch's
allocator, on that stream) and can be captured into a graph.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from ... import _capi
from ...kv8_cache import KV8Cache

# (tokens_per_split, max_splits) for every attention call of the process instead of the rules below; tests set it
FORCED_SPLIT: Optional[Tuple[int, int]] = None


def store_kvcache_8bit(
    k: torch.Tensor,                    # [num_tokens, num_kv_heads, head_dim]
    v: torch.Tensor,
    cache: KV8Cache,
    block_table: torch.Tensor,          # [max_seqs, max_blocks_per_seq] int32
    model_config,
    engine_config,
    infer_state,
    cur_layer: int,
    prefix_lens: Optional[torch.Tensor] = None,   # [num_prefill_seqs] int32 cached tokens before each chunk
) -> None:
    """Prefill rows go to positions ``prefix_lens[b] + t`` of their sequences, decode rows to position ``len - 1``.

    A block's scale is the least power of two that holds its rows.  Rows that join a block later can only raise it;
    the codes already there are then rounded to the new scale.  Rows of the cache beyond those written keep their codes.
    A sequence appears once in a batch; a row without a block in the pool is not stored."""
    _capi.check(_capi.binding().store(
        _capi.entry("mkv_store8"), k, v, cache.k, cache.v, cache.scales, block_table, model_config, engine_config,
        infer_state, cur_layer, prefix_lens))


def rotary_embedding_and_store_kvcache_8bit(
    q: torch.Tensor,                    # [num_tokens, num_q_heads, head_dim], rotated into q_out
    k: torch.Tensor,                    # [num_tokens, num_kv_heads, head_dim], left as it is
    v: torch.Tensor,
    cos: torch.Tensor,                  # [positions, rotary_dim / 2] fp32, rows by position
    sin: torch.Tensor,
    cache: KV8Cache,
    block_table: torch.Tensor,
    model_config,
    engine_config,
    infer_state,
    cur_layer: int,
    layout: str = "half",               # or "interleaved", as for rotary_embedding
    q_out: Optional[torch.Tensor] = None,         # None: q itself; otherwise a tensor that overlaps no input
    prefix_lens: Optional[torch.Tensor] = None,
) -> None:
    """``rotary_embedding`` of q and k by their positions in the sequences, then ``store_kvcache_8bit``, in one launch.
    The rotated k goes to the cache only, rounded once, from 32 bits to its code.  The rotary dim must be a multiple of
    16.  A row whose position lies outside the tables is not stored and its q becomes NaN."""
    _capi.check(_capi.binding().store(
        _capi.entry("mkv_store8"), k, v, cache.k, cache.v, cache.scales, block_table, model_config, engine_config,
        infer_state, cur_layer, prefix_lens, q, cos, sin, layout, q_out))


def choose_split_8bit(n: int, num_kv_heads: int, max_len: int, units: int = 256, num_q_heads: Optional[int] = None,
                      head_dim: int = 128) -> Tuple[int, int]:
    """``(tokens_per_split, max_splits)`` of a decode launch over ``n`` rows on ``units`` compute units: the ranges with the
    least estimated time, their joining included.  ``paged_attention_8bit`` takes them so; a caller of ``mkv_attn8_decode``
    passes them."""
    return _capi.binding().decode_split(n, num_kv_heads, max_len, units, num_q_heads or num_kv_heads, head_dim)


def paged_attention_8bit(
    q: torch.Tensor,                    # [num_decoding_seqs, num_q_heads, head_dim]
    cache: KV8Cache,
    block_table: torch.Tensor,
    model_config,
    engine_config,
    infer_state,
    cur_layer: int,
    o: torch.Tensor,                    # [num_decoding_seqs, num_q_heads * head_dim] (or 3-D), written
) -> None:
    """Decode attention: row i over the first ``decoding_seq_lens[i]`` positions of its sequence; zeros where there is
    nothing to attend to."""
    _capi.check(_capi.binding().decode(
        _capi.entry("mkv_attn8_decode"), q, cache.k, cache.v, cache.scales, block_table, model_config, engine_config,
        infer_state, cur_layer, o, FORCED_SPLIT))


def choose_prefill_split_8bit(num_seqs: int, num_q_heads: int, num_kv_heads: int, max_len: int, max_keys: int,
                              units: int = 256, head_dim: int = 128) -> Tuple[int, int]:
    """``(tokens_per_split, max_splits)`` of a chunk launch, chosen like a decode launch's."""
    return _capi.binding().prefill_split(num_seqs, num_q_heads, num_kv_heads, max_len, max_keys, units, head_dim)


def chunked_prefill_attention_8bit(
    q: torch.Tensor,                    # [num_prefill_tokens, num_q_heads, head_dim]
    cache: KV8Cache,
    block_table: torch.Tensor,
    model_config,
    engine_config,
    infer_state,
    cur_layer: int,
    o: torch.Tensor,                    # [num_prefill_tokens, num_q_heads * head_dim] (or 3-D), written
    prefix_lens: Optional[torch.Tensor] = None,   # [num_prefill_seqs] int32 cached tokens before each chunk
    max_prefix_len: int = 0,            # host-side upper bound of prefix_lens (0 = unknown): picks the launch shape only
) -> None:
    """Chunk b = rows ``prefill_seq_start_locs[b] : + prefill_seq_lens[b]`` of ``q`` at positions ``prefix_lens[b] ..`` of
    sequence ``seq_ids[b]``, its own rows appended before; the row at position p attends to cached positions <= p.  A
    whole prompt is a chunk without a prefix.  Rows of ``o`` that belong to no chunk are left as they are."""
    _capi.check(_capi.binding().prefill(
        _capi.entry("mkv_attn8_prefill"), q, cache.k, cache.v, cache.scales, block_table, model_config, engine_config,
        infer_state, cur_layer, o, prefix_lens, max_prefix_len, FORCED_SPLIT))
