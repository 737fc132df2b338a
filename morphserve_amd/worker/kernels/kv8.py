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

import contextlib
import ctypes as C
from typing import Optional, Tuple

import torch

from ... import _capi
from ...kv8_cache import KV8Cache
from .paged_attn import target_workgroups

DTYPES = {torch.float16: _capi.F16, torch.bfloat16: _capi.BF16}
LAYOUTS = {"half": _capi.ROPE_HALF, "interleaved": _capi.ROPE_INTERLEAVED}
TILE = 64                               # tokens the kernels take at a time: splits are multiples of it


def _require(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _rows(x: torch.Tensor, what: str, like: torch.Tensor, tokens: int, heads: int, dim: int) -> int:
    """Checks ``x`` [tokens, heads, dim] and returns the distance of its rows in elements."""
    _require(tuple(x.shape) == (tokens, heads, dim), f"{what} must be {(tokens, heads, dim)}, got {tuple(x.shape)}")
    _require(x.dtype == like.dtype and x.device == like.device, f"{what} must be {like.dtype} on {like.device}")
    s0, s1, s2 = x.stride()
    _require((s2 == 1 or dim == 1) and (s1 == dim or heads == 1), f"the heads of a row of {what} must be contiguous")
    return s0 if tokens > 1 else heads * dim


def _out_rows(o: torch.Tensor, what: str, like: torch.Tensor, tokens: int, heads: int, dim: int) -> int:
    """The same for an output, which may also be [tokens, heads * dim]; its rows must not overlap."""
    if o.dim() == 2 and o.shape[1] == heads * dim and (o.stride(1) == 1):
        o = o.unflatten(1, (heads, dim))
    stride = _rows(o, what, like, tokens, heads, dim)
    _require(stride >= heads * dim, f"rows of {what} overlap")
    return stride


def _on(device: torch.device):
    """Makes ``device`` the current one for a launch, where it is not."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _ints(t: Optional[torch.Tensor], what: str, device: torch.device, least: int) -> int:
    """Address of a contiguous int32 tensor of at least ``least`` elements."""
    _require(t is not None and t.dtype == torch.int32 and t.is_contiguous() and t.device == device and t.numel() >= least,
             f"{what} must hold {least} contiguous int32 on {device}")
    return t.data_ptr()


def _batch(block_table: torch.Tensor, infer_state, device: torch.device, prefill: bool, decode: bool,
           prefix_lens: Optional[torch.Tensor] = None) -> _capi.MkvBatch:
    """The step's prefill rows, decode rows or both, as the C entries take them."""
    st = infer_state
    skipped = 0 if prefill else st.num_prefill_seqs
    num_prefill = st.num_prefill_seqs - skipped
    num_decode = st.num_decoding_seqs if decode else 0
    _require(block_table.dim() == 2, "block_table must be [max_seqs, max_blocks_per_seq]")
    table = _ints(block_table, "block_table", device, 0)
    seq_ids = _ints(st.seq_ids, "infer_state.seq_ids", device, skipped + num_prefill + num_decode) + 4 * skipped
    starts = lens = prefixes = decoding = None
    if num_prefill:
        starts = _ints(st.prefill_seq_start_locs, "infer_state.prefill_seq_start_locs", device, num_prefill)
        lens = _ints(st.prefill_seq_lens, "infer_state.prefill_seq_lens", device, num_prefill)
        if prefix_lens is not None:
            prefixes = _ints(prefix_lens, "prefix_lens", device, num_prefill)
    if num_decode:
        decoding = _ints(st.decoding_seq_lens, "infer_state.decoding_seq_lens", device, num_decode)
    return _capi.MkvBatch(table, block_table.shape[1], block_table.shape[0], seq_ids, starts, lens, prefixes, decoding,
                          num_prefill, st.num_prefill_tokens if prefill else 0, st.max_prefill_len if prefill else 0,
                          num_decode)


def _geometry(cache: KV8Cache, model_config, engine_config, x: torch.Tensor):
    """The pool descriptor, checked against the configs and the type and device of the rows."""
    pool = cache.descriptor()
    _require(x.dtype in DTYPES, f"rows must be float16 or bfloat16, got {x.dtype}")
    _require(x.is_cuda and x.device == cache.k.device, f"rows on {x.device}, the cache on {cache.k.device}")
    _require(pool.num_kv_heads == model_config.num_kv_heads and pool.head_dim == model_config.head_dim,
             f"the cache has {pool.num_kv_heads} heads x {pool.head_dim}, the model {model_config.num_kv_heads} x "
             f"{model_config.head_dim}")
    _require(pool.block_size == engine_config.block_size,
             f"the cache has blocks of {pool.block_size} tokens, the engine of {engine_config.block_size}")
    return pool


def _tables(cos: torch.Tensor, sin: torch.Tensor, device: torch.device) -> Tuple[int, int]:
    """(positions, rotary dim) of a pair of fp32 tables"""
    _require(cos.dim() == 2 and cos.shape == sin.shape and cos.dtype == sin.dtype == torch.float32 and
             cos.is_contiguous() and sin.is_contiguous() and cos.device == sin.device == device,
             f"cos and sin must be contiguous float32 [positions, rotary_dim / 2] on {device}")
    return cos.shape[0], 2 * cos.shape[1]


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
    pool = _geometry(cache, model_config, engine_config, k)
    tokens = infer_state.num_prefill_tokens + infer_state.num_decoding_seqs
    ks = _rows(k, "k", k, tokens, pool.num_kv_heads, pool.head_dim)
    vs = _rows(v, "v", k, tokens, pool.num_kv_heads, pool.head_dim)
    batch = _batch(block_table, infer_state, k.device, True, True, prefix_lens)
    with _on(k.device):
        _capi.check(_capi.lib().mkv_store8(
            C.byref(pool), C.byref(batch), DTYPES[k.dtype], k.data_ptr(), v.data_ptr(), ks, vs, cur_layer,
            _capi.ROPE_NONE, None, None, 0, 0, 0, None, None, 0, 0, _capi.current_stream()))


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
    q_out: Optional[torch.Tensor] = None,         # None: q itself
    prefix_lens: Optional[torch.Tensor] = None,
) -> None:
    """``rotary_embedding`` of q and k by their positions in the sequences, then ``store_kvcache_8bit``, in one launch.
    The rotated k goes to the cache only, rounded once, from 32 bits to its code.  The rotary dim must be a multiple of
    16.  A row whose position lies outside the tables is not stored and its q becomes NaN."""
    pool = _geometry(cache, model_config, engine_config, k)
    _require(layout in LAYOUTS, f"layout must be one of {sorted(LAYOUTS)}, got {layout!r}")
    tokens = infer_state.num_prefill_tokens + infer_state.num_decoding_seqs
    heads, dim = model_config.num_q_heads, pool.head_dim
    q_out = q if q_out is None else q_out
    qs = _rows(q, "q", k, tokens, heads, dim)
    os_ = _out_rows(q_out, "q_out", k, tokens, heads, dim)
    ks = _rows(k, "k", k, tokens, pool.num_kv_heads, dim)
    vs = _rows(v, "v", k, tokens, pool.num_kv_heads, dim)
    positions, rotary_dim = _tables(cos, sin, k.device)
    batch = _batch(block_table, infer_state, k.device, True, True, prefix_lens)
    with _on(k.device):
        _capi.check(_capi.lib().mkv_store8(
            C.byref(pool), C.byref(batch), DTYPES[k.dtype], k.data_ptr(), v.data_ptr(), ks, vs, cur_layer,
            LAYOUTS[layout], q.data_ptr(), q_out.data_ptr(), qs, os_, heads, cos.data_ptr(), sin.data_ptr(), positions,
            rotary_dim, _capi.current_stream()))


def _scratch(rows: int, splits: int, dim: int, device: torch.device):
    """Partials of ``rows`` output rows and their log sums, for one call: torch's allocator hands the memory on in stream
    order, and a captured call gets it from its graph's own pool."""
    if splits == 1:
        return None, None, None
    buf = torch.empty(rows * splits * (dim + 1), dtype=torch.float32, device=device)
    return buf, buf.data_ptr(), buf.data_ptr() + 4 * rows * splits * dim


def choose_split_8bit(n: int, num_kv_heads: int, max_len: int, target_wgs: Optional[int] = None) -> Tuple[int, int]:
    """``(tokens_per_split, max_splits)`` of a decode launch: enough workgroups for the device, none with less than a
    tile for each of its four waves."""
    target = target_workgroups() if target_wgs is None else target_wgs
    max_len = max(int(max_len), 1)
    splits = min(-(-target // max(1, n * num_kv_heads)), max(1, max_len // (4 * TILE)))
    tps = -(-max_len // splits)
    tps = -(-tps // TILE) * TILE
    return tps, -(-max_len // tps)


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
    pool = _geometry(cache, model_config, engine_config, q)
    n, heads, dim = infer_state.num_decoding_seqs, model_config.num_q_heads, pool.head_dim
    qs = _rows(q, "q", q, n, heads, dim)
    os_ = _out_rows(o, "o", q, n, heads, dim)
    if n == 0:
        return
    batch = _batch(block_table, infer_state, q.device, False, True)
    room = block_table.shape[1] * pool.block_size
    known = int(getattr(infer_state, "max_decoding_len", 0) or 0)
    with _on(q.device):
        tps, splits = choose_split_8bit(n, pool.num_kv_heads, min(known, room) if known else room)
        keep, mid_o, mid_lse = _scratch(n * heads, splits, dim, q.device)
        _capi.check(_capi.lib().mkv_attn8_decode(
            C.byref(pool), C.byref(batch), DTYPES[q.dtype], q.data_ptr(), o.data_ptr(), qs, os_, heads,
            float(infer_state.softmax_scale), cur_layer, tps, splits, mid_o, mid_lse, _capi.current_stream()))


def choose_prefill_split_8bit(num_seqs: int, num_q_heads: int, num_kv_heads: int, max_len: int, max_keys: int,
                              target_wgs: Optional[int] = None) -> Tuple[int, int]:
    """``(tokens_per_split, max_splits)`` of a chunk launch: the keys are cut only where the row tiles alone leave
    compute units idle, into ranges of at least four tiles."""
    target = target_workgroups() if target_wgs is None else target_wgs
    row_tiles = -(-max(max_len, 1) * (num_q_heads // num_kv_heads) // 128)
    max_keys = max(int(max_keys), 1)
    splits = min(max(1, target // max(1, num_seqs * num_kv_heads * row_tiles)), max(1, max_keys // (4 * TILE)))
    tps = -(-max_keys // splits)
    tps = -(-tps // TILE) * TILE
    return tps, -(-max_keys // tps)


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
    pool = _geometry(cache, model_config, engine_config, q)
    tokens, heads, dim = infer_state.num_prefill_tokens, model_config.num_q_heads, pool.head_dim
    qs = _rows(q, "q", q, tokens, heads, dim)
    os_ = _out_rows(o, "o", q, tokens, heads, dim)
    if infer_state.num_prefill_seqs == 0 or tokens == 0:
        return
    batch = _batch(block_table, infer_state, q.device, True, False, prefix_lens)
    room = block_table.shape[1] * pool.block_size
    max_len = infer_state.max_prefill_len
    keys = max_len if prefix_lens is None else max_len + max_prefix_len if max_prefix_len else room
    with _on(q.device):
        tps, splits = choose_prefill_split_8bit(infer_state.num_prefill_seqs, heads, pool.num_kv_heads, max_len,
                                                min(keys, room))
        keep, mid_o, mid_lse = _scratch(tokens * heads, splits, dim, q.device)
        _capi.check(_capi.lib().mkv_attn8_prefill(
            C.byref(pool), C.byref(batch), DTYPES[q.dtype], q.data_ptr(), o.data_ptr(), qs, os_, heads,
            float(infer_state.softmax_scale), cur_layer, tps, splits, mid_o, mid_lse, _capi.current_stream()))
