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
from typing import Dict, Optional, Tuple

import torch

from ... import _capi
from ...kv8_cache import KV8Cache

DTYPES = {torch.float16: _capi.F16, torch.bfloat16: _capi.BF16}
LAYOUTS = {"half": _capi.ROPE_HALF, "interleaved": _capi.ROPE_INTERLEAVED}
BLOCK = 16                              # tokens per block
TILE = 64                               # tokens the kernels take at a time: splits are multiples of it


# A small call's time is the host's, so the checks below are written for the case that they pass: no message is formed, and
# no tensor attribute is read twice, before something is wrong.
def _rows(x: torch.Tensor, what: str, dtype: torch.dtype, device: torch.device, tokens: int, heads: int, dim: int) -> int:
    """Checks ``x`` [tokens, heads, dim] and returns the distance of its rows in elements."""
    if x.shape != (tokens, heads, dim):
        raise ValueError(f"{what} must be {(tokens, heads, dim)}, got {tuple(x.shape)}")
    if x.dtype != dtype or x.device != device:
        raise ValueError(f"{what} must be {dtype} on {device}, got {x.dtype} on {x.device}")
    s0, s1, s2 = x.stride()
    if (s2 != 1 and dim != 1) or (s1 != dim and heads != 1):
        raise ValueError(f"the heads of a row of {what} must be contiguous")
    return s0 if tokens > 1 else heads * dim


def _out_rows(o: torch.Tensor, what: str, dtype: torch.dtype, device: torch.device, tokens: int, heads: int, dim: int) -> int:
    """The same for an output, which may also be [tokens, heads * dim]; its rows must not overlap."""
    if o.dim() == 2 and o.shape[1] == heads * dim and o.stride(1) == 1:
        o = o.unflatten(1, (heads, dim))
    stride = _rows(o, what, dtype, device, tokens, heads, dim)
    if stride < heads * dim:
        raise ValueError(f"rows of {what} overlap")
    return stride


_here = contextlib.nullcontext()


def _on(device: torch.device):
    """Makes ``device`` the current one for a launch, where it is not."""
    return _here if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _ints(t: Optional[torch.Tensor], what: str, device: torch.device, least: int) -> int:
    """Address of a contiguous int32 tensor of at least ``least`` elements."""
    if t is None or t.dtype != torch.int32 or t.device != device or t.numel() < least or not t.is_contiguous():
        raise ValueError(f"{what} must hold {least} contiguous int32 on {device}")
    return t.data_ptr()


def _batch(block_table: torch.Tensor, infer_state, device: torch.device, prefill: bool, decode: bool,
           prefix_lens: Optional[torch.Tensor] = None) -> _capi.MkvBatch:
    """The step's prefill rows, decode rows or both, as the C entries take them."""
    st = infer_state
    num_prefill, num_decode = st.num_prefill_seqs, st.num_decoding_seqs if decode else 0
    skipped = 0
    if not prefill:
        skipped, num_prefill = num_prefill, 0
    if block_table.dim() != 2:
        raise ValueError("block_table must be [max_seqs, max_blocks_per_seq]")
    rows, width = block_table.shape
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
    return _capi.MkvBatch(table, width, rows, seq_ids, starts, lens, prefixes, decoding, num_prefill,
                          st.num_prefill_tokens if prefill else 0, st.max_prefill_len if prefill else 0, num_decode)


def _geometry(cache: KV8Cache, model_config, engine_config, dtype: torch.dtype, device: torch.device):
    """The pool descriptor and its (kv heads, head dim), checked against the configs and the type and device of the rows."""
    pool = cache.descriptor()
    if dtype not in DTYPES:
        raise ValueError(f"rows must be float16 or bfloat16, got {dtype}")
    if device.type != "cuda" or device != cache.device:
        raise ValueError(f"rows on {device}, the cache on {cache.device}")
    _, _, heads, block, dim = cache.shape
    if heads != model_config.num_kv_heads or dim != model_config.head_dim:
        raise ValueError(f"the cache has {heads} heads x {dim}, the model {model_config.num_kv_heads} x {model_config.head_dim}")
    if block != engine_config.block_size:
        raise ValueError(f"the cache has blocks of {block} tokens, the engine of {engine_config.block_size}")
    return pool, heads, dim


def _tables(cos: torch.Tensor, sin: torch.Tensor, device: torch.device) -> Tuple[int, int]:
    """(positions, rotary dim) of a pair of fp32 tables"""
    shape = cos.shape
    if (len(shape) != 2 or shape != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32 or
            cos.device != device or sin.device != device or not cos.is_contiguous() or not sin.is_contiguous()):
        raise ValueError(f"cos and sin must be contiguous float32 [positions, rotary_dim / 2] on {device}")
    return shape[0], 2 * shape[1]


def _layout(layout: str) -> int:
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}, got {layout!r}")
    return LAYOUTS[layout]


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
    dtype, dev = k.dtype, k.device
    pool, heads, dim = _geometry(cache, model_config, engine_config, dtype, dev)
    tokens = infer_state.num_prefill_tokens + infer_state.num_decoding_seqs
    ks, vs = _rows(k, "k", dtype, dev, tokens, heads, dim), _rows(v, "v", dtype, dev, tokens, heads, dim)
    batch = _batch(block_table, infer_state, dev, True, True, prefix_lens)
    with _on(dev):
        _capi.check(_capi.lib().mkv_store8(
            C.byref(pool), C.byref(batch), DTYPES[dtype], k.data_ptr(), v.data_ptr(), ks, vs, cur_layer,
            _capi.ROPE_NONE, None, None, 0, 0, 0, None, None, 0, 0, _stream(dev)))


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
    dtype, dev = k.dtype, k.device
    pool, kv_heads, dim = _geometry(cache, model_config, engine_config, dtype, dev)
    rope = _layout(layout)
    tokens, heads = infer_state.num_prefill_tokens + infer_state.num_decoding_seqs, model_config.num_q_heads
    q_out = q if q_out is None else q_out
    qs, qos = _rows(q, "q", dtype, dev, tokens, heads, dim), _out_rows(q_out, "q_out", dtype, dev, tokens, heads, dim)
    ks, vs = _rows(k, "k", dtype, dev, tokens, kv_heads, dim), _rows(v, "v", dtype, dev, tokens, kv_heads, dim)
    positions, rotary_dim = _tables(cos, sin, dev)
    batch = _batch(block_table, infer_state, dev, True, True, prefix_lens)
    with _on(dev):
        _capi.check(_capi.lib().mkv_store8(
            C.byref(pool), C.byref(batch), DTYPES[dtype], k.data_ptr(), v.data_ptr(), ks, vs, cur_layer, rope, q.data_ptr(),
            q_out.data_ptr(), qs, qos, heads, cos.data_ptr(), sin.data_ptr(), positions, rotary_dim, _stream(dev)))


def _scratch(rows: int, splits: int, dim: int, device: torch.device):
    """Partials of ``rows`` output rows and their log sums, for one call: torch's allocator hands the memory on in stream
    order, and a captured call gets it from its graph's own pool."""
    if splits == 1:
        return None, None, None
    buf = torch.empty(rows * splits * (dim + 1), dtype=torch.float32, device=device)
    return buf, buf.data_ptr(), buf.data_ptr() + 4 * rows * splits * dim


_cus: Dict[int, int] = {}


def _compute_units() -> int:
    """Of the current device; an MI355X's where there is none (tests of the split arithmetic)."""
    if not torch.cuda.is_initialized():
        return 256
    dev = torch.cuda.current_device()
    if dev not in _cus:
        _cus[dev] = torch.cuda.get_device_properties(dev).multi_processor_count
    return _cus[dev]


def choose_split_8bit(n: int, num_kv_heads: int, max_len: int, target_wgs: Optional[int] = None) -> Tuple[int, int]:
    """``(tokens_per_split, max_splits)`` of a decode launch: enough workgroups for the device, none with less than a
    tile for each of its four waves."""
    target = 2 * _compute_units() if target_wgs is None else target_wgs
    max_len = max(max_len, 1)
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
    dtype, dev = q.dtype, q.device
    pool, kv_heads, dim = _geometry(cache, model_config, engine_config, dtype, dev)
    n, heads = infer_state.num_decoding_seqs, model_config.num_q_heads
    qs, os_ = _rows(q, "q", dtype, dev, n, heads, dim), _out_rows(o, "o", dtype, dev, n, heads, dim)
    if n == 0:
        return
    batch = _batch(block_table, infer_state, dev, False, True)
    room = block_table.shape[1] * BLOCK
    known = infer_state.max_decoding_len
    with _on(dev):
        tps, splits = choose_split_8bit(n, kv_heads, min(known, room) if known > 0 else room)
        keep, mid_o, mid_lse = _scratch(n * heads, splits, dim, dev)
        _capi.check(_capi.lib().mkv_attn8_decode(
            C.byref(pool), C.byref(batch), DTYPES[dtype], q.data_ptr(), o.data_ptr(), qs, os_, heads,
            infer_state.softmax_scale, cur_layer, tps, splits, mid_o, mid_lse, _stream(dev)))


def choose_prefill_split_8bit(num_seqs: int, num_q_heads: int, num_kv_heads: int, max_len: int, max_keys: int,
                              target_wgs: Optional[int] = None) -> Tuple[int, int]:
    """``(tokens_per_split, max_splits)`` of a chunk launch: the keys are cut only where the row tiles alone leave
    compute units idle, into ranges of at least four tiles."""
    target = 2 * _compute_units() if target_wgs is None else target_wgs
    row_tiles = -(-max(max_len, 1) * (num_q_heads // num_kv_heads) // 128)
    max_keys = max(max_keys, 1)
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
    dtype, dev = q.dtype, q.device
    pool, kv_heads, dim = _geometry(cache, model_config, engine_config, dtype, dev)
    tokens, heads, seqs = infer_state.num_prefill_tokens, model_config.num_q_heads, infer_state.num_prefill_seqs
    qs, os_ = _rows(q, "q", dtype, dev, tokens, heads, dim), _out_rows(o, "o", dtype, dev, tokens, heads, dim)
    if seqs == 0 or tokens == 0:
        return
    batch = _batch(block_table, infer_state, dev, True, False, prefix_lens)
    room = block_table.shape[1] * BLOCK
    max_len = infer_state.max_prefill_len
    keys = max_len if prefix_lens is None else max_len + max_prefix_len if max_prefix_len else room
    with _on(dev):
        tps, splits = choose_prefill_split_8bit(seqs, heads, kv_heads, max_len, min(keys, room))
        keep, mid_o, mid_lse = _scratch(tokens * heads, splits, dim, dev)
        _capi.check(_capi.lib().mkv_attn8_prefill(
            C.byref(pool), C.byref(batch), DTYPES[dtype], q.data_ptr(), o.data_ptr(), qs, os_, heads,
            infer_state.softmax_scale, cur_layer, tps, splits, mid_o, mid_lse, _stream(dev)))
