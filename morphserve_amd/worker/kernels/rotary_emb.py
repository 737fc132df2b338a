"""Rotary position embedding, alone or fused with the KV append.

``rotary_embedding_inplace`` keeps the operator surface of
MorphServe/worker/kernels/rotary_emb.py:44-58.  ``rotary_embedding_and_store_kvcache``
is the pair the transformer layer runs back to back
(MorphServe/worker/layers/transformer_layer.py:93-126) in ONE launch: q and k are
rotated in place (prefill attention still reads the batch's own k) and the rotated k
and v rows go straight to their cache slots, prefill and decode rows alike.
``rotary_tables`` builds the cos / sin cache of MorphServe/worker/model.py:230-241.

``rotary_embedding`` is the rotary operator in the forms the reference lacks: half and interleaved pairs, part of the
head, fp16 or bf16, rows of any stride, in place or into other tensors, the angles looked up by position in the fp32
tables of ``rotary_scaled_tables`` (plain, or scaled for contexts longer than the trained one).
"""
from __future__ import annotations

import ctypes as C
import math
from typing import List, Optional, Tuple, Union

import torch

from ... import _capi
from . import _deferred
from ._pool import pool_from_args


def rotary_tables(head_dim: int, max_position_embeddings: int, rope_theta: float = 10000.0,
                  rope_scaling: float = 1.0, device: str = "cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """``(_cos_cached, _sin_cached)``: fp16 ``[max_position_embeddings * scaling + 128, head_dim / 2]``."""
    max_seq_len = max_position_embeddings * rope_scaling
    inv_freq = 1.0 / (rope_theta ** (torch.arange(0, head_dim, 2, device=device, dtype=torch.float32) / head_dim))
    t = torch.arange(max_seq_len + 128, device=device, dtype=torch.float32) / rope_scaling
    freqs = torch.outer(t, inv_freq)
    return torch.cos(freqs).to(torch.float16), torch.sin(freqs).to(torch.float16)


def _check(q, k, infer_state):
    assert q.is_contiguous() and k.is_contiguous() and q.dtype == torch.float16 and k.dtype == torch.float16
    cos, sin = infer_state.position_cos, infer_state.position_sin
    assert cos is not None and sin is not None, "infer_state carries no position_cos / position_sin"
    assert cos.is_contiguous() and sin.is_contiguous() and cos.dtype == torch.float16
    assert cos.shape == (q.shape[0], q.shape[2] // 2) == sin.shape, "one cos / sin row per token"
    assert k.shape[0] == q.shape[0] and k.shape[2] == q.shape[2]
    return cos, sin


def rotary_embedding_inplace(
    q: torch.Tensor,    # [num_tokens, num_q_heads, head_dim]
    k: torch.Tensor,    # [num_tokens, num_kv_heads, head_dim]
    infer_state,
) -> None:
    cos, sin = _check(q, k, infer_state)
    _capi.check(_capi.lib().mkv_rope_store_kvcache(
        q.data_ptr(), k.data_ptr(), None, cos.data_ptr(), sin.data_ptr(), None, None, 0, None, None, None, None,
        0, q.shape[0], 0, q.shape[1], k.shape[1], q.shape[2], 0, 0, _capi.current_stream()))


def rotary_embedding_and_store_kvcache(
    q: torch.Tensor,    # [num_tokens, num_q_heads, head_dim], rotated in place
    k: torch.Tensor,    # [num_tokens, num_kv_heads, head_dim], rotated in place
    v: torch.Tensor,    # [num_tokens, num_kv_heads, head_dim]
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_cache_new: List[torch.Tensor],
    v_cache_new: List[torch.Tensor],
    block_table: torch.Tensor,
    model_config,
    engine_config,
    infer_state,
    cur_layer: int,
) -> None:
    cos, sin = _check(q, k, infer_state)
    assert v.is_contiguous() and v.shape == k.shape and block_table.is_contiguous()
    assert q.shape[0] == infer_state.num_tokens
    pool = pool_from_args(k_cache, v_cache, k_cache_new, v_cache_new, infer_state)
    st = infer_state
    _deferred.flush()
    _capi.check(_capi.lib().mkv_rope_store_kvcache(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), cos.data_ptr(), sin.data_ptr(), C.byref(pool),
        block_table.data_ptr(), block_table.shape[1], st.seq_ids.data_ptr(),
        _capi.ptr(st.prefill_seq_start_locs), _capi.ptr(st.prefill_seq_lens), _capi.ptr(st.decoding_seq_lens),
        st.num_prefill_seqs, st.num_prefill_tokens, st.num_decoding_seqs, q.shape[1], k.shape[1], q.shape[2],
        cur_layer, 1, _capi.current_stream()))


# the keys that each scaling rule reads, and those that any dict may hold: the rule's name, and what the arguments say already
_SCALING_KEYS = {
    "default": (),
    "linear": ("factor",),
    "dynamic": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor"),
    "yarn": ("factor", "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate"),
}
_COMMON_KEYS = ("rope_type", "type", "rope_theta", "partial_rotary_factor", "original_max_position_embeddings", "finetuned")


def _scaling_rule(scaling: dict, theta: float) -> str:
    """The rule's name; ``ValueError`` for one that is not known, and for keys that it would leave unread."""
    kinds = {str(scaling[key]) for key in ("rope_type", "type") if scaling.get(key) is not None} or {"default"}
    if len(kinds) > 1 or not kinds <= _SCALING_KEYS.keys():
        raise ValueError(f"unknown rotary scaling {' / '.join(sorted(map(repr, kinds)))}")
    kind = kinds.pop()
    unread = [key for key in scaling if key not in _SCALING_KEYS[kind] + _COMMON_KEYS]
    if unread:
        raise ValueError(f"rotary scaling {kind!r} does not know {', '.join(map(repr, unread))}")
    if _number(scaling, "rope_theta", theta) != theta:
        raise ValueError(f"rope_theta is {theta}, the scaling's {scaling['rope_theta']}")
    return kind


def _number(scaling: dict, key: str, usual: Optional[float] = None) -> float:
    value = scaling.get(key)
    if value is None:
        value = usual
    try:
        value = float(value)
    except (TypeError, ValueError):
        raise ValueError(f"rotary scaling needs a number as {key!r}, got {value!r}") from None
    if not math.isfinite(value):
        raise ValueError(f"rotary scaling needs a finite {key!r}, got {value}")
    return value


def _scaled_inv_freq(rotary_dim: int, theta: float, scaling: dict, seq_len: int) -> Tuple[torch.Tensor, float]:
    """Inverse frequencies in 64 bits and the factor of the cosines and sines, for one scaling rule."""
    kind = _scaling_rule(scaling, theta)
    pair = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    inv = theta ** (-pair / rotary_dim)
    if kind == "default":
        return inv, 1.0
    factor = _number(scaling, "factor")
    if factor < 1:
        raise ValueError(f"a rotary scaling factor is at least 1, got {factor}")
    if kind == "linear":                                    # positions / factor
        return inv / factor, 1.0
    old = _number(scaling, "original_max_position_embeddings")
    if old <= 0:
        raise ValueError(f"original_max_position_embeddings must be positive, got {old}")
    if kind == "dynamic":                                   # a larger base, by how far the context exceeds the trained one
        if rotary_dim <= 2:
            raise ValueError("rotary scaling 'dynamic' needs a rotary dim above 2")
        grown = max(1.0, factor * max(seq_len, old) / old - (factor - 1))
        return (theta * grown ** (rotary_dim / (rotary_dim - 2))) ** (-pair / rotary_dim), 1.0
    if kind == "llama3":                                    # slow pairs / factor, fast pairs kept, a ramp between
        low, high = _number(scaling, "low_freq_factor", 1.0), _number(scaling, "high_freq_factor", 4.0)
        if high <= low:
            raise ValueError("high_freq_factor must exceed low_freq_factor")
        turns = old * inv / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return inv * keep + inv / factor * (1 - keep), 1.0
    # yarn: the ramp runs over the pairs' numbers
    fast, slow = _number(scaling, "beta_fast", 32.0), _number(scaling, "beta_slow", 1.0)
    if not fast > slow > 0 or theta <= 1:
        raise ValueError(f"rotary scaling 'yarn' needs beta_fast > beta_slow > 0 and a base above 1, got {fast}, {slow}, {theta}")
    pair_of = lambda turns: rotary_dim * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
    first, last = pair_of(fast), pair_of(slow)
    truncate = scaling.get("truncate")
    if truncate not in (None, True, False):
        raise ValueError(f"truncate is true or false, got {truncate!r}")
    if truncate is None or truncate:                        # the ramp's ends at whole pairs
        first, last = math.floor(first), math.ceil(last)
    first, last = max(first, 0), min(last, rotary_dim - 1)
    ramp = ((pair / 2 - first) / max(last - first, 0.001)).clamp(0, 1)
    if scaling.get("attention_factor") is not None:
        attention = _number(scaling, "attention_factor")
    else:                                                   # two scales, of the angles' and of all dims: their ratio
        of = lambda key, usual: 0.1 * _number(scaling, key, usual) * math.log(factor) + 1.0  # noqa: E731
        attention = of("mscale", 1.0) / of("mscale_all_dim", 0.0)
    return inv / factor * ramp + inv * (1 - ramp), attention


def rotary_scaled_tables(rotary_dim: int, num_positions: int, rope_theta: float = 10000.0,
                         rope_scaling: Union[None, float, dict] = None,
                         device: str = "cuda") -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 ``(cos, sin)`` [num_positions, rotary_dim / 2], angles computed in 64 bits (a far position times a frequency
    loses its phase in 32).  ``rope_scaling``: ``None``, a number (linear), or the dict of a model's config with
    ``rope_type`` one of ``default``, ``linear``, ``dynamic``, ``llama3``, ``yarn`` (``mscale``, ``mscale_all_dim`` and
    ``truncate`` included).  ``dynamic`` takes ``num_positions`` as the context's length.  A rule, or a key of the dict, that is
    not known is refused with ``ValueError``, and so is a ``rope_theta`` in it that differs from the argument."""
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if rope_scaling is None:
        rope_scaling = {}
    elif not isinstance(rope_scaling, dict):
        rope_scaling = {"rope_type": "linear", "factor": rope_scaling}
    theta = float(rope_theta)
    if not (theta > 0 and math.isfinite(theta)) or num_positions < 0:
        raise ValueError(f"rotary tables need a positive base and a number of positions, got {rope_theta}, {num_positions}")
    inv, mul = _scaled_inv_freq(rotary_dim, theta, rope_scaling, num_positions)
    angle = torch.outer(torch.arange(num_positions, dtype=torch.float64, device=device), inv.to(device))
    return (torch.cos(angle) * mul).float(), (torch.sin(angle) * mul).float()


def rotary_embedding(
    q: torch.Tensor,                    # [num_tokens, num_q_heads, head_dim] fp16 or bf16
    k: Optional[torch.Tensor],          # [num_tokens, num_kv_heads, head_dim], or None
    positions: torch.Tensor,            # [num_tokens] int32
    cos: torch.Tensor,                  # [max positions, rotary_dim / 2] fp32
    sin: torch.Tensor,
    layout: str = "half",               # pairs (d, d + rotary_dim / 2); "interleaved": pairs (2d, 2d + 1)
    q_out: Optional[torch.Tensor] = None,         # None: in place; otherwise a tensor that does not overlap q
    k_out: Optional[torch.Tensor] = None,
) -> None:
    """Rotates the first ``rotary_dim`` dims of every head by its token's position, in 32 bits, and keeps the others.  A
    token whose position lies outside the tables gets NaN in its rotated dims."""
    _capi.check(_capi.binding().rope(_capi.entry("mkv_rope_positions"), q, k, positions, cos, sin, layout, q_out, k_out))
