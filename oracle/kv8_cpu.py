"""The 8-bit paged cache and the rotary forms, restated plainly on the CPU: 64-bit arithmetic, one row, head and block at
a time.  There is no counterpart in the reference (its cache is fp16, MorphServe/worker/model.py:180-190); these
definitions are this repository's own.

k codes [N, L, Hkv, 16, D], v codes [N, L, Hkv, D, 16], both as uint8 bit patterns; scales [L, Hkv, N, 2] uint8 biased
exponents; a code stands for ``code * 2 ** (scale - 127)``.
"""
from __future__ import annotations

import math

import numpy as np

B = 16
QMAX = {"e4m3": 448.0, "int8": 127.0}
# rows beyond this magnitude saturate: the largest value whose code cannot stand for an infinity of the type
MOST = {"f16": 1.875 * 2.0 ** 15, "bf16": 1.875 * 2.0 ** 127}


def _e4m3_values() -> np.ndarray:
    out = np.zeros(256)
    for u in range(256):
        e, m = (u >> 3) & 15, u & 7
        mag = math.nan if (u & 127) == 127 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[u] = -mag if u & 128 else mag
    return out


E4M3 = _e4m3_values()
INT8 = np.arange(256, dtype=np.uint8).view(np.int8).astype(np.float64)


def decode(codes: np.ndarray, kind: str) -> np.ndarray:
    return (E4M3 if kind == "e4m3" else INT8)[codes]


def encode(x: np.ndarray, kind: str) -> np.ndarray:
    """nearest code, ties to even; |x| <= QMAX; NaN: a NaN (e4m3) or 0 (int8)"""
    x = np.asarray(x, dtype=np.float64)
    if kind == "int8":
        return np.rint(np.where(np.isnan(x), 0, x)).astype(np.int8).view(np.uint8)
    grid = E4M3[:127]                                       # 0 .. 448 ascending: code u has magnitude grid[u]
    mag = np.where(np.isnan(x), 0, np.abs(x))
    hi = np.clip(np.searchsorted(grid, mag), 1, 126)
    lo = hi - 1
    below, above = mag - grid[lo], grid[hi] - mag
    code = np.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi).astype(np.uint8)
    code = np.where(np.isnan(x), 127, code).astype(np.uint8)
    return (code | np.where(np.signbit(x), 128, 0).astype(np.uint8)).astype(np.uint8)


def exponent(amax: float, kind: str) -> int:
    """least biased exponent e >= 1 with amax <= QMAX * 2 ** (e - 127)"""
    e = 1
    while amax > QMAX[kind] * 2.0 ** (e - 127):
        e += 1
    return e


def clamp(x: np.ndarray, dtype: str) -> np.ndarray:
    return np.where(np.isnan(x), x, np.clip(x, -MOST[dtype], MOST[dtype]))


def join(codes: np.ndarray, scale: int, rows: np.ndarray, a: int, kind: str, dtype: str):
    """Rows [a, a + len(rows)) join a slab [16, D] of codes: (new codes, new scale)."""
    x = clamp(rows.astype(np.float64), dtype)
    finite = np.abs(x[~np.isnan(x)])
    e = exponent(float(finite.max(initial=0.0)), kind)
    codes = codes.copy()
    if a > 0:
        e = max(e, scale)
        if e != scale:
            old = decode(codes[:a], kind) * (2.0 ** (scale - e) if scale else 0.0)
            codes[:a] = encode(old, kind)
    codes[a:a + len(x)] = encode(x * 2.0 ** (127 - e), kind)
    return codes, e


def rows_of(starts, lens, prefixes, num_prefill_tokens, dec_lens, dtype_rows):
    """(batch slot, first position, first row, number of rows) of every run of rows in a batch"""
    out = [(b, int(p), int(s), int(n)) for b, (s, n, p) in enumerate(zip(starts, lens, prefixes)) if n > 0]
    return out + [(len(lens) + i, int(n) - 1, num_prefill_tokens + i, 1) for i, n in enumerate(dec_lens) if n > 0]


def store(kc, vc, scales, k, v, table, seq_ids, runs, layer, kind, dtype, num_positions=None):
    """Appends the runs of rows (``rows_of``) in place.  k, v [rows, Hkv, D] float; rows at positions >= num_positions,
    without a table row or without a block in the pool are not stored."""
    n_blocks, _, heads, _, _ = kc.shape
    for slot, pos, row, count in runs:
        seq = int(seq_ids[slot])
        if not 0 <= seq < table.shape[0]:
            continue
        end = pos + count if num_positions is None else min(pos + count, num_positions)
        for j in range(pos // B, (pos + count - 1) // B + 1):
            lo, hi = max(pos, j * B), min(end, (j + 1) * B)
            if j >= table.shape[1] or lo >= hi:
                continue
            pid = int(table[seq, j])
            if not 0 <= pid < n_blocks:
                continue
            src = slice(row + lo - pos, row + hi - pos)
            for h in range(heads):
                kc[pid, layer, h], scales[layer, h, pid, 0] = join(
                    kc[pid, layer, h], int(scales[layer, h, pid, 0]), k[src, h], lo - j * B, kind, dtype)
                new, scales[layer, h, pid, 1] = join(
                    vc[pid, layer, h].T, int(scales[layer, h, pid, 1]), v[src, h], lo - j * B, kind, dtype)
                vc[pid, layer, h] = new.T


def rotate(x: np.ndarray, positions, cos, sin, layout: str, dtype=np.float64) -> np.ndarray:
    """x [rows, heads, D] rotated by the tables' rows; ``dtype`` is the arithmetic's (products and sums each rounded)"""
    x = x.astype(dtype)
    half = cos.shape[1]
    pos = np.asarray(positions, dtype=np.int64)
    known = (pos >= 0) & (pos < cos.shape[0])
    c = np.where(known[:, None], cos[np.where(known, pos, 0)], np.nan).astype(dtype)[:, None]
    s = np.where(known[:, None], sin[np.where(known, pos, 0)], np.nan).astype(dtype)[:, None]
    a, b = (slice(0, half), slice(half, 2 * half)) if layout == "half" else (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
    out = x.copy()
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., a] * s + x[..., b] * c
    return out


def gather(kc, vc, scales, table_row, keys, layer, head, kind):
    """K, V [keys, D] of a sequence in 64 bits and which of its positions exist"""
    dim = kc.shape[4]
    k, v, there = np.zeros((keys, dim)), np.zeros((keys, dim)), np.zeros(keys, dtype=bool)
    for j in range(-(-keys // B)):
        pid = int(table_row[j]) if j < len(table_row) else -1
        if not 0 <= pid < kc.shape[0]:
            continue
        at = slice(j * B, min((j + 1) * B, keys))
        n = at.stop - at.start
        e = scales[layer, head, pid].astype(np.float64) - 127
        k[at] = decode(kc[pid, layer, head, :n], kind) * 2.0 ** e[0]
        v[at] = decode(vc[pid, layer, head].T[:n], kind) * 2.0 ** e[1]
        there[at] = True
    return k, v, there


def attend(q, kc, vc, scales, table, seq, last, layer, kind, scale):
    """q [rows, Hq, D], row r of one sequence sees positions <= last[r].  Returns the output and what its error is bounded
    by: ``sum p |v|``, the largest ``scale sum |q k|``, the number of keys and the largest |v|, each [rows, Hq, ...]."""
    rows, hq, dim = q.shape
    heads = kc.shape[2]
    group = hq // heads
    out = np.zeros((rows, hq, dim))
    mean = np.zeros((rows, hq, dim))
    big = np.zeros((rows, hq, 1))
    most = np.zeros((rows, hq, 1))
    keys = max([int(x) + 1 for x in last] + [0])
    if not 0 <= seq < table.shape[0] or keys == 0:
        return out, mean, big, np.zeros((rows, 1, 1)), most
    for h in range(heads):
        k, v, there = gather(kc, vc, scales, table[seq], keys, layer, h, kind)
        sees = there[None] & (np.arange(keys)[None] <= np.asarray(last)[:, None])
        for g in range(h * group, (h + 1) * group):
            s = np.where(sees, q[:, g].astype(np.float64) @ k.T * scale, -np.inf)
            top = np.where(sees.any(1), s.max(1), 0.0)
            p = np.where(sees, np.exp(s - top[:, None]), 0.0)
            total = p.sum(1, keepdims=True)
            p = np.where(total > 0, p / np.where(total > 0, total, 1), 0.0)
            out[:, g], mean[:, g] = p @ np.where(there[:, None], v, 0), p @ np.abs(v)
            big[:, g, 0] = np.where(sees, np.abs(q[:, g]).astype(np.float64) @ np.abs(k).T * scale, 0).max(1)
            most[:, g, 0] = np.abs(v).max(initial=0)
    return out, mean, big, np.asarray(last, dtype=np.float64).reshape(-1, 1, 1) + 1, most


def attend_bound(out, mean, big, keys, most, dim, dtype):
    """How far an output of the kernels may be from ``attend``'s, element by element.

    u is half a step of the element type.  The output is rounded once: u |o|.  Every probability is rounded once: u times
    sum p |v|.  Scores are sums of ``dim`` exact products in 32 bits: relative to sum |q k|, off by (dim + 8) 2^-24, which is
    the absolute error of an exponent and so the relative one of a probability, above and below the fraction line: twice.
    Sums over the keys: (keys + 64) 2^-24, twice (numerator, denominator); exponentials, scales, joins of splits: 2^-18.
    fp16 probabilities below 2^-14 lose 2^-25 each, against a sum of at least 1; outputs below 2^-14, 2^-25.
    bf16 and 32-bit numbers below 2^-126 may be taken as 0, so each of these loses less than 2^-126: a probability (against a
    sum of at least 1, since the maximum's own is at least 1 before the division), times |v|; a probability times the scale of
    int8 codes, times a code of at most 127; the output."""
    u = 2.0 ** -11 if dtype == "f16" else 2.0 ** -8
    rel = u + 2 * (dim + 8) * 2.0 ** -24 * big + 2 * (keys + 64) * 2.0 ** -24 + 2.0 ** -18
    tiny = 2.0 ** -25 * (1 + keys * most) if dtype == "f16" else 2.0 ** -126 * (1 + keys * (most + 127))
    return u * np.abs(out) + mean * rel + tiny
