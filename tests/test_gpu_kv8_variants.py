"""The 8-bit cache's attention where its values are the smallest and the largest that a type has, and in the launch shapes that
small batches do not take; against ``oracle/kv8_cpu.py`` and its bound."""
import itertools

import numpy as np
import pytest
import torch

from kv8_helpers import Batch, assert_within, rounded
from oracle import kv8_cpu as K
from morphserve_amd import chunked_prefill_attention_8bit, paged_attention_8bit
from morphserve_amd.worker.kernels import kv8

pytestmark = pytest.mark.gpu

TYPES = list(itertools.product(("f16", "bf16"), ("e4m3", "int8")))


def chunks(b, cuda, q):
    qg = rounded(q, b.dtype).to(cuda)
    o = torch.full((sum(b.chunks), b.hq, b.dim), float("nan"), dtype=qg.dtype, device=cuda)
    chunked_prefill_attention_8bit(qg, b.cache(cuda), b.block_table(cuda), b.model, b.engine, b.state(cuda), b.layer, o,
                                   prefix_lens=b.prefix_tensor(cuda), max_prefix_len=max(b.prefixes))
    return o


def decode(b, cuda, q):
    qg = rounded(q, b.dtype).to(cuda)
    o = torch.full((len(b.dec), b.hq, b.dim), float("nan"), dtype=qg.dtype, device=cuda)
    paged_attention_8bit(qg, b.cache(cuda), b.block_table(cuda), b.model, b.engine, b.state(cuda), b.layer, o)
    return o


def set_values(b, make):
    """V of every position anew: ``make(rows)`` [rows, dim] for each block and head, codes and scale by the append's rule."""
    for s, total in zip(b.seq_ids, b.total):
        for j in range(-(-total // K.B)):
            n, pid = min(K.B, total - j * K.B), b.table[s, j]
            for h in range(b.hkv):
                slab, b.scales[b.layer, h, pid, 1] = K.join(b.vc[pid, b.layer, h].T, 0, make(n), 0, b.kind, b.dtype)
                b.vc[pid, b.layer, h] = slab.T


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_smallest_values(cuda, monkeypatch, dtype, kind, dim, splits):
    """V of multiples of 2^-24 only, fp16's smallest step: a block's scale goes down to 2^-30 (int8) or 2^-32 (e4m3)."""
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, splits))
    b = Batch(60, hq=4, hkv=2, dim=dim, dtype=dtype, kind=kind, chunks=[40, 70], prefixes=[30, 0], dec=[150, 7, 64])
    tops = iter(itertools.cycle((1, 2, 3, 4, 5)))
    set_values(b, lambda n: b.rng.integers(0, next(tops) + 1, (n, dim)) * b.rng.choice([-1, 1], (n, dim)) * 2.0 ** -24)
    q = b.new_rows(b.hq)
    n = sum(b.chunks)
    assert_within(chunks(b, cuda, q[:n]), *b.expect_chunks(q[:n]), "chunks")
    assert_within(decode(b, cuda, q[n:]), *b.expect_decode(q[n:]), "decode rows")


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_old_codes_behind_the_largest_values(cuda, monkeypatch, dtype, kind, splits):
    """Every old code behind a sequence's last position: at the scale of the type's largest values some of them (-128, 448)
    stand for more than the type holds, and they must not reach a row by way of a weight of 0."""
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, splits))
    b = Batch(61, hq=4, hkv=2, dtype=dtype, kind=kind, chunks=[40, 67, 5], prefixes=[30, 0, 128], dec=[150, 7, 70])
    # the largest that fp16 holds, and that 32-bit sums with weights up to 2^8 hold for bf16
    most = 61440.0 if dtype == "f16" else 2.0 ** 118
    set_values(b, lambda n: b.rng.choice([-1.0, 1.0, 0.5, 0.25], (n, b.dim)) * most)
    for s, total in zip(b.seq_ids, b.total):
        pid, last = b.table[s, (total - 1) // K.B], total % K.B
        if last:
            b.vc[pid, b.layer, :, :, last:] = b.rng.choice([0x80, 0x7e, 0xfe, 0x7f, 0xff], (b.hkv, b.dim, K.B - last))
    q = b.new_rows(b.hq)
    n = sum(b.chunks)
    assert_within(chunks(b, cuda, q[:n]), *b.expect_chunks(q[:n]), "chunks")
    assert_within(decode(b, cuda, q[n:]), *b.expect_decode(q[n:]), "decode rows")
