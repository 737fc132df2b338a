"""The 8-bit paged cache on the GPU against ``oracle/kv8_cpu.py`` (64 bits): appended codes and scales byte for byte over
the whole pool, attention within the bound that its roundings allow (``kv8_cpu.attend_bound``)."""
import itertools

import numpy as np
import pytest
import torch

from kv8_helpers import Batch, as_np, assert_cache, assert_within, rounded
from oracle import kv8_cpu as K
from morphserve_amd import (BlockManager, KV8Cache, allocate_kv8_cache, attention_section, chunked_prefill_attention_8bit,
                            paged_attention_8bit, rotary_embedding_and_store_kvcache_8bit, rotary_scaled_tables,
                            store_kvcache_8bit)
from morphserve_amd.worker.kernels import kv8

pytestmark = pytest.mark.gpu

TYPES = list(itertools.product(("f16", "bf16"), ("e4m3", "int8")))


def fused(batch, dev, *parts):
    """The parts as slices of one projection's rows, as a model has them."""
    x = rounded(np.concatenate(parts, axis=1), batch.dtype).to(dev)
    out, at = [], 0
    for p in parts:
        out.append(x[:, at:at + p.shape[1]])
        at += p.shape[1]
    return out


def run_store(b, cuda, k, v, layout=None, q=None, cos=None, sin=None, cache=None, **kw):
    cache = b.cache(cuda) if cache is None else cache
    prefix = b.prefix_tensor(cuda) if any(b.prefixes) else None
    if layout is None:
        kg, vg = fused(b, cuda, k, v)
        store_kvcache_8bit(kg, vg, cache, b.block_table(cuda), b.model, b.engine, b.state(cuda), b.layer, prefix_lens=prefix)
        return cache, None
    qg, kg, vg = fused(b, cuda, q, k, v)
    q_out = torch.full((b.tokens, b.hq, b.dim), 7.0, dtype=qg.dtype, device=cuda)
    tables = [torch.from_numpy(x).to(cuda) for x in (cos, sin)]
    rotary_embedding_and_store_kvcache_8bit(qg, kg, vg, *tables, cache, b.block_table(cuda), b.model, b.engine,
                                            b.state(cuda), b.layer, layout=layout, q_out=q_out, prefix_lens=prefix, **kw)
    assert np.array_equal(as_np(kg), k)                      # k itself stays
    return cache, q_out


MIXED = dict(chunks=[1, 15, 0, 16, 17, 40, 129, 3], prefixes=[0, 0, 7, 16, 5, 31, 100, 13], dec=[1, 16, 17, 0, 300, 33, 32])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_store(cuda, dtype, kind, dim):
    b = Batch(1, hkv=3, hq=3, dim=dim, dtype=dtype, kind=kind, live="before", **MIXED)
    k, v = b.new_rows(b.hkv), b.new_rows(b.hkv)
    cache, _ = run_store(b, cuda, k, v)
    K.store(b.kc, b.vc, b.scales, k, v, b.table, b.seq_ids, b.runs, b.layer, kind, dtype)
    assert_cache(cache, b)


@pytest.mark.parametrize("layout,dim,rotary", [("half", 128, 128), ("half", 128, 48), ("interleaved", 128, 128),
                                               ("interleaved", 64, 16), ("half", 64, 64), ("half", 64, 32)])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_rotary_store(cuda, dtype, kind, layout, dim, rotary):
    b = Batch(2, hkv=2, hq=6, dim=dim, dtype=dtype, kind=kind, live="before", **MIXED)
    q, k, v = b.new_rows(b.hq), b.new_rows(b.hkv), b.new_rows(b.hkv)
    cos, sin = (t.numpy() for t in rotary_scaled_tables(rotary, 400, 10000.0, None, "cpu"))
    cache, q_out = run_store(b, cuda, k, v, layout, q, cos, sin)
    # the codes follow from 32-bit products and sums, each rounded: the oracle does the same for them
    k32 = K.rotate(k, b.positions, cos, sin, layout, np.float32)
    K.store(b.kc, b.vc, b.scales, k32, v, b.table, b.seq_ids, b.runs, b.layer, kind, dtype)
    assert_cache(cache, b)
    # q: a row without a position is NaN in its rotated dims; the others are rounded once from three roundings of 32 bits
    want = K.rotate(q, b.positions, cos, sin, layout)
    size = K.rotate(np.abs(q), b.positions, np.abs(cos), -np.abs(sin), layout)
    size = np.maximum(np.abs(size), np.abs(K.rotate(np.abs(q), b.positions, np.abs(cos), np.abs(sin), layout)))
    half_step = 2.0 ** -11 if dtype == "f16" else 2.0 ** -8
    known = b.positions >= 0
    assert np.isnan(as_np(q_out)[~known][..., :rotary]).all()
    assert_within(q_out[torch.from_numpy(known).to(cuda)], want[known],
                  (half_step * np.abs(want) + 2.0 ** -22 * size + 2.0 ** -25)[known])


def test_rotary_store_in_place(cuda):
    b = Batch(3, hq=4, live="before", chunks=[20, 33], dec=[5, 40])
    q, k, v = b.new_rows(b.hq), b.new_rows(b.hkv), b.new_rows(b.hkv)
    cos, sin = rotary_scaled_tables(128, 64, device=cuda)
    _, q_out = run_store(b, cuda, k, v, "half", q, cos.cpu().numpy(), sin.cpu().numpy())
    qg, kg, vg = fused(b, cuda, q, k, v)
    cache = b.cache(cuda)
    rotary_embedding_and_store_kvcache_8bit(qg, kg, vg, cos, sin, cache, b.block_table(cuda), b.model, b.engine,
                                            b.state(cuda), b.layer)
    assert torch.equal(qg, q_out)


@pytest.mark.parametrize("dtype,kind", TYPES)
def test_store_of_extreme_values(cuda, dtype, kind):
    """Zeros, the type's smallest and largest, infinities and NaN."""
    b = Batch(4, dtype=dtype, kind=kind, live="before", chunks=[16, 16, 16, 5, 16], dec=[17, 1, 8, 32])
    k, v = b.new_rows(b.hkv), b.new_rows(b.hkv)
    fi = torch.finfo(torch.float16 if dtype == "f16" else torch.bfloat16)
    for x in (k, v):
        x[0:16] = 0
        x[16:32] = fi.smallest_normal * np.random.default_rng(0).integers(-3, 4, x[16:32].shape) / 4
        x[32:40] = fi.max
        x[40, 0, 3], x[41, 1, 5], x[42, 0, 0] = np.inf, -np.inf, np.nan
        x[-1, 0, 1], x[-2, 1, 2] = np.nan, -np.inf
    k, v = as_np(rounded(k, dtype)), as_np(rounded(v, dtype))
    cache, _ = run_store(b, cuda, k, v)
    K.store(b.kc, b.vc, b.scales, k, v, b.table, b.seq_ids, b.runs, b.layer, kind, dtype)
    assert_cache(cache, b)


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_token_by_token_raises_the_scale(cuda, kind):
    """One sequence grows token by token, now louder, now quieter; every step against the oracle."""
    b = Batch(5, kind=kind, live="before", dec=[1], spare=4)
    b.table[b.seq_ids[0], :3] = [0, 3, 1]
    cache = b.cache(cuda)
    for n in range(1, 40):
        b.dec = b.total = [n]
        loud = 2.0 ** b.rng.integers(-6, 7)
        k, v = as_np(rounded(b.rng.standard_normal((1, 2, 128)) * loud, "f16")), b.new_rows(2, 5)
        run_store(b, cuda, k, v, cache=cache)
        K.store(b.kc, b.vc, b.scales, k, v, b.table, b.seq_ids, b.runs, b.layer, kind, "f16")
        assert_cache(cache, b, f"token {n}")


def test_store_skips_what_has_no_place(cuda):
    """Table entries outside the pool, sequence ids outside the table, positions behind the table row and behind the
    rotary tables: nothing is written for them, and q of a row without an angle is NaN."""
    b = Batch(6, hq=2, live="before", chunks=[40, 20, 20, 90], prefixes=[0, 0, 3, 0], dec=[20, 33, 50, 7])
    b.table[b.seq_ids[0], 1] = -1
    b.table[b.seq_ids[1], 0] = b.n_blocks
    b.table[b.seq_ids[4], 1] = 2 ** 31 - 1
    b.seq_ids[2], b.seq_ids[5], b.seq_ids[7] = -1, b.rows, 2 ** 31 - 1
    b.table = np.ascontiguousarray(b.table[:, :4])           # the chunk of 90 rows has no place behind position 64
    q, k, v = b.new_rows(b.hq), b.new_rows(b.hkv), b.new_rows(b.hkv)
    cos, sin = (t.numpy() for t in rotary_scaled_tables(64, 45, device="cpu"))
    cache, q_out = run_store(b, cuda, k, v, "half", q, cos, sin)
    K.store(b.kc, b.vc, b.scales, K.rotate(k, b.positions, cos, sin, "half", np.float32), v, b.table, b.seq_ids, b.runs,
            b.layer, "e4m3", "f16", num_positions=45)
    assert_cache(cache, b)
    lost = torch.isnan(q_out).any(2).any(1).cpu().numpy()
    assert np.array_equal(lost, b.positions >= 45)


# ---- attention ----------------------------------------------------------------------------------------------------------
def decode(b, cuda, q, o=None, table=None):
    qg = rounded(q, b.dtype).to(cuda)
    o = torch.full((len(b.dec), b.hq * b.dim), float("nan"), dtype=qg.dtype, device=cuda) if o is None else o
    paged_attention_8bit(qg, b.cache(cuda), b.block_table(cuda), b.model, b.engine, b.state(cuda), b.layer, o)
    return o


EDGES = [0, 1, 2, 15, 16, 17, 31, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_decode_lengths(cuda, dtype, kind, dim):
    b = Batch(10, hq=8, hkv=2, dim=dim, dtype=dtype, kind=kind, dec=EDGES)
    q = b.new_rows(b.hq)
    want, bound = b.expect_decode(q)
    o = decode(b, cuda, q)
    assert_within(o, want, bound)
    assert not o[0].any()                                    # nothing to attend to


@pytest.mark.parametrize("group", range(1, 17))
def test_decode_groups(cuda, group):
    dtype, kind = TYPES[group % 4]
    b = Batch(11, hq=3 * group, hkv=3, dtype=dtype, kind=kind, dec=[77, 200, 5])
    q = b.new_rows(b.hq)
    assert_within(decode(b, cuda, q), *b.expect_decode(q))


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 40])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_decode_splits(cuda, monkeypatch, dtype, kind, splits):
    """The same lengths cut into few and many ranges, empty ones and a bound that is too small among them."""
    b = Batch(12, hq=6, hkv=2, dtype=dtype, kind=kind, dec=[1, 64, 130, 0, 700, 2600, 65])
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, splits))
    q = b.new_rows(b.hq)
    assert_within(decode(b, cuda, q), *b.expect_decode(q))


def test_decode_with_missing_blocks(cuda):
    """Blocks that the table does not name are not attended to; a sequence without any gets zeros."""
    for seed, (dtype, kind) in enumerate(TYPES):
        b = Batch(13 + seed, hq=4, hkv=2, dtype=dtype, kind=kind, dec=[100, 40, 200, 16, 90, 300])
        b.table[b.seq_ids[0], 1] = -1
        b.table[b.seq_ids[1], :] = [-1, b.n_blocks, 2 ** 31 - 1] + [-1] * (b.width - 3)
        b.table[b.seq_ids[2], :4] = -5
        b.table[b.seq_ids[5], 18] = b.n_blocks
        b.seq_ids[4] = b.rows
        q = b.new_rows(b.hq)
        want, bound = b.expect_decode(q)
        o = decode(b, cuda, q)
        assert_within(o, want, bound)
        assert not o[1].any() and not o[4].any()


def test_decode_of_scales_far_apart(cuda):
    """Blocks whose values differ by many orders of magnitude, within one tile and across tiles."""
    for dtype, kind in TYPES:
        b = Batch(20, hq=4, hkv=1, dtype=dtype, kind=kind, dec=[64, 200, 333])
        live = b.table[b.seq_ids[1], :13]
        far = 14 if dtype == "f16" else 40
        b.scales[b.layer, 0, live, 1] = 112 + b.rng.integers(-far, far // 2, len(live))
        b.scales[b.layer, 0, live, 0] = 112 + b.rng.integers(-far, 3, len(live))
        q = b.new_rows(b.hq)
        assert_within(decode(b, cuda, q), *b.expect_decode(q), f"{dtype} {kind}")


def test_decode_takes_rows_of_any_stride_and_leaves_the_rest(cuda):
    b = Batch(21, hq=8, hkv=2, chunks=[5, 9], dec=[33, 100, 64])
    q = b.new_rows(b.hq)
    want, bound = b.expect_decode(q[14:])
    wide = torch.full((17, 13, 128), 3.0, dtype=torch.float16, device=cuda)
    wide[:, 2:10] = rounded(q, "f16").to(cuda)
    o = torch.full((20, 1100), 5.0, dtype=torch.float16, device=cuda)
    paged_attention_8bit(wide[14:, 2:10], b.cache(cuda), b.block_table(cuda), b.model, b.engine, b.state(cuda), b.layer,
                         o[14:17, 8:1032])
    assert_within(o[14:17, 8:1032].unflatten(1, (8, 128)), want, bound)
    o[14:17, 8:1032] = 5.0
    assert (o == 5.0).all()


def test_far_blocks(cuda):
    """Block addresses beyond 2^32 bytes: append, decode and chunk attention there."""
    layers, heads, dim, blocks = 32, 8, 128, 9000            # 512 KiB a block: 4.4 GiB of K and of V
    b = Batch(22, hq=16, hkv=heads, chunks=[30], prefixes=[50], dec=[200, 17], layers=1, layer=0, live="before")
    cache = allocate_kv8_cache(blocks, (layers, heads, 16, dim), device=cuda)
    move = torch.arange(b.n_blocks, device=cuda) + (blocks - b.n_blocks)
    last = layers - 1
    cache.k[move, last] = torch.from_numpy(b.kc[:, 0]).to(cuda).view(cache.k.dtype)
    cache.v[move, last] = torch.from_numpy(b.vc[:, 0]).to(cuda).view(cache.k.dtype)
    cache.scales[last][:, move] = torch.from_numpy(b.scales[0]).to(cuda)
    table = b.block_table(cuda)
    table[table >= 0] += blocks - b.n_blocks
    b.model.num_layers = layers
    q, k, v = b.new_rows(b.hq), b.new_rows(heads), b.new_rows(heads)
    qg, kg, vg = fused(b, cuda, q, k, v)
    st, o = b.state(cuda), torch.empty(b.tokens, b.hq, dim, dtype=torch.float16, device=cuda)
    prefix = b.prefix_tensor(cuda)
    store_kvcache_8bit(kg, vg, cache, table, b.model, b.engine, st, last, prefix_lens=prefix)
    chunked_prefill_attention_8bit(qg[:30], cache, table, b.model, b.engine, st, last, o[:30], prefix_lens=prefix)
    paged_attention_8bit(qg[30:], cache, table, b.model, b.engine, st, last, o[30:])
    K.store(b.kc, b.vc, b.scales, k, v, b.table, b.seq_ids, b.runs, 0, "e4m3", "f16")
    assert np.array_equal(cache.k[move, last].view(torch.uint8).cpu().numpy(), b.kc[:, 0])
    assert np.array_equal(cache.v[move, last].view(torch.uint8).cpu().numpy(), b.vc[:, 0])
    assert_within(o[:30], *b.expect_chunks(q[:30]))
    assert_within(o[30:], *b.expect_decode(q[30:]))
    rest = torch.ones(blocks, dtype=torch.bool, device=cuda)
    rest[move] = False
    assert not cache.k.view(torch.uint8)[rest].any() and not cache.v.view(torch.uint8)[rest].any()


# ---- chunked prefill ---------------------------------------------------------------------------------------------------
def prefill(b, cuda, q, hint=True, prefix="given"):
    qg = rounded(q, b.dtype).to(cuda)
    o = torch.full((sum(b.chunks), b.hq, b.dim), float("nan"), dtype=qg.dtype, device=cuda)
    chunked_prefill_attention_8bit(qg, b.cache(cuda), b.block_table(cuda), b.model, b.engine, b.state(cuda), b.layer, o,
                                   prefix_lens=b.prefix_tensor(cuda) if prefix == "given" else None,
                                   max_prefix_len=max(b.prefixes) if hint else 0)
    return o


CHUNKS = dict(chunks=[1, 0, 15, 16, 17, 64, 65, 33, 130, 2], prefixes=[0, 9, 0, 0, 64, 1, 63, 200, 15, 500])


@pytest.mark.parametrize("hq,hkv", [(2, 2), (8, 2), (5, 1), (16, 1)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_chunks(cuda, dtype, kind, dim, hq, hkv):
    b = Batch(30, hq=hq, hkv=hkv, dim=dim, dtype=dtype, kind=kind, **CHUNKS)
    q = b.new_rows(b.hq)
    assert_within(prefill(b, cuda, q), *b.expect_chunks(q))


@pytest.mark.parametrize("splits", [1, 2, 5, 30])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_chunks_split_over_the_keys(cuda, monkeypatch, dtype, kind, splits):
    b = Batch(31, hq=6, hkv=2, dtype=dtype, kind=kind, **CHUNKS)
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, splits))
    q = b.new_rows(b.hq)
    assert_within(prefill(b, cuda, q), *b.expect_chunks(q))


@pytest.mark.parametrize("splits", [4, 5, 8, 9])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_rows_split_over_the_keys(cuda, monkeypatch, dim, splits):
    """Partials joined by a wave a row and by four, ranges without a key among them."""
    b = Batch(36, hq=16, hkv=4, dim=dim, dtype="bf16", chunks=[140, 3, 0, 131], prefixes=[100, 260, 30, 0])
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, splits))
    q = b.new_rows(b.hq)
    assert_within(prefill(b, cuda, q), *b.expect_chunks(q))


@pytest.mark.parametrize("hint", [True, False])
@pytest.mark.parametrize("seqs", [2, 70])
def test_row_tiles_in_order_of_length(cuda, seqs, hint):
    """More row tiles than fit the chip, of chunks that differ in length and prefix: they go out by length, and every one
    goes out (70 chunks: more than a wave has lanes)."""
    rng = np.random.default_rng(seqs)
    chunks = [300, 2100] if seqs == 2 else [int(x) for x in rng.integers(0, 40, seqs - 3)] + [150, 400, 33]
    prefixes = [2000, 0] if seqs == 2 else [int(x) for x in rng.integers(0, 90, seqs - 3)] + [2100, 30, 0]
    b = Batch(35, hq=16, hkv=16, dim=64, chunks=chunks, prefixes=prefixes, layers=1, layer=0)
    q = b.new_rows(b.hq)
    assert_within(prefill(b, cuda, q, hint=hint), *b.expect_chunks(q))


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,chunks", [(16, "short"), (64, [600, 513, 257])])
def test_several_rounds_of_row_tiles(cuda, heads, chunks, kind):
    """Enough row tiles for several rounds of workgroups, of chunks with one to five of them; prefixes that end inside a block."""
    rng = np.random.default_rng(38)
    chunks = [int(x) for x in rng.integers(0, 200, 40)] + [300, 129, 128, 1, 257] if chunks == "short" else chunks
    b = Batch(38, hq=heads, hkv=heads, dim=64, kind=kind, chunks=chunks, prefixes=[int(x) for x in rng.integers(0, 30, len(chunks))],
              layers=1, layer=0)
    q = b.new_rows(b.hq)
    assert_within(prefill(b, cuda, q), *b.expect_chunks(q))


@pytest.mark.parametrize("dtype,kind", [("f16", "e4m3"), ("bf16", "int8")])
@pytest.mark.parametrize("chunks,prefixes", [([600, 513, 257], [3, 17, 0]), ([60, 700, 520], [2000, 0, 40]), ([700, 300], [0, 5])])
def test_wide_row_tiles(cuda, dtype, kind, chunks, prefixes):
    """Row tiles of 256, 128 head dims: in pairs, in order of length, and as they come."""
    b = Batch(48, hq=64, hkv=64, dtype=dtype, kind=kind, chunks=chunks, prefixes=prefixes, layers=1, layer=0)
    q = b.new_rows(b.hq)
    assert_within(prefill(b, cuda, q), *b.expect_chunks(q))


@pytest.mark.parametrize("hq,hkv", [(4, 4), (8, 1)])
def test_whole_prompts(cuda, hq, hkv):
    b = Batch(32, hq=hq, hkv=hkv, chunks=[300, 1, 257, 512])
    q = b.new_rows(b.hq)
    assert_within(prefill(b, cuda, q, prefix=None), *b.expect_chunks(q))


def test_chunks_with_missing_blocks(cuda):
    for dtype, kind in TYPES:
        b = Batch(33, hq=4, hkv=2, dtype=dtype, kind=kind, chunks=[40, 20, 30, 25], prefixes=[100, 0, 70, 3])
        b.table[b.seq_ids[0], 0] = -1
        b.table[b.seq_ids[0], 5] = b.n_blocks
        b.table[b.seq_ids[1], :] = -1
        b.seq_ids[3] = -7
        q = b.new_rows(b.hq)
        want, bound = b.expect_chunks(q)
        o = prefill(b, cuda, q, hint=False)
        assert_within(o, want, bound)
        assert not o[40:60].any() and not o[90:].any()


@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("dtype,dim,hq", [("f16", 128, 4), ("bf16", 128, 16), ("f16", 64, 32), ("bf16", 64, 2)])
def test_nan_reaches_the_rows_that_see_its_key(cuda, monkeypatch, dtype, dim, hq, splits, which):
    """A NaN among the keys is in the sums of the rows at and behind its position, and in no other's: not through a weight of
    0 either.  K's spoils a row's whole head, V's the head dims that hold one."""
    b = Batch(37, hq=hq, hkv=2, dim=dim, dtype=dtype, chunks=[150, 20, 64, 5, 130], prefixes=[70, 3, 0, 300, 0], dec=[90, 40])
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, splits))
    q = b.new_rows(hq)
    n, group = sum(b.chunks), hq // 2
    first = b.prefixes + [0, 0]
    #       sequence, position, head, dim
    plant = [(0, 10, 0, 3), (0, 100, 1, 5), (0, 219, 0, dim - 1), (0, 130, 0, 17), (1, 12, 0, 0), (2, 63, 1, 7), (2, 1, 0, 9),
             (3, 304, 1, 33), (4, 64, 1, 2), (4, 65, 1, 2), (4, 127, 0, 50), (5, 89, 0, 1), (5, 20, 0, 21), (6, 39, 1, 4)]
    spoiled = np.zeros((b.tokens, hq, dim), dtype=bool)
    codes = []
    for i, (s, pos, h, d) in enumerate(plant):
        in_k = which == "k" or (which == "both" and i % 3 == 0)
        pid = b.table[b.seq_ids[s], pos // 16]
        at = (b.kc, (pid, b.layer, h, pos % 16, d)) if in_k else (b.vc, (pid, b.layer, h, d, pos % 16))
        at[0][at[1]] = 0                                    # the rows that do not see it do not care
        codes.append((at, 0x7f if i % 2 else 0xff))
        heads, dims = slice(h * group, (h + 1) * group), slice(None) if in_k else d
        if s < len(b.chunks):
            row0 = int(b.starts[s]) + max(pos - first[s], 0)
            spoiled[row0:int(b.starts[s]) + b.chunks[s], heads, dims] = True
        else:
            spoiled[n + s - len(b.chunks), heads, dims] = True
    want, bound = b.expect_chunks(q[:n])
    want_d, bound_d = b.expect_decode(q[n:])
    for (array, at), code in codes:
        array[at] = code
    got = torch.cat([prefill(b, cuda, q[:n]), decode(b, cuda, q[n:]).view(-1, hq, dim)])
    assert np.array_equal(torch.isnan(got).cpu().numpy(), spoiled)
    got[torch.from_numpy(spoiled).to(cuda)] = 0
    want, bound = np.concatenate([want, want_d]), np.concatenate([bound, bound_d])
    assert_within(got, np.where(spoiled, 0, want), np.where(spoiled, 1, bound))


@pytest.mark.parametrize("splits", [1, 3])
@pytest.mark.parametrize("dtype,kind", TYPES)
def test_infinite_rows_stay_their_own(cuda, monkeypatch, dtype, kind, splits):
    """A q row with an infinity or a NaN spoils its own head, not the rows that share its tile."""
    b = Batch(39, hq=8, hkv=2, dtype=dtype, kind=kind, chunks=[40, 90], prefixes=[100, 5], dec=[200, 30])
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, splits))
    q = b.new_rows(b.hq)
    n = sum(b.chunks)
    (want, bound), (want_d, bound_d) = b.expect_chunks(q[:n]), b.expect_decode(q[n:])
    want, bound = np.concatenate([want, want_d]), np.concatenate([bound, bound_d])
    bad = [(0, 3, np.nan), (17, 0, np.inf), (39, 7, -np.inf), (40, 1, np.nan), (129, 5, np.inf), (130, 2, np.nan), (131, 6, np.inf)]
    for row, head, x in bad:
        q[row, head, 11] = x
    got = torch.cat([prefill(b, cuda, q[:n]), decode(b, cuda, q[n:]).view(-1, b.hq, b.dim)])
    keep = np.ones((b.tokens, b.hq), dtype=bool)
    for row, head, x in bad:
        keep[row, head] = False
        if np.isnan(x):
            assert torch.isnan(got[row, head]).all()
    at = np.nonzero(keep)
    assert_within(got[torch.from_numpy(keep).to(cuda)], want[at], bound[at])


@pytest.mark.parametrize("splits", [1, 3])
def test_rows_of_no_chunk_stay(cuda, monkeypatch, splits):
    """Rows between and behind the chunks are neither read nor written."""
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, splits))
    b = Batch(34, hq=4, hkv=2, chunks=[20, 33], prefixes=[10, 100])
    q = b.new_rows(b.hq)
    want, bound = b.expect_chunks(q)
    st = b.state(cuda)
    st.num_prefill_tokens = 70
    st.prefill_seq_start_locs = torch.tensor([3, 30], dtype=torch.int32, device=cuda)
    qg = torch.full((70, 4, 128), float("nan"), dtype=torch.float16, device=cuda)
    o = torch.full((70, 4, 128), 2.0, dtype=torch.float16, device=cuda)
    qg[3:23], qg[30:63] = rounded(q[:20], "f16").to(cuda), rounded(q[20:], "f16").to(cuda)
    chunked_prefill_attention_8bit(qg, b.cache(cuda), b.block_table(cuda), b.model, b.engine, st, b.layer, o,
                                   prefix_lens=b.prefix_tensor(cuda), max_prefix_len=100)
    assert_within(torch.cat([o[3:23], o[30:63]]), want, bound)
    assert (o[:3] == 2).all() and (o[23:30] == 2).all() and (o[63:] == 2).all()


# ---- together -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,kind", TYPES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_serving_steps(cuda, dtype, kind, layout):
    """A batch lives through ``attention_section``: prompts in two chunks each, then decode steps, blocks from the
    BlockManager, the cache and the outputs against the oracle after every step."""
    hq, hkv, dim, layers, layer = 8, 2, 128, 2, 1
    b = Batch(40, hq=hq, hkv=hkv, dim=dim, dtype=dtype, kind=kind, layers=layers, layer=layer)
    n_blocks, rows, width = 64, 6, 12
    b.n_blocks = n_blocks
    b.kc = np.zeros((n_blocks, layers, hkv, 16, dim), dtype=np.uint8)
    b.vc = np.zeros((n_blocks, layers, hkv, dim, 16), dtype=np.uint8)
    b.scales = np.full((layers, hkv, n_blocks, 2), 127, dtype=np.uint8)
    cache = allocate_kv8_cache(n_blocks, (layers, hkv, 16, dim), b.cache(cuda).k.dtype, cuda)
    bm = BlockManager("GPU", n_blocks, rows, width, 16)
    cos, sin = rotary_scaled_tables(dim, 256, 500000.0, {"rope_type": "llama3", "factor": 8.0,
                                                          "original_max_position_embeddings": 128}, cuda)
    steps = [([37, 50], [0, 0], [0, 1], [], []), ([20, 9], [37, 50], [0, 1], [], []), ([33], [0], [2], [58, 60], [0, 1])]
    steps += [([], [], [], [58 + i, 60 + i, 33 + i], [0, 1, 2]) for i in range(1, 7)]
    for chunks, prefixes, chunk_ids, dec, dec_ids in steps:
        b.chunks, b.prefixes, b.dec = chunks, prefixes, dec
        b.tokens, b.seq_ids = sum(chunks) + len(dec), np.asarray(chunk_ids + dec_ids, dtype=np.int32)
        b.starts = np.concatenate([[0], np.cumsum(chunks)])[:len(chunks)].astype(np.int32)
        total = [p + n for p, n in zip(prefixes, chunks)] + dec
        bm.allocate_blocks_for_seqs(torch.tensor(b.seq_ids, device=cuda), torch.tensor(total, dtype=torch.int32, device=cuda))
        b.table = bm.block_table.cpu().numpy()
        q, k, v = b.new_rows(hq), b.new_rows(hkv), b.new_rows(hkv)
        qg, kg, vg = fused(b, cuda, q, k, v)
        o = torch.full((b.tokens, hq * dim), float("nan"), dtype=qg.dtype, device=cuda)
        attention_section(qg, kg, vg, o, cache, None, [], [], bm.block_table, b.model, b.engine, b.state(cuda), layer,
                          rotary_tables=(cos, sin), rotary_layout=layout,
                          prefix_lens=b.prefix_tensor(cuda) if any(prefixes) else None, max_prefix_len=max(prefixes + [0]))
        k32 = K.rotate(k, b.positions, cos.cpu().numpy(), sin.cpu().numpy(), layout, np.float32)
        K.store(b.kc, b.vc, b.scales, k32, v, b.table, b.seq_ids, b.runs, layer, kind, dtype)
        assert_cache(cache, b)
        q_rot = as_np(qg)                                    # rotated in place; its own test holds it to the formula
        p = sum(chunks)
        if p:
            assert_within(o[:p], *b.expect_chunks(q_rot[:p]), "chunks")
        if dec:
            assert_within(o[p:], *b.expect_decode(q_rot[p:]), "decode rows")


@pytest.mark.parametrize("side", [False, True])
def test_graph_and_other_stream(cuda, side):
    """Append, chunk and decode attention captured together and replayed over new rows; two graphs share nothing."""
    b = Batch(41, hq=8, hkv=2, live="before", chunks=[30, 5], prefixes=[0, 400], dec=[64, 900, 17])
    st, table, prefix = b.state(cuda), b.block_table(cuda), b.prefix_tensor(cuda)
    cache = b.cache(cuda)
    stream = torch.cuda.Stream()
    q = torch.empty(b.tokens, 8, 128, dtype=torch.float16, device=cuda)
    k, v = torch.empty(b.tokens, 2, 128, dtype=torch.float16, device=cuda), torch.empty(b.tokens, 2, 128, dtype=torch.float16, device=cuda)

    def step(o):
        store_kvcache_8bit(k, v, cache, table, b.model, b.engine, st, b.layer, prefix_lens=prefix)
        chunked_prefill_attention_8bit(q[:35], cache, table, b.model, b.engine, st, b.layer, o[:35], prefix_lens=prefix,
                                       max_prefix_len=400)
        paged_attention_8bit(q[35:], cache, table, b.model, b.engine, st, b.layer, o[35:])

    fill = lambda: [t.copy_(torch.randn(t.shape, device=cuda)) for t in (q, k, v)]  # noqa: E731
    outs = [torch.empty_like(q) for _ in range(3)]
    fill()
    step(outs[2])
    torch.cuda.synchronize()
    graphs = []
    for o in outs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream if side else None):
            step(o)
        graphs.append(graph)
    saved = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales)]
    for turn in range(4):
        fill()
        results = []
        for run in (graphs[0].replay, graphs[1].replay, lambda: step(outs[2])):
            for t, old in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales), saved):
                t.copy_(old)
            run()
            torch.cuda.synchronize()
            results.append([cache.k.view(torch.uint8).clone(), cache.v.view(torch.uint8).clone(), cache.scales.clone()])
        for got in results[:2]:
            assert all(torch.equal(x, y) for x, y in zip(got, results[2])), f"turn {turn}"
        assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[2]), f"turn {turn}"


def test_calls_on_two_streams_at_once(cuda):
    """Two batches over one cache, their split partials in flight at the same time."""
    b = Batch(42, hq=8, hkv=2, dec=[3000, 2500, 64])
    q = b.new_rows(b.hq)
    want, bound = b.expect_decode(q)
    cache, table, st = b.cache(cuda), b.block_table(cuda), b.state(cuda)
    qg = rounded(q, "f16").to(cuda)
    outs = [torch.empty_like(qg) for _ in range(8)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        with torch.cuda.stream(streams[i % 2]):
            paged_attention_8bit(qg, cache, table, b.model, b.engine, st, b.layer, o)
    torch.cuda.synchronize()
    for o in outs:
        assert_within(o, want, bound)
        assert torch.equal(o, outs[0])


def test_state_whose_tensors_are_made_at_every_access(cuda, monkeypatch):
    """The call's scratch must not take the memory of a tensor that only the call still holds."""
    b = Batch(45, hq=8, hkv=2, chunks=[70, 9], prefixes=[100, 0], dec=[3000, 2500, 64])
    kept = b.state(cuda)

    class State:
        def __getattr__(self, name):
            value = getattr(kept, name)
            return value.clone() if isinstance(value, torch.Tensor) else value

    monkeypatch.setattr(b, "state", lambda device: State())
    monkeypatch.setattr(kv8, "FORCED_SPLIT", (64, 2))       # partials of a few hundred bytes and more
    q = b.new_rows(b.hq)
    n = sum(b.chunks)
    want, bound = b.expect_decode(q[n:])
    assert_within(decode(b, cuda, q[n:]), want, bound)
    assert_within(prefill(b, cuda, q[:n]), *b.expect_chunks(q[:n]))


def test_negative_prefixes_count_as_none(cuda):
    b = Batch(46, hq=4, hkv=2, chunks=[20, 40], prefixes=[0, 0])
    q = b.new_rows(b.hq)
    want = prefill(b, cuda, q)
    b.prefixes = [-1, -(2 ** 31)]
    assert torch.equal(prefill(b, cuda, q, hint=False), want)
    results = []
    for prefixes in ([0, 0], b.prefixes):
        b.prefixes = prefixes
        cache, st = b.cache(cuda), b.state(cuda)
        k = rounded(q[:, :2], "f16").to(cuda)
        store_kvcache_8bit(k, k, cache, b.block_table(cuda), b.model, b.engine, st, b.layer, prefix_lens=b.prefix_tensor(cuda))
        results.append([cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.scales])
    assert all(torch.equal(x, y) for x, y in zip(*results))


def test_empty_calls(cuda):
    b = Batch(43, chunks=[], dec=[])
    st, cache, table = b.state(cuda), b.cache(cuda), torch.full((3, 2), -1, dtype=torch.int32, device=cuda)
    q, k = torch.empty(0, 8, 128, dtype=torch.float16, device=cuda), torch.empty(0, 2, 128, dtype=torch.float16, device=cuda)
    store_kvcache_8bit(k, k, cache, table, b.model, b.engine, st, 0)
    paged_attention_8bit(q, cache, table, b.model, b.engine, st, 0, q)
    chunked_prefill_attention_8bit(q, cache, table, b.model, b.engine, st, 0, q)
    torch.cuda.synchronize()
    assert_cache(cache, b)


def test_refusals(cuda):
    b = Batch(44, hq=8, hkv=2, chunks=[5], dec=[9])
    st, cache, table = b.state(cuda), b.cache(cuda), b.block_table(cuda)
    q = torch.zeros(6, 8, 128, dtype=torch.float16, device=cuda)
    k = torch.zeros(6, 2, 128, dtype=torch.float16, device=cuda)
    args = (table, b.model, b.engine, st, 0)
    before = cache.k.view(torch.uint8).clone()
    bad = [
        lambda: store_kvcache_8bit(k.float(), k.float(), cache, *args),
        lambda: store_kvcache_8bit(k, k.bfloat16(), cache, *args),
        lambda: store_kvcache_8bit(k[:5], k[:5], cache, *args),
        lambda: store_kvcache_8bit(k, k, cache, table.long(), *args[1:]),
        lambda: store_kvcache_8bit(k, k, cache, *args, prefix_lens=torch.zeros(0, dtype=torch.int32, device=cuda)),
        lambda: store_kvcache_8bit(k.cpu(), k.cpu(), cache, *args),
        lambda: store_kvcache_8bit(k.transpose(0, 1).contiguous().transpose(0, 1), k, cache, *args),
        lambda: paged_attention_8bit(q[:2], cache, *args, q[:2]),
        lambda: paged_attention_8bit(q[5:], cache, *args, q[5:].float()),
        lambda: paged_attention_8bit(q[5:], cache, *args, torch.zeros(1, 8, 64, dtype=torch.float16, device=cuda)),
        lambda: chunked_prefill_attention_8bit(q, cache, *args, q),
        lambda: chunked_prefill_attention_8bit(q[:5], cache, *args, q[0:1].expand(5, 8, 128)),
        lambda: attention_section(q, k, k, q.view(6, -1), cache, None, [], [], *args),       # no rotary tables
        lambda: attention_section(q, k, k, q.view(6, -1), cache, cache.k, [], [], *args, rotary=False),
        lambda: rotary_embedding_and_store_kvcache_8bit(q, k, k, *rotary_scaled_tables(128, 9, device=cuda), cache, *args,
                                                        layout="other"),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    from morphserve_amd._capi import MorphKVError
    bad = [
        lambda: store_kvcache_8bit(k, k, cache, *args[:4], 2),                                 # no such layer
        lambda: store_kvcache_8bit(torch.zeros(6 * 256 + 1, dtype=torch.float16, device=cuda)[1:].view(6, 2, 128), k, cache, *args),
        lambda: rotary_embedding_and_store_kvcache_8bit(q, k, k, *rotary_scaled_tables(24, 9, device=cuda), cache, *args),
        lambda: paged_attention_8bit(torch.zeros(8 * 128 + 1, dtype=torch.float16, device=cuda)[1:].view(1, 8, 128), cache, *args, q[5:]),
    ]
    for call in bad:
        with pytest.raises(MorphKVError):
            call()
    torch.cuda.synchronize()
    assert torch.equal(before, cache.k.view(torch.uint8))
    assert isinstance(cache, KV8Cache)
