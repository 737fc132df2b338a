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


# Launch shapes of chunk attention: rows of a row tile, and whether row tiles go out in pairs or in order of length.  Each takes
# more row tiles than small batches have.
EIGHT = dict(hq=32, hkv=32, chunks=[400, 300, 130, 390, 257, 65, 512, 128], prefixes=[0, 17, 5, 30, 0, 29, 1, 9])
FIVE = dict(hq=64, hkv=64, dim=64, chunks=[520, 257, 130, 65, 513], prefixes=[3, 17, 0, 30, 1])
WIDE = dict(hq=64, hkv=64, chunks=[520, 513, 257], prefixes=[3, 17, 0])
SORTED = dict(hq=64, hkv=64, chunks=[60, 520, 300], prefixes=[2000, 0, 40])
ALONE = dict(hq=64, hkv=64, chunks=[520, 300], prefixes=[0, 5])
SHAPES = {"128 rows in pairs": EIGHT, "128 rows of 64 dims in pairs": FIVE, "256 rows in pairs": WIDE, "256 rows by length": SORTED,
          "256 rows": ALONE}


def shaped(name, dtype, kind):
    """A batch of the shape, its cached codes drawn and not rounded from values: quick for many heads."""
    b = Batch(62, dtype=dtype, kind=kind, layers=1, layer=0, live="before", **SHAPES[name])
    top = 0x60 if kind == "e4m3" else 0x80                  # e4m3: up to 32, no NaN
    b.kc, b.vc = b.kc % top, b.vc % top
    for x in (b.kc, b.vc):
        x |= b.rng.integers(0, 2, x.shape, dtype=np.uint8) << 7
    b.scales = b.rng.integers(120, 125, b.scales.shape, dtype=np.uint8) - (0 if kind == "e4m3" else 2)
    return b


def check_shape(name, b, cuda):
    """The batch takes the launch shape that its name says, on this card."""
    units = torch.cuda.get_device_properties(cuda).multi_processor_count
    rows, per = max(b.chunks) * (b.hq // b.hkv), int(name.split()[0])
    columns = b.hkv * len(b.chunks)
    cells = columns * -(-rows // per)
    assert per == (256 if b.dim == 128 and rows > 512 and columns * -(-rows // 256) >= units else 128)
    by_length = cells > 2 * units and max(b.chunks) + max(b.prefixes) > 31 * 64
    assert by_length == ("by length" in name)
    assert ("in pairs" in name) == (not by_length and cells >= units * (2 if per == 256 else 4 if b.dim == 128 else 6))


@pytest.mark.parametrize("name,dtype", zip(SHAPES, itertools.cycle(("bf16", "f16"))))
def test_shapes(cuda, name, dtype):
    b = shaped(name, dtype, "int8")
    check_shape(name, b, cuda)
    q = b.new_rows(b.hq)
    assert_within(chunks(b, cuda, q), *b.expect_chunks(q))


@pytest.mark.parametrize("name,dtype", zip(SHAPES, itertools.cycle(("f16", "bf16"))))
def test_nan_reaches_the_rows_that_see_its_key(cuda, name, dtype):
    """In every launch shape: a NaN among V's codes is in its head dim of the rows at and behind its position, one among K's in
    every dim of them, and in no other row -- not in those of an earlier row tile that shares its key tile either."""
    b = shaped(name, dtype, "e4m3")
    check_shape(name, b, cuda)
    q = b.new_rows(b.hq)
    spoiled, codes = np.zeros(q.shape, dtype=bool), []
    for s, (n, p) in enumerate(zip(b.chunks, b.prefixes)):
        # around the ends of the row tiles, of key tiles and of the sequence
        spots = {0, p, p + n - 1, (p + n - 1) // 64 * 64, p + n // 2}
        spots |= {p + r + d for r in range(128, n, 128) for d in (-1, 0, 1, 30)}
        for i, pos in enumerate(sorted(x for x in spots if 0 <= x < p + n)):
            head, dim, in_k = (7 * i + 3 * s) % b.hq, (13 * i + 5 * s) % b.dim, i % 4 == 3
            pid = b.table[b.seq_ids[s], pos // K.B]
            array, at = (b.kc, (pid, 0, head, pos % K.B, dim)) if in_k else (b.vc, (pid, 0, head, dim, pos % K.B))
            array[at] = 0                                   # the rows that do not see it do not care
            codes.append((array, at, 0x7f if i % 2 else 0xff))
            first = int(b.starts[s]) + max(pos - p, 0)
            spoiled[first:int(b.starts[s]) + n, head, slice(None) if in_k else dim] = True
    want, bound = b.expect_chunks(q)
    for array, at, code in codes:
        array[at] = code
    got = chunks(b, cuda, q)
    wrong = np.argwhere(torch.isnan(got).cpu().numpy() != spoiled)
    assert not len(wrong), f"{len(wrong)} values, at {wrong[:4].tolist()}"
    got[torch.from_numpy(spoiled).to(cuda)] = 0
    assert_within(got, np.where(spoiled, 0, want), np.where(spoiled, 1, bound))


@pytest.mark.parametrize("dtype,kind", TYPES)
def test_the_same_call_gives_the_same_bits(cuda, dtype, kind):
    """Partials are joined in one order, whatever the order in which they were made."""
    b = Batch(64, hq=16, hkv=4, dtype=dtype, kind=kind, chunks=[200, 3, 65], prefixes=[900, 2000, 0], dec=[3000, 70, 1500])
    q, n = b.new_rows(b.hq), sum(b.chunks)
    first = chunks(b, cuda, q[:n]), decode(b, cuda, q[n:])
    for _ in range(10):
        assert torch.equal(chunks(b, cuda, q[:n]), first[0]) and torch.equal(decode(b, cuda, q[n:]), first[1])


def test_c_entries_with_descriptor_and_chosen_ranges(cuda):
    """A caller of the C entries takes the pool from ``KV8Cache.descriptor`` and the ranges from the package's rules: the bits
    of the Python calls."""
    import ctypes as C
    from morphserve_amd import _capi
    b = Batch(65, hq=8, hkv=2, chunks=[20, 3], prefixes=[900, 2000], dec=[3000, 70])
    q, n = b.new_rows(b.hq), sum(b.chunks)
    want = chunks(b, cuda, q[:n]), decode(b, cuda, q[n:])
    cache, table, st, prefix = b.cache(cuda), b.block_table(cuda), b.state(cuda), b.prefix_tensor(cuda)
    pool, units = cache.descriptor(), torch.cuda.get_device_properties(cuda).multi_processor_count
    batch = _capi.MkvBatch(table.data_ptr(), table.shape[1], table.shape[0], st.seq_ids.data_ptr(), st.prefill_seq_start_locs.data_ptr(),
                           st.prefill_seq_lens.data_ptr(), prefix.data_ptr(), st.decoding_seq_lens.data_ptr(), len(b.chunks), n,
                           st.max_prefill_len, len(b.dec))
    qg = rounded(q, "f16").to(cuda)
    o = torch.empty_like(qg)
    for entry, rows, split in (("mkv_attn8_prefill", slice(0, n), kv8.choose_prefill_split_8bit(2, 8, 2, 20, 20 + 2000, units, 128)),
                               ("mkv_attn8_decode", slice(n, b.tokens), kv8.choose_split_8bit(2, 2, 3000, units, 8, 128))):
        x, y = qg[rows], o[rows]
        mid = torch.empty(x.shape[0] * 8 * split[1], 128 + 1, dtype=torch.float32, device=cuda)
        assert split[1] > 1
        _capi.check(getattr(_capi.lib(), entry)(C.byref(pool), C.byref(batch), _capi.F16, x.data_ptr(), y.data_ptr(), 1024, 1024, 8, b.scale,
                                                b.layer, *split, mid.data_ptr(), mid.view(-1)[mid.shape[0] * 128:].data_ptr(),
                                                _capi.current_stream()))
    assert torch.equal(o[:n], want[0]) and torch.equal(o[n:], want[1])
