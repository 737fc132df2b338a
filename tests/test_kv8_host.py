"""CPU checks around the 8-bit cache and the rotary forms: the oracle itself, table scaling, and that bad arguments are
refused before anything is launched."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from oracle import kv8_cpu as K
from morphserve_amd import KV8Cache, _capi, allocate_kv8_cache, rotary_embedding, rotary_scaled_tables
from morphserve_amd.worker.kernels import kv8


# ---- the oracle ---------------------------------------------------------------------------------------------------------
def test_codes_round_to_nearest_even():
    grid = K.E4M3[:127]
    assert grid[-1] == 448 and grid[1] == 2.0 ** -9 and (np.diff(grid) > 0).all()
    x = np.concatenate([grid, (grid[1:] + grid[:-1]) / 2, np.random.default_rng(0).uniform(0, 448, 5000)])
    x = np.concatenate([x, -x]).astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(K.encode(x, "e4m3"), want)
    assert np.array_equal(K.decode(K.encode(grid, "e4m3"), "e4m3"), grid)
    assert K.encode(np.asarray([0.5, 1.5, -2.5, 127, -127, np.nan]), "int8").view(np.int8).tolist() == [0, 2, -2, 127, -127, 0]


@pytest.mark.parametrize("kind", ["e4m3", "int8"])
def test_exponents_and_joins(kind):
    top = K.QMAX[kind]
    for e in (1, 5, 120, 130):
        edge = top * 2.0 ** (e - 127)
        assert K.exponent(edge, kind) == e and K.exponent(np.nextafter(edge, np.inf), kind) == e + 1
    assert K.exponent(0.0, kind) == 1
    rng = np.random.default_rng(1)
    slab, scale = rng.integers(0, 256, (16, 8), dtype=np.uint8), 200
    rows = rng.standard_normal((6, 8))
    slab, scale = K.join(slab, scale, rows[:4], 0, kind, "f16")              # a fresh block forgets its old scale
    kept = slab.copy()
    step = 2.0 ** (scale - 127) * (0.5 if kind == "int8" else 16)            # half a step of the largest codes
    assert np.abs(K.decode(slab[:4], kind) * 2.0 ** (scale - 127) - rows[:4]).max() <= step
    slab, louder = K.join(slab, scale, rows[4:] * 64, 4, kind, "f16")
    assert louder > scale and np.array_equal(slab[6:], kept[6:])
    step = 2.0 ** (louder - 127) * (0.5 if kind == "int8" else 16)
    assert np.abs(K.decode(slab[:4], kind) * 2.0 ** (louder - 127) - rows[:4]).max() <= 2 * step
    again, same = K.join(slab, louder, rows[4:] / 64, 6, kind, "f16")        # a quieter row does not lower it
    assert same == louder and np.array_equal(again[:6], slab[:6])


def test_attention_of_the_oracle():
    """One block, equal keys: the mean of the values; a mask: the first value; against softmax in torch."""
    rng = np.random.default_rng(2)
    kc, vc = np.zeros((2, 1, 1, 16, 64), dtype=np.uint8), np.zeros((2, 1, 1, 64, 16), dtype=np.uint8)
    scales = np.full((1, 1, 2, 2), 127, dtype=np.uint8)
    v = rng.standard_normal((20, 1, 64))
    table, ids = np.asarray([[1, 0]], dtype=np.int32), [0]
    K.store(kc, vc, scales, np.zeros((20, 1, 64)), v, table, ids, [(0, 0, 0, 20)], 0, "int8", "f16")
    _, vals, _ = K.gather(kc, vc, scales, table[0], 20, 0, 0, "int8")
    assert np.abs(vals - v[:, 0]).max() <= 2.0 ** -6
    q = rng.standard_normal((2, 3, 64))
    o = K.attend(q, kc, vc, scales, table, 0, [0, 19], 0, "int8", 0.125)[0]
    assert np.allclose(o[0], vals[0]) and np.allclose(o[1], vals.mean(0))
    K.store(kc, vc, scales, rng.standard_normal((20, 1, 64)), v, table, ids, [(0, 0, 0, 20)], 0, "e4m3", "f16")
    k, vals, _ = K.gather(kc, vc, scales, table[0], 20, 0, 0, "e4m3")
    want = torch.softmax(torch.from_numpy(q[1] @ k.T * 0.125), -1).numpy() @ vals
    assert np.allclose(K.attend(q, kc, vc, scales, table, 0, [0, 19], 0, "e4m3", 0.125)[0][1], want)


def test_rotation_of_the_oracle():
    x = np.random.default_rng(3).standard_normal((4, 2, 10))
    cos, sin = (t.numpy() for t in rotary_scaled_tables(6, 9, 100.0, device="cpu"))
    for layout in ("half", "interleaved"):
        y = K.rotate(x, [0, 1, 5, 8], cos, sin, layout)
        assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 6:], x[..., 6:])
        assert np.allclose((y ** 2).sum(-1), (x ** 2).sum(-1))                              # a rotation keeps lengths
    pair = K.rotate(np.asarray([[[1.0, 0.0]]]), [1], np.cos([[0.0], [0.3]]), np.sin([[0.0], [0.3]]), "half")[0, 0]
    assert np.allclose(pair, [math.cos(0.3), math.sin(0.3)])


# ---- rotary tables ------------------------------------------------------------------------------------------------------
def test_table_scalings():
    d, theta, n = 32, 10000.0, 64
    inv = theta ** (-np.arange(0, d, 2) / d)
    angle = lambda t: np.arctan2(t[1].double().numpy(), t[0].double().numpy())  # noqa: E731
    assert np.allclose(angle(rotary_scaled_tables(d, n, theta, None, "cpu"))[1], inv, atol=1e-7)
    for same in ({}, {"rope_type": "default"}, {"type": "default"}, 1.0):
        assert torch.equal(rotary_scaled_tables(d, n, theta, same, "cpu")[1], rotary_scaled_tables(d, n, theta, None, "cpu")[1])
    assert np.allclose(angle(rotary_scaled_tables(d, n, theta, 4.0, "cpu"))[1], inv / 4, atol=1e-7)
    assert np.allclose(angle(rotary_scaled_tables(d, n, theta, {"type": "linear", "factor": 4}, "cpu"))[1], inv / 4, atol=1e-7)
    # dynamic: untouched up to the trained length, the slowest pair slowed by the growth beyond it
    dyn = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 32}
    assert np.allclose(angle(rotary_scaled_tables(d, 32, theta, dyn, "cpu"))[1], inv, atol=1e-7)
    grown = 2.0 * 64 / 32 - 1
    assert np.allclose(angle(rotary_scaled_tables(d, 64, theta, dyn, "cpu"))[1][[0, -1]], [inv[0], inv[-1] / grown], atol=1e-7)
    # llama3: pairs that turn fast kept, slow ones divided
    l3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 256}
    got, turns = angle(rotary_scaled_tables(d, n, theta, l3, "cpu"))[1], 256 * inv / (2 * np.pi)
    assert np.allclose(got[turns > 4], inv[turns > 4], atol=1e-7) and np.allclose(got[turns < 1], inv[turns < 1] / 8, atol=1e-7)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and (got[mid] < inv[mid]).all() and (got[mid] > inv[mid] / 8).all()
    # yarn: the same ends, and cosines scaled
    yarn = {"rope_type": "yarn", "factor": 8.0, "original_max_position_embeddings": 1024}
    cos, sin = rotary_scaled_tables(d, n, theta, yarn, "cpu")
    assert cos[0, 0].item() == pytest.approx(0.1 * math.log(8) + 1)
    got = angle((cos, sin))[1]
    assert got[0] == pytest.approx(inv[0], abs=1e-6) and got[-1] == pytest.approx(inv[-1] / 8, rel=1e-4)
    assert rotary_scaled_tables(d, n, theta, {**yarn, "attention_factor": 1.0}, "cpu")[0][0, 0] == 1


def yarn_by_hand(dim, theta, factor, old, fast=32.0, slow=1.0, truncate=True):
    """Angles of position 1, pair by pair: a pair that turns more than ``fast`` times over the trained length is kept, one that
    turns less than ``slow`` times divided by the factor, and between them goes a ramp over the pairs' numbers."""
    border = [dim * math.log(old / (turns * 2 * math.pi)) / (2 * math.log(theta)) for turns in (fast, slow)]
    lo, hi = (math.floor(border[0]), math.ceil(border[1])) if truncate else border
    lo, hi = max(lo, 0), min(hi, dim - 1)
    angles = []
    for i in range(dim // 2):
        plain, part = theta ** (-2 * i / dim), min(max((i - lo) / (hi - lo), 0), 1)
        angles.append(plain * (1 - part) + plain / factor * part)
    return np.asarray(angles)


def angles_of(tables):
    return np.arctan2(tables[1].double().numpy(), tables[0].double().numpy())[1]


@pytest.mark.parametrize("scales,want", [
    (dict(mscale=1.0, mscale_all_dim=1.0), 1.0), (dict(mscale=0.707, mscale_all_dim=0.707), 1.0),
    (dict(mscale=1.0), 0.1 * math.log(40) + 1), (dict(mscale_all_dim=0), 0.1 * math.log(40) + 1),
    (dict(mscale=0.5, mscale_all_dim=2.0), (0.05 * math.log(40) + 1) / (0.2 * math.log(40) + 1)),
    (dict(mscale=0.5, mscale_all_dim=2.0, attention_factor=1.25), 1.25)])
def test_yarn_with_two_scales(scales, want):
    """64 rotary dims, 4096 trained positions, a factor of 40: the cosines' and sines' factor is the ratio of the two scales."""
    config = {"rope_type": "yarn", "factor": 40, "original_max_position_embeddings": 4096, "beta_fast": 32, "beta_slow": 1, **scales}
    tables = rotary_scaled_tables(64, 8, 10000.0, config, "cpu")
    size = torch.hypot(tables[0].double(), tables[1].double())
    assert np.allclose(size.numpy(), want, rtol=2.0 ** -22)
    assert np.allclose(angles_of(tables), yarn_by_hand(64, 10000.0, 40, 4096), rtol=2.0 ** -22, atol=0)


@pytest.mark.parametrize("truncate", [True, False, None])
@pytest.mark.parametrize("dim,theta,factor,old", [(64, 150000.0, 32, 4096), (128, 1e6, 4, 32768), (32, 10000.0, 8, 1024)])
def test_yarn_ramp_with_and_without_whole_ends(dim, theta, factor, old, truncate):
    config = {"rope_type": "yarn", "factor": factor, "original_max_position_embeddings": old}
    if truncate is not None:
        config["truncate"] = truncate
    got = angles_of(rotary_scaled_tables(dim, 8, theta, config, "cpu"))
    want, other = (yarn_by_hand(dim, theta, factor, old, truncate=t) for t in (truncate is not False, truncate is False))
    assert np.allclose(got, want, rtol=2.0 ** -22, atol=0) and not np.allclose(got, other, rtol=1e-3, atol=0)


@pytest.mark.parametrize("args", [(7, 4), (0, 4), (8, 4, 1e4, {"rope_type": "linear", "factor": 0.5}), (8, 4, 1e4, {"rope_type": "odd", "factor": 2, "original_max_position_embeddings": 8}),
                                  (8, 4, 1e4, {"rope_type": "yarn", "factor": 2}), (2, 4, 1e4, {"rope_type": "dynamic", "factor": 2, "original_max_position_embeddings": 8}),
                                  (8, 4, 1e4, {"rope_type": "llama3", "factor": 2, "low_freq_factor": 4, "high_freq_factor": 4, "original_max_position_embeddings": 8})])
def test_table_refusals(args):
    with pytest.raises(ValueError):
        rotary_scaled_tables(*args, device="cpu")


@pytest.mark.parametrize("scaling", [
    {"rope_type": "longrope"}, {"type": "su", "factor": 4}, {"rope_type": "default", "type": "linear", "factor": 2},
    {"rope_type": "linear"}, {"rope_type": "linear", "factor": None}, {"rope_type": "linear", "factor": "two"},
    {"rope_type": "linear", "factor": math.nan}, {"rope_type": "linear", "factor": math.inf}, math.nan, "two",
    {"rope_type": "dynamic", "factor": 2}, {"rope_type": "llama3", "factor": 2, "original_max_position_embeddings": None},
    {"rope_type": "yarn", "original_max_position_embeddings": 64},
    {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": -64},
    {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 64, "beta_fast": 1, "beta_slow": 32},
    {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 64, "beta_slow": 0},
    {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 64, "truncate": "no"},
    {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 64, "attention_factor": "big"},
    {"rope_type": "yarn", "factor": 2, "original_max_position_embeddings": 64, "low_freq_factor": 1},
    {"rope_type": "linear", "factor": 2, "mscale": 1.0}, {"rope_type": "default", "factor": 2},
    {"rope_type": "default", "mrope_section": [16, 24, 24]}, {"nonsense": 3}, {"rope_type": "linear", "factor": 2, "rope_theta": 5e5},
    {"rope_type": ["linear"], "factor": 2}])
def test_scalings_that_are_refused(scaling):
    """Rules and keys that are not known, and values that are no numbers: a table made without them would be a wrong one."""
    with pytest.raises(ValueError):
        rotary_scaled_tables(32, 4, 1e4, scaling, "cpu")


@pytest.mark.parametrize("args", [(32, -1), (32, 4, 0.0), (32, 4, math.nan), (32, 4, 1.0, {"type": "yarn", "factor": 2, "original_max_position_embeddings": 64})])
def test_bases_and_lengths_that_are_refused(args):
    with pytest.raises(ValueError):
        rotary_scaled_tables(*args, device="cpu")


def test_keys_that_say_nothing_of_the_angles():
    plain = rotary_scaled_tables(32, 40, 5e5, {"type": "linear", "factor": 2}, "cpu")
    same = {"rope_type": "linear", "type": "linear", "factor": 2.0, "rope_theta": 5e5, "original_max_position_embeddings": 64,
            "finetuned": True, "partial_rotary_factor": 0.5}
    assert all(torch.equal(x, y) for x, y in zip(plain, rotary_scaled_tables(32, 40, 5e5, same, "cpu")))
    yarn = {"type": "yarn", "factor": 4, "original_max_position_embeddings": 64}
    none = dict.fromkeys(("rope_type", "beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate"))
    for x, y in zip(rotary_scaled_tables(32, 40, 5e5, yarn, "cpu"), rotary_scaled_tables(32, 40, 5e5, {**yarn, **none}, "cpu")):
        assert torch.equal(x, y)


# ---- the cache object -----------------------------------------------------------------------------------------------------
def test_cache_object():
    cache = allocate_kv8_cache(5, (2, 3, 16, 64), torch.int8, "cpu")
    pool = cache.descriptor()
    assert (pool.num_blocks, pool.num_layers, pool.num_kv_heads, pool.block_size, pool.head_dim, pool.kind) == (5, 2, 3, 16, 64, 1)
    assert (pool.k, pool.v, pool.scales) == tuple(t.data_ptr() for t in (cache.k, cache.v, cache.scales)) and cache.num_blocks == 5
    k, v, s = cache.k, cache.v, cache.scales
    for bad in ((k.half(), v.half(), s), (k, v.view(torch.uint8), s), (k, k, s), (k, v, s[:1]), (k, v, s.int()),
                (k[:, :, :, :, :32], v[:, :, :, :32], s), (k[:0], v[:0], s[:, :, :0]), (k[0], v[0], s), (k[::2], v[::2], s[:, :, ::2])):
        with pytest.raises(ValueError):
            KV8Cache(*bad).descriptor()
    with pytest.raises(ValueError):
        allocate_kv8_cache(5, (2, 3, 16, 64), torch.float16, "cpu")


def test_split_rules():
    for n, heads, longest in ((1, 1, 1), (1, 8, 100), (5, 8, 60000), (64, 8, 1536), (300, 32, 70), (1, 1, 10 ** 6)):
        tps, splits = kv8.choose_split_8bit(n, heads, longest, 512)
        assert tps % 64 == 0 and splits >= 1 and tps * splits >= longest and tps * (splits - 1) < longest
    for seqs, hq, hkv, rows, keys in ((1, 8, 8, 1, 1), (6, 64, 8, 16, 16000), (8, 32, 32, 512, 512), (1, 1, 1, 10 ** 5, 10 ** 5)):
        tps, splits = kv8.choose_prefill_split_8bit(seqs, hq, hkv, rows, keys, 512)
        assert tps % 64 == 0 and splits >= 1 and tps * splits >= keys and tps * (splits - 1) < keys


# ---- refusals of the C entries: none of these calls reaches a launch ---------------------------------------------------
A = 1 << 20          # an address that is never followed


def pool8(**kw):
    p = _capi.MkvPool8(A, A, A, 10, 2, 4, 16, 128, 0, 0)
    for name, value in kw.items():
        setattr(p, name, value)
    return p


def batch8(**kw):
    b = _capi.MkvBatch(A, 8, 4, A, A, A, A, A, 1, 5, 5, 1)
    for name, value in kw.items():
        setattr(b, name, value)
    return b


def store(p=None, b=None, dtype=0, k=A, v=A, ks=512, vs=512, layer=0, rope=0, q=A, qo=A, qs=512, qos=512, hq=4, cos=A, sin=A,
          positions=9, rotary=32):
    p, b = pool8() if p is None else p, batch8() if b is None else b
    return _capi.lib().mkv_store8(C.byref(p), C.byref(b), dtype, k, v, ks, vs, layer, rope, q, qo, qs, qos, hq, cos, sin,
                                  positions, rotary, None)


def attn(entry, p=None, b=None, dtype=0, q=A, o=A, qs=1024, os_=1024, hq=8, layer=0, tps=64, splits=2, mid_o=A, lse=A):
    p, b = pool8() if p is None else p, batch8() if b is None else b
    return getattr(_capi.lib(), entry)(C.byref(p), C.byref(b), dtype, q, o, qs, os_, hq, 0.1, layer, tps, splits, mid_o, lse, None)


BAD_POOLS = [dict(k=None), dict(v=None), dict(scales=None), dict(num_layers=0), dict(num_kv_heads=0), dict(block_size=32),
             dict(head_dim=96), dict(kind=2), dict(num_blocks=0), dict(num_blocks=2 ** 31), dict(k=A + 8), dict(v=A + 1), dict(scales=A + 1)]
BAD_BATCHES = [dict(block_table=None), dict(seq_ids=None), dict(max_blocks_per_seq=-1), dict(max_blocks_per_seq=2 ** 27),
               dict(table_rows=-1), dict(num_prefill_seqs=-1), dict(num_decoding_seqs=-1), dict(max_prefill_len=-1)]


@pytest.mark.parametrize("entry", ["store", "mkv_attn8_decode", "mkv_attn8_prefill"])
def test_bad_pools_and_batches(entry):
    call = store if entry == "store" else lambda **kw: attn(entry, **kw)
    for bad in BAD_POOLS:
        assert call(p=pool8(**bad)) == _capi.MKV_EINVAL, bad
    for bad in BAD_BATCHES:
        assert call(b=batch8(**bad)) == _capi.MKV_EINVAL, bad
    assert call(dtype=2) == _capi.MKV_EINVAL and call(layer=2) == _capi.MKV_EINVAL and call(layer=-1) == _capi.MKV_EINVAL
    lib = _capi.lib()
    assert lib.mkv_store8(None, None, 0, A, A, 0, 0, 0, 0, None, None, 0, 0, 0, None, None, 0, 0, None) == _capi.MKV_EINVAL
    assert call(b=batch8(num_prefill_seqs=0, num_decoding_seqs=0)) == _capi.MKV_OK          # nothing to do


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(k=A + 8), dict(vs=516), dict(rope=3), dict(b=batch8(decoding_lens=None)),
                                 dict(b=batch8(prefill_lens=None)), dict(rope=1, q=None), dict(rope=1, cos=None), dict(rope=1, rotary=24),
                                 dict(rope=2, rotary=0), dict(rope=1, rotary=144), dict(rope=1, hq=0), dict(rope=1, q=A + 2),
                                 dict(rope=1, qs=513), dict(rope=1, sin=A + 4), dict(rope=1, positions=-1), dict(rope=1, positions=0), dict(rope=1, qos=1024)])
def test_bad_store(bad):
    assert store(**bad) == _capi.MKV_EINVAL
    assert _capi.lib().mkv_last_error()


@pytest.mark.parametrize("entry", ["mkv_attn8_decode", "mkv_attn8_prefill"])
@pytest.mark.parametrize("bad", [dict(q=None), dict(o=None), dict(hq=0), dict(hq=6), dict(hq=68), dict(tps=0), dict(tps=96), dict(splits=0),
                                 dict(mid_o=None), dict(lse=None), dict(mid_o=A + 4), dict(q=A + 2), dict(qs=1028)])
def test_bad_attention(entry, bad):
    assert attn(entry, **bad) == _capi.MKV_EINVAL


@pytest.mark.parametrize("entry", ["mkv_attn8_decode", "mkv_attn8_prefill"])
@pytest.mark.parametrize("tps,splits", [(2 ** 30, 16), (2 ** 31 - 64, 5), (2 ** 20, 2 ** 14), (64, 2 ** 28)])
def test_ranges_whose_ends_have_no_32_bit_number(entry, tps, splits):
    assert attn(entry, tps=tps, splits=splits) == _capi.MKV_EINVAL
    assert b"ranges" in _capi.lib().mkv_last_error()


def test_launches_too_large():
    """2^32 threads and more in one launch."""
    many = dict(num_prefill_seqs=2000, max_prefill_len=2 ** 17)
    assert store(b=batch8(**many)) == _capi.MKV_EINVAL and b"too many rows" in _capi.lib().mkv_last_error()
    assert attn("mkv_attn8_prefill", b=batch8(num_prefill_seqs=60000, max_prefill_len=2 ** 20)) == _capi.MKV_EINVAL
    assert b"too many rows" in _capi.lib().mkv_last_error()
    assert attn("mkv_attn8_prefill", b=batch8(num_prefill_seqs=1, max_prefill_len=2 ** 22)) == _capi.MKV_EINVAL
    assert attn("mkv_attn8_decode", b=batch8(num_decoding_seqs=65536)) == _capi.MKV_EINVAL
    assert attn("mkv_attn8_decode", p=pool8(num_kv_heads=64), hq=1024, b=batch8(num_decoding_seqs=40000)) == _capi.MKV_EINVAL


@pytest.mark.parametrize("bad", [dict(dtype=5), dict(layout=0), dict(layout=3), dict(tokens=-1), dict(hq=0), dict(hkv=-1), dict(rotary=7),
                                 dict(rotary=0), dict(rotary=66), dict(q=None), dict(k=None), dict(pos=None), dict(cos=None),
                                 dict(positions=-1), dict(qs=100), dict(dim=0), dict(qos=512), dict(kos=256)])
def test_bad_rotary(bad):
    a = dict(dtype=0, layout=1, q=A, k=A, qo=A, ko=A, qs=256, ks=128, qos=256, kos=128, pos=A, cos=A, sin=A, positions=9, tokens=3,
             hq=4, hkv=2, dim=64, rotary=32)
    a.update(bad)
    assert _capi.lib().mkv_rope_positions(*[a[x] for x in ("dtype", "layout", "q", "k", "qo", "ko", "qs", "ks", "qos", "kos", "pos", "cos",
                                                            "sin", "positions", "tokens", "hq", "hkv", "dim", "rotary")], None) == _capi.MKV_EINVAL


def test_rows_on_the_cpu_are_refused():
    cos, sin = rotary_scaled_tables(32, 4, device="cpu")
    with pytest.raises(ValueError):
        rotary_embedding(torch.zeros(2, 2, 64, dtype=torch.float16), None, torch.zeros(2, dtype=torch.int32), cos, sin)


# ---- the attention section ------------------------------------------------------------------------------------------------
def section(monkeypatch, **change):
    """``attention_section`` over an 8-bit cache on the CPU, its launches recorded instead of made: what was launched."""
    from helpers import Cfg
    from morphserve_amd.worker.layers import transformer_layer as layer
    calls = []
    for name in ("store_kvcache_8bit", "rotary_embedding_and_store_kvcache_8bit", "chunked_prefill_attention_8bit", "paged_attention_8bit"):
        monkeypatch.setattr(layer, name, lambda *a, _name=name, **kw: calls.append(_name))
    cache = allocate_kv8_cache(4, (1, 2, 16, 64), device="cpu")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    a = dict(q=torch.zeros(6, 4, 64, dtype=torch.float16), o=torch.zeros(6, 256, dtype=torch.float16), heads=4, softmax_scale=0.125,
             max_prefix_len=0, prefill=5, dec=1)
    a.update(change)
    k = torch.zeros(6, 2, 64, dtype=torch.float16)
    st = Cfg(seq_ids=i32(0, 1), num_prefill_seqs=1, num_prefill_tokens=a["prefill"], prefill_seq_start_locs=i32(0), prefill_seq_lens=i32(5),
             max_prefill_len=5, num_decoding_seqs=a["dec"], decoding_seq_lens=i32(3), max_decoding_len=3, softmax_scale=a["softmax_scale"])
    model = Cfg(num_layers=1, num_q_heads=a["heads"], num_kv_heads=2, head_dim=64)
    tables = rotary_scaled_tables(64, 8, device="cpu")
    try:
        layer.attention_section(a["q"], k, k, a["o"], cache, None, [], [], torch.zeros(2, 2, dtype=torch.int32), model,
                                Cfg(block_size=16, max_blocks_per_seq=2), st, 0, rotary_tables=tables, max_prefix_len=a["max_prefix_len"])
    except ValueError:
        return "refused" if not calls else calls
    return calls


def test_section_launches(monkeypatch):
    want = ["rotary_embedding_and_store_kvcache_8bit", "chunked_prefill_attention_8bit", "paged_attention_8bit"]
    assert section(monkeypatch) == want
    assert section(monkeypatch, o=torch.zeros(6, 4, 64, dtype=torch.float16)) == want
    assert section(monkeypatch, q=torch.zeros(6, 8, 64, dtype=torch.float16)[:, 2:6], o=torch.zeros(6, 300, dtype=torch.float16)[:, 8:264][:, :256]) == "refused"
    assert section(monkeypatch, o=torch.zeros(6, 304, dtype=torch.float16)[:, 8:264]) == want


@pytest.mark.parametrize("change", [
    dict(o=torch.zeros(5, 256, dtype=torch.float16)), dict(o=torch.zeros(6, 255, dtype=torch.float16)), dict(o=torch.zeros(6, 256)),
    dict(o=torch.zeros(6, 512, dtype=torch.float16)[:, ::2]), dict(o=torch.zeros(1, 256, dtype=torch.float16).expand(6, 256)),
    dict(o=torch.zeros(6 * 256 + 1, dtype=torch.float16)[1:].view(6, 256)), dict(o=None), dict(q=torch.zeros(6, 3, 64, dtype=torch.float16)),
    dict(q=torch.zeros(7, 4, 64, dtype=torch.float16)), dict(softmax_scale=0.0), dict(softmax_scale=-1.0), dict(softmax_scale=math.nan),
    dict(softmax_scale="big"), dict(max_prefix_len=-1), dict(max_prefix_len=0.5), dict(prefill=6), dict(dec=2), dict(dec=-1, prefill=7),
    dict(heads=3, q=torch.zeros(6, 3, 64, dtype=torch.float16), o=torch.zeros(6, 192, dtype=torch.float16)),
    dict(heads=34, q=torch.zeros(6, 34, 64, dtype=torch.float16), o=torch.zeros(6, 34 * 64, dtype=torch.float16))])
def test_section_refuses_before_it_launches(monkeypatch, change):
    """A call that its attention would refuse leaves q and the cache as they are: done again, it must not rotate q twice."""
    assert section(monkeypatch, **change) == "refused"


@pytest.mark.parametrize("entry", ["mkv_attn8_decode", "mkv_attn8_prefill"])
def test_more_ranges_than_a_launch_has_threads(entry):
    """2^24 ranges of 256 threads each are 2^32 threads."""
    for splits in (2 ** 24, 2 ** 25, 2 ** 27):
        assert attn(entry, tps=64, splits=splits) == _capi.MKV_EINVAL, splits


# ---- the native module beside the library -----------------------------------------------------------------------------------
def test_library_is_linked_without_the_native_module(monkeypatch, tmp_path):
    """A tree whose Python or torch headers do not fit the module still yields the library, which needs neither."""
    from morphserve_amd.csrc import build
    linked = []

    def no_module():
        raise RuntimeError("no Python.h")

    monkeypatch.setattr(build, "HERE", str(tmp_path))
    monkeypatch.setattr(build, "_compile", lambda src, obj_dir, defines=(): src)
    monkeypatch.setattr(build, "_link", lambda objs, out: linked.append(out))
    monkeypatch.setattr(build, "_build_binding", no_module)
    with pytest.raises(RuntimeError, match="Python.h"):
        build.build_library(verbose=False)
    assert linked == [build.LIB_PATH, build.DIAG_LIB_PATH]


def test_module_of_another_python_or_torch(monkeypatch, tmp_path):
    """Its file name carries the interpreter's tag, and one that does not load says what to do."""
    import sysconfig
    from morphserve_amd.csrc import build
    suffix = sysconfig.get_config_var("EXT_SUFFIX")
    assert build.BINDING_PATH.endswith("_binding" + suffix)
    monkeypatch.setattr(_capi, "_binding", None)
    monkeypatch.setattr(_capi, "_HERE", str(tmp_path))
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "_binding.so").write_bytes(b"of whatever interpreter")
    with pytest.raises(ImportError, match="is missing: build it"):
        _capi.binding()
    (tmp_path / "csrc" / ("_binding" + suffix)).write_bytes(b"no module")
    for _ in range(2):                                      # a failed load is not taken for the module the next time
        with pytest.raises(ImportError, match="build it again with"):
            _capi.binding()


@pytest.mark.parametrize("bad", [dict(scale=0.0), dict(scale=-0.1), dict(scale=math.nan), dict(scale=-math.inf), dict(o=A + 8), dict(os_=1028)])
def test_bad_chunk_attention(bad):
    """What the chunk entry refuses and the decode entry does not."""
    a = dict(o=A, os_=1024, scale=0.1)
    a.update(bad)
    assert _capi.lib().mkv_attn8_prefill(C.byref(pool8()), C.byref(batch8()), 0, A, a["o"], 1024, a["os_"], 8, a["scale"], 0, 64, 2, A, A,
                                         None) == _capi.MKV_EINVAL
    assert (b"softmax_scale" if "scale" in bad else b"aligned") in _capi.lib().mkv_last_error()
