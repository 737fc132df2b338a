"""Seeded batches over an 8-bit cache, on the host (oracle arrays) and on the GPU."""
from __future__ import annotations

import numpy as np
import torch

from helpers import Cfg
from oracle import kv8_cpu as K

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def rounded(x: np.ndarray, dtype: str) -> torch.Tensor:
    return torch.from_numpy(np.asarray(x, dtype=np.float32)).to(DTYPES[dtype])


def as_np(t: torch.Tensor) -> np.ndarray:
    return t.detach().float().cpu().numpy()


class Batch:
    """Chunks (lengths, cached prefixes) and decode rows (lengths, the new token included) over a scattered pool whose
    unused codes are old bytes of any kind, NaN among them."""

    def __init__(self, seed, hq=8, hkv=2, dim=128, dtype="f16", kind="e4m3", chunks=(), prefixes=None, dec=(), layers=2,
                 layer=1, spare=3, live="all"):
        rng = self.rng = np.random.default_rng(seed)
        self.hq, self.hkv, self.dim, self.dtype, self.kind, self.layer = hq, hkv, dim, dtype, kind, layer
        self.chunks = [int(x) for x in chunks]
        self.prefixes = [0] * len(self.chunks) if prefixes is None else [int(x) for x in prefixes]
        self.dec = [int(x) for x in dec]
        self.total = [p + n for p, n in zip(self.prefixes, self.chunks)] + self.dec
        need = [-(-n // K.B) for n in self.total]
        self.n_blocks = sum(need) + spare
        self.width = max(need + [0]) + 2
        self.rows = len(self.total) + 3
        ids = rng.permutation(self.n_blocks)
        self.seq_ids = rng.permutation(self.rows)[:len(self.total)].astype(np.int32)
        self.table = np.full((self.rows, self.width), -1, dtype=np.int32)
        at = 0
        for s, nb in zip(self.seq_ids, need):
            self.table[s, :nb] = ids[at:at + nb]
            at += nb
        shape = (self.n_blocks, layers, hkv, K.B, dim)
        self.kc = rng.integers(0, 256, shape, dtype=np.uint8)
        self.vc = rng.integers(0, 256, (self.n_blocks, layers, hkv, dim, K.B), dtype=np.uint8)
        self.scales = rng.integers(0, 250, (layers, hkv, self.n_blocks, 2), dtype=np.uint8)
        # what is cached: every position but those a store would append (live="before"), or all of them
        cached = self.total if live == "all" else self.prefixes + [max(n - 1, 0) for n in self.dec]
        for s, n in zip(self.seq_ids, cached):
            for j in range(-(-n // K.B)):
                b = min(K.B, n - j * K.B)
                for h in range(hkv):
                    pid = self.table[s, j]
                    for which in (0, 1):
                        x = rng.standard_normal((b, dim)) * 2.0 ** rng.integers(-3, 3)
                        x[:, rng.integers(dim)] *= 8
                        old = self.kc[pid, layer, h] if which == 0 else self.vc[pid, layer, h].T
                        new, e = K.join(old, 0, x, 0, kind, dtype)
                        if which == 0:
                            self.kc[pid, layer, h] = new
                        else:
                            self.vc[pid, layer, h] = new.T
                        self.scales[layer, h, pid, which] = e
        self.tokens = sum(self.chunks) + len(self.dec)
        self.starts = np.concatenate([[0], np.cumsum(self.chunks)])[:len(self.chunks)].astype(np.int32)
        self.scale = dim ** -0.5
        self.model = Cfg(num_layers=layers, num_q_heads=hq, num_kv_heads=hkv, head_dim=dim)
        self.engine = Cfg(block_size=K.B, max_blocks_per_seq=self.width)

    # rows of q, k, v rounded to the type, as numpy (exact) -- positions follow the batch
    def new_rows(self, heads, spread=2):
        x = self.rng.standard_normal((self.tokens, heads, self.dim)) * 2.0 ** self.rng.integers(-spread, spread + 1,
                                                                                                  (self.tokens, heads, 1))
        return as_np(rounded(x, self.dtype))

    @property
    def positions(self):
        pos = [p + t for p, n in zip(self.prefixes, self.chunks) for t in range(n)] + [n - 1 for n in self.dec]
        return np.asarray(pos, dtype=np.int64)

    @property
    def runs(self):
        return K.rows_of(self.starts, self.chunks, self.prefixes, sum(self.chunks), self.dec, None)

    def state(self, dev):
        i32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=dev)  # noqa: E731
        return Cfg(batch_size=len(self.total), num_tokens=self.tokens, seq_ids=i32(self.seq_ids), softmax_scale=self.scale,
                   num_prefill_seqs=len(self.chunks), num_prefill_tokens=sum(self.chunks),
                   prefill_seq_start_locs=i32(self.starts), prefill_seq_lens=i32(self.chunks),
                   max_prefill_len=max(self.chunks + [0]), num_decoding_seqs=len(self.dec),
                   decoding_seq_lens=i32(self.dec), max_decoding_len=max(self.dec + [0]), ignore_kvcache=False)

    def prefix_tensor(self, dev):
        return torch.tensor(np.asarray(self.prefixes, dtype=np.int32), device=dev)

    def cache(self, dev):
        from morphserve_amd import KV8Cache
        code = CODES[self.kind]
        return KV8Cache(torch.from_numpy(self.kc.copy()).to(dev).view(code), torch.from_numpy(self.vc.copy()).to(dev).view(code),
                        torch.from_numpy(self.scales.copy()).to(dev))

    def block_table(self, dev):
        return torch.from_numpy(self.table.copy()).to(dev)

    # the oracle's answers
    def expect_decode(self, q):
        return self._attend(q, [(len(self.chunks) + i, [n - 1], slice(i, i + 1)) for i, n in enumerate(self.dec)])

    def expect_chunks(self, q):
        return self._attend(q, [(b, [p + t for t in range(n)], slice(int(s), int(s) + n))
                                for b, (s, n, p) in enumerate(zip(self.starts, self.chunks, self.prefixes))])

    def _attend(self, q, parts):
        want, bound = np.zeros(q.shape), np.zeros(q.shape)
        for slot, last, at in parts:
            if not last:
                continue
            got = K.attend(q[at], self.kc, self.vc, self.scales, self.table, int(self.seq_ids[slot]), last, self.layer,
                           self.kind, self.scale)
            want[at] = got[0]
            bound[at] = K.attend_bound(*got, self.dim, self.dtype)
        return want, bound


def assert_within(got: torch.Tensor, want: np.ndarray, bound: np.ndarray, what=""):
    g = got.detach().double().cpu().numpy().reshape(want.shape)
    assert np.isfinite(g).all(), f"{what}: not finite"
    off = np.abs(g - want) / bound
    at = np.unravel_index(np.argmax(off), off.shape)
    assert off.max(initial=0) <= 1, f"{what}: {off[at]:.2f} of the bound at {at}: got {g[at]!r}, want {want[at]!r}"


def assert_cache(cache, batch, what=""):
    """Every code and scale of the pool equal to the oracle's; NaN codes as NaN."""
    for name, got, want in (("scales", cache.scales, batch.scales), ("k", cache.k, batch.kc), ("v", cache.v, batch.vc)):
        g = got.view(torch.uint8).cpu().numpy()
        same = g == want
        if name != "scales" and batch.kind == "e4m3":
            same |= np.isnan(K.E4M3[g]) & np.isnan(K.E4M3[want])
        assert same.all(), f"{what}: {name} differs at {np.argwhere(~same)[:4].tolist()} ({(~same).sum()} in all)"
