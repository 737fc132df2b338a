"""Measured cases of the 8-bit paged cache and the rotary operators, with their plain forms.

The cache: K codes [blocks, layers, kv heads, 16, D], V codes [blocks, layers, kv heads, D, 16], both e4m3 or int8, and
uint8 ``scales`` [layers, kv heads, blocks, 2] (K, V): a code stands for ``code * 2**(scale - 127)``.  Blocks belong to
sequences through ``block_table`` rows.
"""
import math
import random
from types import SimpleNamespace

import torch

own = False

B = 16                                     # tokens per block
FP8 = torch.float8_e4m3fn
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
QMAX = {"e4m3": 448.0, "int8": 127.0}


def listed():
    f8, i8 = "e4m3", "int8"
    return [
        # one new token for each of 64 sequences of 1024 to 1536 tokens: latency counts
        dict(name="rotary decode rows", op="rotary", tokens=64, hq=32, hkv=8, d=128, r=128, layout="half",
             scaling="llama3", type="f16", far=1536),
        # a long ragged prefill batch, rows cut out of a fused projection, half of each head, far positions
        dict(name="rotary long prefill", op="rotary", tokens=16385, hq=32, hkv=8, d=128, r=64, layout="interleaved",
             scaling="yarn", type="bf16", far=131072),
        # the append of a decode step
        dict(name="store decode rows", op="store", chunks=0, clo=0, chi=0, plo=0, phi=0, n=64, lo=1024, hi=1536,
             hq=32, hkv=8, d=128, r=128, layout="half", type="f16", kind=f8),
        # eight whole prompts of 512 tokens, multi-head attention
        dict(name="store prompts", op="store", chunks=8, clo=512, chi=512, plo=0, phi=0, n=0, lo=0, hi=0,
             hq=32, hkv=32, d=128, r=128, layout="half", type="f16", kind=f8),
        # a mixed batch: ragged chunks over ragged cached prefixes, and decode rows
        dict(name="store mixed batch", op="store", chunks=5, clo=33, chi=700, plo=0, phi=2000, n=57, lo=1, hi=1536,
             hq=64, hkv=8, d=128, r=64, layout="interleaved", type="bf16", kind=i8),
        # a small decode batch of short contexts, multi-head attention: latency counts
        dict(name="decode short contexts", op="decode", n=8, lo=64, hi=512, hq=32, hkv=32, d=128, type="f16", kind=f8),
        # the decode step of a serving batch
        dict(name="decode serving batch", op="decode", n=64, lo=1024, hi=1536, hq=32, hkv=8, d=128, type="f16", kind=f8),
        # a larger model's decode step
        dict(name="decode large batch", op="decode", n=128, lo=1024, hi=1536, hq=64, hkv=8, d=128, type="bf16", kind=i8),
        # few sequences, long contexts: the work has to be split over the tokens
        dict(name="decode long contexts", op="decode", n=5, lo=20000, hi=60000, hq=32, hkv=8, d=128, type="bf16", kind=f8),
        # whole prompts, multi-head attention
        dict(name="prefill prompts", op="chunk", chunks=8, clo=512, chi=512, plo=0, phi=0, hq=32, hkv=32, d=128,
             type="f16", kind=f8),
        # ragged chunks of long prompts over what is cached of them
        dict(name="prefill ragged chunks", op="chunk", chunks=4, clo=500, chi=2048, plo=1000, phi=8192, hq=32, hkv=8,
             d=128, type="bf16", kind=i8),
        # a few rows each over long contexts, as when drafted tokens are verified
        dict(name="prefill few rows", op="chunk", chunks=6, clo=1, chi=16, plo=8000, phi=16000, hq=64, hkv=8, d=128,
             type="f16", kind=f8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "store", "decode", "chunk"])
    hq, hkv = rng.choice([(32, 8), (32, 32), (64, 8), (28, 4), (16, 1), (12, 4), (8, 8), (15, 3), (40, 8)])
    c = dict(op=op, hq=hq, hkv=hkv, d=rng.choice([64, 128, 128]), type=rng.choice(["f16", "bf16"]))
    if op == "rotary":
        c.update(tokens=_log(rng, 1, 16000 * 40 // (hq + hkv)), r=2 * rng.randint(4, c["d"] // 2),
                 layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "llama3", "yarn"]),
                 far=_log(rng, 512, 131072))
        return c
    c["kind"] = rng.choice(["e4m3", "int8"])
    if op == "decode":
        hi = _log(rng, 16, 60000)
        most = max(1, min(256, 5 * 40000 * 8 // (hi * hkv)))
        c.update(n=_log(rng, 1, most), lo=max(1, hi // rng.choice([1, 2, 5])), hi=hi)
        return c
    chi = _log(rng, 1, 2048)
    phi = rng.choice([0, _log(rng, 1, 8192)])
    # at most about the rows x keys of the largest listed case
    most = max(1, min(16, 4 * 1300 * 5500 * 32 // (chi * (phi + chi) * hq)))
    c.update(chunks=rng.randint(1, most), clo=max(1, chi // rng.choice([1, 2, 5])), chi=chi, plo=phi // 3, phi=phi)
    if op == "store":
        c.update(n=rng.choice([0, _log(rng, 1, 128)]), lo=1, hi=_log(rng, 2, 2000),
                 r=16 * rng.randint(1, c["d"] // 16), layout=rng.choice(["half", "interleaved"]))
    return c


# ---- shapes that follow from a case ----------------------------------------------------------------------------------
def _lens(count, lo, hi, salt):
    rng = random.Random("%s %d %d %d" % (salt, count, lo, hi))
    return [rng.randint(lo, hi) for _ in range(count)]


def _shape(c):
    """chunk lengths, cached prefixes, decode lengths (the new token included)"""
    chunks = _lens(c.get("chunks", 0), c.get("clo", 0), c.get("chi", 0), "chunk")
    prefix = _lens(c.get("chunks", 0), c.get("plo", 0), c.get("phi", 0), "prefix")
    return chunks, prefix, _lens(c.get("n", 0), c.get("lo", 0), c.get("hi", 0), "decode")


def work(c):
    if c["op"] == "rotary":
        rows = c["tokens"] * (c["hq"] + c["hkv"])
        return {"bytes": 4 * rows * c["d"] + 4 * c["tokens"] * c["r"] + 4 * c["tokens"], "flops": 3 * rows * c["r"]}
    chunks, prefix, dec = _shape(c)
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    tokens = sum(chunks) + len(dec)
    if c["op"] == "store":
        touched = sum(-(-(p + n) // B) - p // B for n, p in zip(chunks, prefix)) + len(dec)
        return {"bytes": tokens * (4 * hq * d + 6 * hkv * d + 4 * c["r"]) + 4 * hkv * touched,
                "flops": tokens * (3 * (hq + hkv) * c["r"] + 4 * hkv * d)}
    keys = sum(dec) + sum(p + n for n, p in zip(chunks, prefix))
    pairs = sum(dec) + sum(n * p + n * (n + 1) // 2 for n, p in zip(chunks, prefix))
    blocks = sum(-(-x // B) for x in dec + [p + n for n, p in zip(chunks, prefix)])
    return {"bytes": 2 * keys * hkv * d + blocks * (2 * hkv + 4) + 4 * tokens * hq * d, "flops": 4 * pairs * hq * d}


# ---- inputs ------------------------------------------------------------------------------------------------------------
def _pow2(e):
    """2**(e - 127) for biased exponents 1 .. 254"""
    return (e.to(torch.int32) << 23).view(torch.float32)


def _round8(x, kind):
    return x.to(FP8) if kind == "e4m3" else torch.round(torch.nan_to_num(x)).to(torch.int8)


def _exponent(amax, kind):
    """The least biased exponent e, at least 1, with amax <= QMAX * 2**(e - 127); of zeros 1."""
    m, x = torch.frexp(amax)
    top, shift = (0.875, 9) if kind == "e4m3" else (127 / 128, 7)
    return torch.where(amax > 0, x - shift + (m > top) + 127, 1).clamp(min=1).to(torch.uint8)


def _tables(r, rows, scaling, far, device):
    """cos and sin of position x frequency, from 64 bits, rounded to 32"""
    base, factor = 500000.0, 8.0
    inv = base ** (-torch.arange(0, r, 2, device=device, dtype=torch.float64) / r)
    mul = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "llama3":
        wave, low, high, old = 2 * math.pi / inv, 1.0, 4.0, far / factor
        mix = ((old / wave - low) / (high - low)).clamp(0, 1)
        inv = inv * mix + inv / factor * (1 - mix)
    elif scaling == "yarn":
        at = lambda turns: r * math.log(max(far / factor, 1) / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(at(32)), 0), min(math.ceil(at(1)), r - 1)
        ramp = ((torch.arange(r // 2, device=device, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        inv = inv / factor * ramp + inv * (1 - ramp)
        mul = 0.1 * math.log(factor) + 1
    angle = torch.arange(rows, device=device, dtype=torch.float64)[:, None] * inv
    return (angle.cos() * mul).float(), (angle.sin() * mul).float()


def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *s: torch.randn(s, generator=g, device=dev)  # noqa: E731
    t, hq, hkv, d = TYPES[c["type"]], c["hq"], c["hkv"], c["d"]
    s = SimpleNamespace(case=c, kind=c.get("kind"), type=t, layer=1)
    if c["op"] == "rotary":
        s.qkv = randn(c["tokens"], hq + 2 * hkv, d).to(t)          # rows of a fused projection
        s.q, s.k = s.qkv[:, :hq], s.qkv[:, hq:hq + hkv]
        s.cos, s.sin = _tables(c["r"], c["far"], c["scaling"], c["far"], dev)
        s.positions = torch.randint(0, c["far"], (c["tokens"],), generator=g, device=dev, dtype=torch.int32)
        s.q_out = torch.empty(c["tokens"], hq, d, dtype=t, device=dev)
        s.k_out = torch.empty(c["tokens"], hkv, d, dtype=t, device=dev)
        return s

    chunks, prefix, dec = _shape(c)
    total = [p + n for n, p in zip(chunks, prefix)] + dec          # tokens each sequence holds after the call
    cached = total if c["op"] != "store" else prefix + [n - 1 for n in dec]
    seqs, layers, tokens = len(total), 2, sum(chunks) + len(dec)
    need = [-(-n // B) for n in total]
    width = max(need) + 1
    blocks = sum(need) + 3
    i32 = dict(dtype=torch.int32, device=dev)
    # every sequence's blocks lie scattered over the pool, its row anywhere in the table
    ids = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    rows = torch.randperm(seqs + 2, generator=g, device=dev)[:seqs].to(torch.int32)
    owned = torch.arange(width, device=dev)[None] < torch.tensor(need, device=dev)[:, None]
    table = torch.full((seqs, width), -1, **i32)
    table[owned] = ids[:sum(need)]
    s.block_table = torch.full((seqs + 2, width), -1, **i32)
    s.block_table[rows.long()] = table
    starts = [sum(chunks[:j]) for j in range(len(chunks))]
    s.prefix_lens = torch.tensor(prefix, **i32)
    s.max_prefix_len = max(prefix, default=0)
    s.infer = SimpleNamespace(
        batch_size=seqs, num_tokens=tokens, seq_ids=rows, softmax_scale=d ** -0.5, num_prefill_seqs=len(chunks),
        num_prefill_tokens=sum(chunks), prefill_seq_start_locs=torch.tensor(starts, **i32),
        prefill_seq_lens=torch.tensor(chunks, **i32), max_prefill_len=max(chunks, default=0),
        num_decoding_seqs=len(dec), decoding_seq_lens=torch.tensor(dec, **i32), max_decoding_len=max(dec, default=0))
    s.model = SimpleNamespace(num_layers=layers, num_q_heads=hq, num_kv_heads=hkv, head_dim=d)
    s.engine = SimpleNamespace(block_size=B, max_blocks_per_seq=width)

    # what is cached: normal values, some head dims of K ten times as large; a block's rows behind its last token, and
    # the blocks that nobody owns, hold old codes of any kind
    code = FP8 if s.kind == "e4m3" else torch.int8
    s.k = torch.zeros(blocks, layers, hkv, B, d, device=dev, dtype=torch.uint8).view(code)
    s.v = torch.zeros(blocks, layers, hkv, d, B, device=dev, dtype=torch.uint8).view(code)
    s.scales = torch.ones(layers, hkv, blocks, 2, device=dev, dtype=torch.uint8)
    end = torch.zeros(blocks, device=dev, dtype=torch.int64)       # cached tokens of each block
    left = torch.tensor(cached, device=dev)[:, None] - B * torch.arange(width, device=dev)[None]
    end[table[owned].long()] = left[owned].clamp(0, B)
    loud = 1 + 9 * (torch.rand(hkv, 1, d, generator=g, device=dev) < 0.02)
    step = max(1, (1 << 26) // (hkv * B * d))                      # bounds the temporaries
    for at in range(0, blocks, step):
        n = min(step, blocks - at)
        live = torch.arange(B, device=dev)[None, :] < end[at:at + n, None]
        for which, to in ((0, s.k), (1, s.v)):
            x = randn(n, hkv, B, d) * (loud if which == 0 else 1)
            e = _exponent((x * live[:, None, :, None]).abs().amax((2, 3)), s.kind)
            q = _round8(x / _pow2(e)[..., None, None], s.kind).view(torch.uint8)
            old = torch.randint(0, 256, q.shape, generator=g, device=dev, dtype=torch.uint8)
            q = torch.where(live[:, None, :, None], q, old)
            to[at:at + n, s.layer].view(torch.uint8).copy_(q if which == 0 else q.transpose(2, 3))
            s.scales[s.layer, :, at:at + n, which] = e.T
    s.q = randn(tokens, hq, d).to(t)
    s.o = torch.empty(tokens, hq, d, dtype=t, device=dev)
    if c["op"] == "store":
        s.new_k, s.new_v = (randn(tokens, hkv, d) * loud[:, 0]).to(t), randn(tokens, hkv, d).to(t)
        s.cos, s.sin = _tables(c["r"], max(total) + 1, "none", 1, dev)
    # where each new row goes: its position, its row of the table, its block among those that receive rows
    s.positions = torch.tensor([p + j for n, p in zip(chunks, prefix) for j in range(n)] + [n - 1 for n in dec], **i32)
    s.batch_row = torch.tensor([b for b, n in enumerate(chunks) for _ in range(n)] +
                               [len(chunks) + i for i in range(len(dec))], device=dev)
    s.keys = max(total, default=0)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------
def _rotate(x, positions, cos, sin, layout):
    r = 2 * cos.shape[1]
    c, n = cos[positions.long()][:, None], sin[positions.long()][:, None]
    x = x.float()
    if layout == "half":
        x0, x1 = x[..., :r // 2], x[..., r // 2:r]
        turned = torch.cat([x0 * c - x1 * n, x0 * n + x1 * c], -1)
    else:
        x0, x1 = x[..., :r:2], x[..., 1:r:2]
        turned = torch.stack([x0 * c - x1 * n, x0 * n + x1 * c], -1).flatten(-2)
    return torch.cat([turned, x[..., r:]], -1)


def _plain_store(s):
    st, lay, kind = s.infer, s.layer, s.kind
    q = _rotate(s.q, s.positions, s.cos, s.sin, s.case["layout"]).to(s.type)
    pos = s.positions.long()
    pid = s.block_table[st.seq_ids.long()[s.batch_row], pos // B].long()
    blocks, item = torch.unique(pid, return_inverse=True)
    first = torch.full(blocks.shape, B, device=pos.device).scatter_reduce(0, item, pos % B, "amin")
    before = (torch.arange(B, device=pos.device)[None] < first[:, None])[:, None, :, None]
    for which, cache, x in ((0, s.k, _rotate(s.new_k, s.positions, s.cos, s.sin, s.case["layout"])),
                            (1, s.v, s.new_v.float())):
        amax = torch.zeros(len(blocks), x.shape[1], device=x.device).scatter_reduce(
            0, item[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
        e, was = _exponent(amax, kind), s.scales[lay, :, blocks, which].T
        e = torch.where((first == 0)[:, None], e, torch.maximum(e, was))
        codes = cache.view(torch.uint8)[blocks, lay]
        codes = codes.transpose(2, 3) if which else codes
        again = codes.contiguous().view(cache.dtype).float() * (_pow2(was) / _pow2(e))[..., None, None]
        codes = torch.where(before, _round8(again, kind).view(torch.uint8), codes)
        codes[item, :, pos % B] = _round8(x / _pow2(e)[item][..., None], kind).view(torch.uint8)
        cache.view(torch.uint8)[blocks, lay] = codes.transpose(2, 3) if which else codes
        s.scales[lay, :, blocks, which] = e.T
    # codes and scales together are the values the cache holds; equal codes and scales are the stricter comparison, and
    # neither side pays for a pass over the whole cache that no user makes
    return q, s.k, s.v, s.scales


def _gather(s, rows, keys):
    """K and V of the sequences in these table rows, [sequences, kv heads, keys, D] in 32 bits"""
    nb = -(-keys // B)
    ids = s.block_table[rows.long(), :nb].long().clamp(min=0)
    f = _pow2(s.scales[s.layer][:, ids])[..., None, None, :]       # [heads, sequences, blocks, 1, 1, 2]
    k = s.k.view(torch.uint8)[ids, s.layer].view(s.k.dtype).float() * f[..., 0].permute(1, 2, 0, 3, 4)
    v = s.v.view(torch.uint8)[ids, s.layer].view(s.v.dtype).float() * f[..., 1].permute(1, 2, 0, 3, 4)
    return k.transpose(1, 2).flatten(2, 3), v.permute(0, 2, 1, 4, 3).flatten(2, 3)


def _attend(q, k, v, last, scale):
    """q [n, kv heads, rows, D]; each row sees the keys up to last [n, rows] (-1: none)"""
    at = torch.arange(k.shape[2], device=q.device)
    sees = (at <= last[..., None])[:, None]                       # [n, 1, rows, keys]
    v = torch.where((at <= last.amax(1)[:, None])[:, None, :, None], v, 0)
    score = (torch.matmul(q, k.transpose(2, 3)) * scale).masked_fill_(~sees, -math.inf)
    p = torch.exp_(score.sub_(score.amax(-1, keepdim=True).clamp(min=-3e38)))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / total.clamp(min=1e-38)


def _plain_decode(s):
    n, hkv, d = s.infer.num_decoding_seqs, s.case["hkv"], s.case["d"]
    k, v = _gather(s, s.infer.seq_ids, s.keys)
    last = (s.infer.decoding_seq_lens.long() - 1)[:, None].expand(-1, s.case["hq"] // hkv)
    o = _attend(s.q.float().view(n, hkv, -1, d), k, v, last, s.infer.softmax_scale)
    return o.reshape(n, -1, d).to(s.type)


def _plain_chunk(s):
    st, hq, hkv, d = s.infer, s.case["hq"], s.case["hkv"], s.case["d"]
    n, rows, group = st.num_prefill_seqs, st.max_prefill_len, hq // hkv
    k, v = _gather(s, st.seq_ids, s.keys)
    at = torch.arange(rows, device=s.q.device)
    real = at[None] < st.prefill_seq_lens[:, None]
    q = torch.zeros(n, rows, hq, d, device=s.q.device)
    q[real] = s.q.float()
    last = torch.where(real, s.prefix_lens[:, None] + at[None], -1)[:, None].expand(-1, group, -1).reshape(n, -1)
    q = q.view(n, rows, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, group * rows, d)
    o = _attend(q, k, v, last, st.softmax_scale)
    o = o.view(n, hkv, group, rows, d).permute(0, 3, 1, 2, 4).reshape(n, rows, hq, d)
    return o[real].to(s.type)


def run(s):
    c = s.case
    if own:
        import morphserve_amd as M
        if c["op"] == "rotary":
            M.rotary_embedding(s.q, s.k, s.positions, s.cos, s.sin, layout=c["layout"], q_out=s.q_out, k_out=s.k_out)
            return s.q_out, s.k_out
        cache = M.KV8Cache(s.k, s.v, s.scales)
        if c["op"] == "store":
            M.rotary_embedding_and_store_kvcache_8bit(
                s.q, s.new_k, s.new_v, s.cos, s.sin, cache, s.block_table, s.model, s.engine, s.infer, s.layer,
                layout=c["layout"], q_out=s.o, prefix_lens=s.prefix_lens if s.max_prefix_len else None)
            return s.o, s.k, s.v, s.scales
        if c["op"] == "decode":
            M.paged_attention_8bit(s.q, cache, s.block_table, s.model, s.engine, s.infer, s.layer, s.o)
        else:
            M.chunked_prefill_attention_8bit(s.q, cache, s.block_table, s.model, s.engine, s.infer, s.layer, s.o,
                                             prefix_lens=s.prefix_lens, max_prefix_len=s.max_prefix_len)
        return s.o
    if c["op"] == "rotary":
        return tuple(_rotate(x, s.positions, s.cos, s.sin, c["layout"]).to(s.type) for x in (s.q, s.k))
    return {"store": _plain_store, "decode": _plain_decode, "chunk": _plain_chunk}[c["op"]](s)


# ---- the definitions in 64 bits, written apart from the plain forms ------------------------------------------------------
def _turned(x, angle_cos, angle_sin, layout):
    """x [rows, heads, D] as complex numbers times cos + i sin"""
    r = 2 * angle_cos.shape[1]
    head, rest = x[..., :r].double(), x[..., r:].double()
    pair = head.unflatten(-1, (2, r // 2)).transpose(-1, -2) if layout == "half" else head.unflatten(-1, (r // 2, 2))
    z = torch.view_as_complex(pair.contiguous()) * torch.complex(angle_cos.double(), angle_sin.double())[:, None]
    pair = torch.view_as_real(z)
    head = pair.transpose(-1, -2).flatten(-2) if layout == "half" else pair.flatten(-2)
    return torch.cat([head, rest], -1)


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rotary":
        at = s.positions.long()
        return tuple(_turned(x, s.cos[at], s.sin[at], c["layout"]) for x in (s.q, s.k))
    chunks, prefix, dec = _shape(c)
    lens, before = chunks + [1] * len(dec), prefix + [n - 1 for n in dec]
    d, hkv, group = c["d"], c["hkv"], c["hq"] // c["hkv"]
    at = s.positions.long()
    if c["op"] == "store":
        q = _turned(s.q, s.cos[at], s.sin[at], c["layout"])
        if s.kind == "int8":                   # whole numbers: rounding decides them, and the plain form holds it
            return q, None, None, None
        out = []
        fresh = (_turned(s.new_k, s.cos[at], s.sin[at], c["layout"]), s.new_v.double())
        for which, codes in ((0, s.k.double()), (1, s.v.double().transpose(3, 4).contiguous())):
            row = 0
            for b, (n, p) in enumerate(zip(lens, before)):
                for j in range(p // B, (p + n - 1) // B + 1):
                    lo, hi = max(p, j * B), min(p + n, (j + 1) * B)
                    pid = int(s.block_table[int(s.infer.seq_ids[b]), j])
                    x = fresh[which][row + lo - p:row + hi - p].transpose(0, 1)        # [heads, rows, D]
                    top = x.abs().amax((1, 2))
                    e = torch.ceil(torch.log2(top / 448))
                    e = torch.where(448 * 2.0 ** (e - 1) >= top, e - 1, e).clamp(min=-126)
                    was = s.scales[s.layer, :, pid, which].double() - 127
                    a = lo - j * B
                    if a:
                        e = torch.maximum(e, was)
                        codes[pid, s.layer, :, :a] *= (2.0 ** (was - e))[:, None, None]
                    codes[pid, s.layer, :, a:a + hi - lo] = x * (2.0 ** -e)[:, None, None]
                row += n
            out.append(codes if which == 0 else codes.transpose(3, 4).contiguous())
        return q, out[0], out[1], None
    out, row = [], 0
    for b, (n, p) in enumerate(zip(lens, before)):
        keys = p + n
        ids = s.block_table[int(s.infer.seq_ids[b]), :-(-keys // B)].long()
        f = 2.0 ** (s.scales[s.layer][:, ids].double() - 127)                          # [heads, blocks, 2]
        k = s.k[ids, s.layer].double() if s.kind == "int8" else s.k.view(torch.uint8)[ids, s.layer].view(FP8).double()
        v = s.v[ids, s.layer].double() if s.kind == "int8" else s.v.view(torch.uint8)[ids, s.layer].view(FP8).double()
        k = (k.transpose(0, 1) * f[..., 0, None, None]).flatten(1, 2)[:, :keys]
        v = (v.transpose(0, 1).transpose(2, 3) * f[..., 1, None, None]).flatten(1, 2)[:, :keys]
        q = s.q[row:row + n].double().view(n, hkv, group, d)
        hidden = torch.arange(keys, device=q.device)[None] > p + torch.arange(n, device=q.device)[:, None]
        o = torch.empty(n, hkv, group, d, dtype=torch.float64, device=q.device)
        for h in range(hkv):
            score = torch.einsum("rgd,kd->grk", q[:, h], k[h]) * s.infer.softmax_scale
            o[:, h] = torch.einsum("grk,kd->rgd", score.masked_fill(hidden, -math.inf).softmax(-1), v[h])
        out.append(o.reshape(n, -1, d))
        row += n
    return torch.cat(out)
