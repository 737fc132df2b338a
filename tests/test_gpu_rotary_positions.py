"""``rotary_embedding`` against 64-bit arithmetic: both layouts, part of the head, any even rotary dim, strides, in place and
not, positions outside the tables."""
import numpy as np
import pytest
import torch

from kv8_helpers import DTYPES, as_np, assert_within, rounded
from oracle import kv8_cpu as K
from morphserve_amd import rotary_embedding, rotary_scaled_tables

pytestmark = pytest.mark.gpu


def expect(x, pos, cos, sin, layout, dtype):
    """The exact rotation and the bound: one rounding to the type, three of 32 bits on the way."""
    want = K.rotate(x, pos, cos, sin, layout)
    a = np.abs(K.rotate(np.abs(x), pos, np.abs(cos), -np.abs(sin), layout))
    b = np.abs(K.rotate(np.abs(x), pos, np.abs(cos), np.abs(sin), layout))
    half_step = 2.0 ** -11 if dtype == "f16" else 2.0 ** -8
    return want, half_step * np.abs(want) + 2.0 ** -22 * np.maximum(a, b) + 2.0 ** -25


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rotary", [(128, 128), (128, 64), (128, 32), (64, 64), (80, 32), (96, 24), (64, 2), (256, 256),
                                        (40, 40), (50, 14), (7, 6), (128, 126)])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rotation(cuda, dtype, dim, rotary, layout):
    rng = np.random.default_rng(dim * 1000 + rotary)
    for tokens, hq, hkv in ((1, 1, 1), (37, 5, 2), (130, 8, 8)):
        q, k = (as_np(rounded(rng.standard_normal((tokens, h, dim)) * 4, dtype)) for h in (hq, hkv))
        cos, sin = rotary_scaled_tables(rotary, 500, 10000.0, device=cuda)
        pos = rng.integers(0, 500, tokens)
        posg = torch.tensor(pos, dtype=torch.int32, device=cuda)
        fused = rounded(np.concatenate([q, k, k], 1), dtype).to(cuda)
        qg, kg = fused[:, :hq], fused[:, hq:hq + hkv]
        q_out = torch.full((tokens, hq * dim + 8), 9.0, dtype=DTYPES[dtype], device=cuda)[:, :hq * dim]
        k_out = torch.empty(tokens, hkv, dim, dtype=DTYPES[dtype], device=cuda)
        c, s = cos.cpu().numpy(), sin.cpu().numpy()
        rotary_embedding(qg, kg, posg, cos, sin, layout=layout, q_out=q_out, k_out=k_out)
        assert np.array_equal(as_np(qg), q) and np.array_equal(as_np(kg), k)
        for got, x in ((q_out, q), (k_out, k)):
            assert_within(got, *expect(x, pos, c, s, layout, dtype), f"{tokens} x {x.shape[1]}")
        rotary_embedding(qg, kg, posg, cos, sin, layout=layout)                     # in place: the same bits
        assert torch.equal(qg.reshape(tokens, -1), q_out) and torch.equal(kg, k_out)
        assert np.array_equal(as_np(fused[:, hq + hkv:]), k)                        # the neighbours stay


def test_without_k_and_misaligned(cuda):
    rng = np.random.default_rng(1)
    q = as_np(rounded(rng.standard_normal((9, 3, 64)), "f16"))
    cos, sin = rotary_scaled_tables(32, 20, device=cuda)
    pos = torch.arange(9, dtype=torch.int32, device=cuda)
    store = torch.zeros(9 * 3 * 64 + 1, dtype=torch.float16, device=cuda)
    qg = store[1:].view(9, 3, 64)
    qg.copy_(rounded(q, "f16"))
    rotary_embedding(qg, None, pos, cos, sin)
    assert_within(qg, *expect(q, np.arange(9), cos.cpu().numpy(), sin.cpu().numpy(), "half", "f16"))
    assert store[0] == 0


def test_positions_outside_the_tables(cuda):
    q = torch.ones(5, 2, 64, dtype=torch.bfloat16, device=cuda)
    cos, sin = rotary_scaled_tables(32, 10, device=cuda)
    pos = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
    rotary_embedding(q, None, pos, cos, sin)
    lost = torch.isnan(q)
    assert lost[[1, 3, 4], :, :32].all() and not lost[:, :, 32:].any() and not lost[[0, 2]].any()
    assert (q[:, :, 32:] == 1).all()


@pytest.mark.parametrize("scaling", [None, 4.0, {"rope_type": "dynamic", "factor": 4.0, "original_max_position_embeddings": 4096},
                                     {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 8192},
                                     {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}])
def test_far_positions(cuda, scaling):
    """Tables made on the GPU and on the CPU agree to a rounding at positions where 32-bit angles would be lost."""
    a = rotary_scaled_tables(128, 131072, 500000.0, scaling, cuda)
    b = rotary_scaled_tables(128, 131072, 500000.0, scaling, "cpu")
    for x, y in zip(a, b):
        assert (x.cpu() - y).abs().max() <= 2.0 ** -23
    rng = np.random.default_rng(2)
    q = as_np(rounded(rng.standard_normal((300, 4, 128)), "f16"))
    pos = rng.integers(0, 131072, 300)
    qg = rounded(q, "f16").to(cuda)
    rotary_embedding(qg, None, torch.tensor(pos, dtype=torch.int32, device=cuda), *a)
    assert_within(qg, *expect(q, pos, a[0].cpu().numpy(), a[1].cpu().numpy(), "half", "f16"))


def test_graph(cuda):
    q, k = torch.empty(50, 4, 128, dtype=torch.float16, device=cuda), torch.empty(50, 2, 128, dtype=torch.float16, device=cuda)
    outs = [(torch.empty_like(q), torch.empty_like(k)) for _ in range(2)]
    cos, sin = rotary_scaled_tables(64, 100, device=cuda)
    pos = torch.arange(50, dtype=torch.int32, device=cuda)
    run = lambda o: rotary_embedding(q, k, pos, cos, sin, "interleaved", *o)  # noqa: E731
    run(outs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(outs[0])
    for _ in range(3):
        q.normal_(), k.normal_()
        graph.replay()
        run(outs[1])
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(*outs))


def test_refusals(cuda):
    q = torch.zeros(4, 2, 64, dtype=torch.float16, device=cuda)
    cos, sin = rotary_scaled_tables(32, 10, device=cuda)
    pos = torch.zeros(4, dtype=torch.int32, device=cuda)
    from morphserve_amd._capi import MorphKVError
    for call in (lambda: rotary_embedding(q.float(), None, pos, cos, sin),
                 lambda: rotary_embedding(q, None, pos.long(), cos, sin),
                 lambda: rotary_embedding(q, None, pos[:3], cos, sin),
                 lambda: rotary_embedding(q, None, pos, cos.half(), sin.half()),
                 lambda: rotary_embedding(q, None, pos, cos, sin[:, :8]),
                 lambda: rotary_embedding(q, None, pos, cos, sin, layout="neox"),
                 lambda: rotary_embedding(q, q.bfloat16(), pos, cos, sin),
                 lambda: rotary_embedding(q.cpu(), None, pos, cos, sin),
                 lambda: rotary_embedding(q, None, pos, cos, sin, q_out=q[:1].expand(4, 2, 64))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(MorphKVError):
        rotary_embedding(q, None, pos, *rotary_scaled_tables(66, 10, device=cuda))
    torch.cuda.synchronize()
    assert not q.any()


def test_an_output_without_its_input_is_refused(cuda):
    q = torch.ones(4, 2, 64, dtype=torch.float16, device=cuda)
    k_out = torch.zeros_like(q)
    with pytest.raises(ValueError):
        rotary_embedding(q, None, torch.ones(4, dtype=torch.int32, device=cuda), *rotary_scaled_tables(32, 10, device=cuda), k_out=k_out)
    torch.cuda.synchronize()
    assert (q == 1).all() and not k_out.any()
