"""The decoder layer of dnn-opt_b200/decode.py: the three operators in one step.

CPU: weight packing and the cache's page bookkeeping.  GPU: a stack of layers
generating tokens against the same computation in 32-bit torch operations.
Both sides round to bf16 at the same places; they differ where sums fall on
either side of a rounding boundary (a relative 2^-8 of single elements), which
a few products and norms later stays within 2 % of the whole.
"""
from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def decode(dn):
    import dnnopt_b200.decode as module
    return module


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("N,K,group", [(5, 64, 32), (3, 100, 32), (7, 33, 64), (4, 129, 128), (2, 1, 32)])
def test_weight_packing(decode, N, K, group, symmetric):
    """A packed weight is within half a step of the one it was made from, rows start at 16 bytes."""
    g = torch.Generator().manual_seed(K)
    w = torch.randn(N, K, generator=g)
    packed, scale, zero = decode.quantize_w4(w, group, symmetric)
    assert packed.shape == (N, (-(-K // 2) + 15) // 16 * 16) and scale.shape == (N, -(-K // group))
    back = decode.dequantize_w4(packed, scale, zero, K, group)
    step = scale.float()[:, torch.arange(K) // group]
    # Half a step of rounding; scales rounded to bf16 can leave the ends short by 2^-8 of 8 (15) steps,
    # the zero point's own rounding by half a step more.
    room = 0.5 + 8 * 2.0 ** -8 if symmetric else 1.0 + 15 * 2.0 ** -8
    assert bool(((back - w).abs() <= room * step + 1e-6).all())


def test_zero_weights_pack(decode):
    for symmetric in (True, False):
        packed, scale, zero = decode.quantize_w4(torch.zeros(2, 40), 32, symmetric)
        assert bool((decode.dequantize_w4(packed, scale, zero, 40, 32) == 0).all())


def test_cache_pages(decode):
    c = decode.PagedCache(2, 1, 16, pages=3, page_size=4, max_pages=2, device="cpu")
    c.grow(4)
    assert c.lens.tolist() == [4, 4] and len(c.free) == 1
    assert sorted(c.table[:, 0].tolist()) == [0, 1] and c.table[:, 1].tolist() == [-1, -1]
    with pytest.raises(RuntimeError):       # two more pages are needed, one is free
        c.grow(1)
    c.release(1)
    assert c.lens.tolist()[1] == 0 and c.table[1].tolist() == [-1, -1]
    assert len(c.free) + len(c.held[0]) == 3


@pytest.mark.gpu
@pytest.mark.parametrize("hidden,heads,kv_heads,dim,ffn,batch", [(256, 8, 2, 64, 512, 1), (512, 4, 4, 128, 1009, 3),
                                                                 (1024, 18, 2, 96, 2048, 9)])
def test_steps_match_the_plain_form(torch_cuda, decode, hidden, heads, kv_heads, dim, ffn, batch):
    c = decode.LayerConfig(hidden, heads, kv_heads, dim, ffn)
    stack = [decode.DecoderLayer(c, seed=i) for i in range(2)]
    cache = decode.PagedCache(batch, kv_heads, dim, pages=batch * 4, page_size=16, max_pages=4, layers=2)
    dense = [[torch.zeros(batch, 0, kv_heads, dim, device="cuda", dtype=torch.bfloat16) for _ in range(2)] for _ in stack]
    g = torch.Generator(device="cuda").manual_seed(1)
    for step in range(20):
        x = torch.randn(batch, hidden, device="cuda", generator=g).bfloat16()
        cache.grow()
        h, z, hp, zp = x.clone(), x.clone(), x.clone(), x.clone()
        for i, layer in enumerate(stack):
            z = layer.step(h, z, cache, i)
            room = torch.zeros(batch, 1, kv_heads, dim, device="cuda", dtype=torch.bfloat16)
            dense[i] = [torch.cat((t, room), 1) for t in dense[i]]
            hp, zp = layer.plain_step(hp, zp, *dense[i])
        for got, want in ((h, hp), (z, zp)):
            assert float((got.float() - want.float()).norm() / want.float().norm()) < 0.02, step
    import dnnopt_b200 as dn
    assert dn.stream_status(torch.cuda.current_stream()) == dn.SUCCESS


@pytest.mark.gpu
def test_step_in_a_graph(torch_cuda, decode):
    """A captured step generates what eager steps do, lengths and pages growing between replays."""
    c = decode.LayerConfig(256, 8, 2, 64, 512)
    layer = decode.DecoderLayer(c)
    caches = [decode.PagedCache(2, 2, 64, pages=8, page_size=16, max_pages=4) for _ in range(2)]
    x = torch.randn(2, 256, device="cuda").bfloat16()
    h = x.clone()
    side = torch.cuda.Stream()
    caches[0].grow()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):       # first calls on the stream allocate its workspace
        layer.step(h, x, caches[0], 0)
    side.synchronize()
    caches[0].release(0)
    caches[0].release(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        z = layer.step(h, x, caches[0], 0)
    for step in range(20):
        x.copy_(torch.randn(2, 256))
        for cache in caches:
            cache.grow()
        h.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        want_h = x.clone()
        want_z = layer.step(want_h, x, caches[1], 0)
        assert torch.equal(h, want_h) and torch.equal(z, want_z), step
