"""What dnn-opt_b200/decode.py takes and refuses.  CPU but for the step over an E4M3 cache."""
from __future__ import annotations

import pytest
import torch


@pytest.fixture(scope="module")
def decode(dn):
    import dnnopt_b200.decode as module
    return module


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.uint8])
def test_cache_types(decode, dtype):
    with pytest.raises(ValueError):
        decode.PagedCache(1, 1, 16, pages=2, page_size=4, max_pages=2, dtype=dtype, device="cpu")


def test_linear_inputs(decode):
    linear = decode.W4Linear(torch.randn(8, 64), 32)
    rows = torch.randn(4, 64).bfloat16()
    for x in (rows.float(), rows.half(), rows[:, :32], rows[0], rows.t().contiguous().t(), rows[:1].expand(4, 64)):
        with pytest.raises(ValueError):
            linear(x)


def test_step_inputs(decode):
    c = decode.LayerConfig(64, 2, 1, 16, 64, group=32)
    layer = decode.DecoderLayer(c, device="cpu")
    cache = decode.PagedCache(2, 1, 16, pages=4, page_size=4, max_pages=2, device="cpu")
    x = torch.randn(2, 64).bfloat16()
    for h, z in ((x.float(), x), (x, x.float()), (x[:1], x[:1]), (torch.cat((x, x)), torch.cat((x, x))),
                 (torch.cat((x, x), 1)[:, :64], x), (x, torch.cat((x, x), 1)[:, ::2])):
        with pytest.raises(ValueError):
            layer.step(h, z, cache, 0)
    for kv_heads, dim in ((2, 16), (1, 32)):
        other = decode.PagedCache(2, kv_heads, dim, pages=4, page_size=4, max_pages=2, device="cpu")
        with pytest.raises(ValueError):
            layer.step(x, x, other, 0)


def test_ended_slots_stay_empty(decode):
    c = decode.PagedCache(3, 1, 16, pages=5, page_size=4, max_pages=2, device="cpu")
    c.grow(4)
    c.release(1)
    free = list(c.free)
    c.grow(1, slots=[0, 2, 2])
    assert c.lens.tolist() == [5, 0, 5] and c.held[1] == [] and len(c.free) == len(free) - 2
    assert c.table[1].tolist() == [-1, -1] and sorted(c.table[[0, 2]].flatten().tolist()) == sorted(c.held[0] + c.held[2])
    c.grow(1, slots=[])
    assert c.lens.tolist() == [5, 0, 5]
    c.grow(4, slots=(1,))
    assert c.lens.tolist() == [5, 4, 5] and len(c.held[1]) == 1
    for slots in ([3], [-1]):
        with pytest.raises(IndexError):
            c.grow(1, slots=slots)


def test_growing_without_pages_changes_nothing(decode):
    c = decode.PagedCache(3, 1, 16, pages=5, page_size=4, max_pages=2, device="cpu")
    c.grow(4)
    before = c.lens.tolist(), c.table.tolist(), list(c.free), [list(h) for h in c.held]
    for tokens, slots in ((1, None), (5, [0]), (9, [1])):     # three pages of two; past max_pages
        with pytest.raises(RuntimeError):
            c.grow(tokens, slots=slots)
        assert before == (c.lens.tolist(), c.table.tolist(), list(c.free), [list(h) for h in c.held])
    c.grow(1, slots=[0, 1])
    assert c.lens.tolist() == [5, 5, 4] and c.free == []


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (4, 4, 128)])
def test_steps_over_an_e4m3_cache(torch_cuda, decode, heads, kv_heads, dim):
    """Keys and values of one byte, stored and read at their own places.  Both sides round to bf16 at the
    same places and to E4M3 when they store: a key or value on a rounding boundary differs by 2^-4 of
    itself, 1 in some hundred does, which stays within 2 % of the whole."""
    import dnnopt_b200 as dn
    B, tokens = 3, 40
    c = decode.LayerConfig(256, heads, kv_heads, dim, 512)
    layer = decode.DecoderLayer(c)
    cache = decode.PagedCache(B, kv_heads, dim, pages=B * 3, page_size=16, max_pages=3, dtype=torch.float8_e4m3fn)
    dense = [torch.zeros(B, tokens, kv_heads, dim, device="cuda", dtype=torch.float8_e4m3fn) for _ in range(2)]
    g = torch.Generator(device="cuda").manual_seed(2)
    for n in range(1, tokens + 1):
        x = torch.randn(B, 256, device="cuda", generator=g).bfloat16()
        cache.grow()
        h = x.clone()
        z = layer.step(h, x, cache, 0)
        want_h, want_z = layer.plain_step(x, x, *[t[:, :n] for t in dense])
        for got, want in ((h, want_h), (z, want_z)):
            assert float((got.float() - want.float()).norm() / want.float().norm()) < 0.02, n
    assert dn.stream_status(torch.cuda.current_stream()) == dn.SUCCESS
    for stored, want in zip((cache.k[0], cache.v[0]), dense):
        rows = stored.view(torch.uint8)[cache.table.long()].view(B, -1, kv_heads, dim)[:, :tokens].view(torch.float8_e4m3fn)
        assert float((rows.float() - want.float()).norm() / want.float().norm()) < 0.02
