"""GPU tests of what the decoder-step operators promise beside their results: what they report, what
they leave alone, what captured graphs may rely on."""
from __future__ import annotations

import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(torch_cuda, dn):
    return torch_cuda


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("max_pages", [0, 4])
@pytest.mark.parametrize("lens", [[5], [5, 0, 0], [0] * 40 + [64, 1]])
def test_lengths_without_pages(gpu, dn, cache, max_pages, lens):
    """A cache without pages has no table to read: lengths above 0 are reported, all outputs are those
    of empty sequences."""
    torch = gpu
    io = torch.float32 if cache == "f32" else torch.bfloat16
    kinds = {"bf16": dn.TYPE_BF16, "e4m3": dn.TYPE_E4M3, "f32": dn.TYPE_F32}
    s = torch.cuda.current_stream()
    assert dn.stream_status(s) == dn.SUCCESS
    B = len(lens)
    q = torch.randn(B, 4, 64, device="cuda").to(io)
    new = torch.randn(B, 2, 64, device="cuda").to(io)
    d = dn.paged_attn_desc(B, 4, 2, 64, 16, 0, max_pages, io_type=kinds["f32" if cache == "f32" else "bf16"],
                           cache_type=kinds[cache])
    for append in (None, new):
        out, lse = torch.full_like(q, 7.0), torch.full((B, 4), 7.0, device="cuda")
        dn.check(dn.cuda_paged_attention(d, q, None, None, None, torch.tensor(lens, dtype=torch.int32).cuda(), out,
                                         lse=lse, k_new=append, v_new=append, stream=s))
        assert dn.stream_status(s) == dn.INVALID_VALUE
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())
        assert dn.stream_status(s) == dn.SUCCESS
