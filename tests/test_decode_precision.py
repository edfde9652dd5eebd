"""GPU tests of what the decoder-step operators keep of their numbers' bits.

Inputs are made so that sums and products that a 32-bit computation would keep
come out alone: a lost digit shows far above the tolerance, which is derived
from FP32 roundings, u = 2^-24 each, and not from the length of the sums.
"""
from __future__ import annotations

import math

import pytest

from test_decode_ops import Paged, U, r_of, types

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gpu(torch_cuda, dn):
    return torch_cuda


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("heads,dim", [(1, 64), (8, 128), (16, 128), (16, 256)])
@pytest.mark.parametrize("second", [1.125, 1.5, 1.625, 1.75])
def test_attention_weights_keep_their_bits(gpu, dn, cache, heads, dim, second):
    """Two tokens whose weighted values cancel: what is left is the error of the weights.

    Scores are 0 and -log(second) from one exact product, values -1 and `second`.
    Scaling the score and adding up in units of log 2 take three roundings of
    |s| < 1, exp is good to 2^-22, each of up to three partial products is added
    with at most 2u and the division takes 2u: in all below 2^-20 of the sum of
    p |v|.  Weights of 16 bits would be off by 2^-18 of half of it."""
    torch = gpu
    p = Paged(torch, dn, [2], heads, 1, dim, 16, cache, scale=math.log(second))
    t = types(torch, dn)[cache][0]
    p.q = torch.zeros_like(p.q)
    p.q[..., 0] = 1.0
    page = int(p.table[0, 0])
    k, v = torch.zeros(2, dim), torch.empty(2, dim)
    k[1, 0], v[0], v[1] = -1.0, -1.0, second
    for c, rows in ((p.k, k), (p.v, v)):
        c[page, :2, 0] = rows.to(t).cuda()
    out, lse = p.run()
    s = float(torch.tensor(math.log(second), dtype=torch.float32))
    w = math.exp(-s)
    want = (w * second - 1.0) / (1.0 + w)
    size = (w * second + 1.0) / (1.0 + w)
    off = float((out.double() - want).abs().max())
    assert off <= r_of(torch, p.q.dtype) * abs(want) + 2.0 ** -20 * size, off / size * 2.0 ** 20
    assert float((lse.double() - math.log1p(w)).abs().max()) <= 2.0 ** -20
