"""GPU tests of what the decoder-step operators keep of their numbers' bits.

Inputs are made so that sums and products that a 32-bit computation would keep
come out alone: a lost digit shows far above the tolerance, which is derived
from FP32 roundings, u = 2^-24 each, and not from the length of the sums.
"""
from __future__ import annotations

import math

import pytest

from test_decode_ops import Paged, U, r_of, types, w4_inputs, w4_run

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



@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("heads,dim", [(1, 64), (8, 64), (8, 128), (8, 256), (16, 64), (16, 128), (16, 256)])
def test_attention_sums_do_not_drift(gpu, dn, cache, heads, dim):
    """One CTA's sum of 65536 values 1/4, and of 64 values that take it back to about zero.

    Their weights are of all sizes, next to 64 tokens of value 0 that come first and weigh most.  Each of
    the four warps adds 1025 numbers, each sum rounded within u of its part of half the sum of p |v| and
    of random sign: 6 sqrt(1025) u is beyond six standard deviations.  Where matrix units add to what they
    truncate, they do so for 1024 tokens, 64 times up to three parts: 192 times up to 2u of sums that are
    half of their last on average.  Over all tokens the truncations would take ten times that."""
    torch = gpu
    t = types(torch, dn)
    pages, page, batch = 1026, 64, 450      # enough sequences that each has a CTA; all of them read the same pages
    io, kind = t["f32" if cache == "f32" else "bf16"], t[cache]
    g = torch.Generator(device="cuda").manual_seed(dim)
    k = torch.zeros(pages, page, 1, dim, device="cuda")
    k[..., 0] = -torch.randn(pages, page, 1, device="cuda", generator=g).abs()
    k[0, ..., 0] = 0.5
    k, L = k.to(kind[0]), pages * page
    w = torch.exp(k[..., 0, 0].double()).cpu()
    x = torch.full((pages, page), 0.25, dtype=torch.float64)
    x[0] = 0.0
    left = float((w[1:-1] * x[1:-1]).sum())
    for i in range(page):
        x[-1, i] = float(torch.tensor(-left / float(w[-1, i:].sum())).to(kind[0]))
        left += float(w[-1, i] * x[-1, i])
    want, size = left / float(w.sum()), float((w * x.abs()).sum() / w.sum())
    assert abs(want) < 2.0 ** -9 and 0.45 < size < 0.55
    v = x.float().cuda()[:, :, None, None].expand(-1, -1, 1, dim).contiguous().to(kind[0])
    q = torch.zeros(batch, heads, dim, device="cuda", dtype=io[0])
    q[..., 0] = 1.0
    table = torch.arange(pages, device="cuda", dtype=torch.int32).expand(batch, -1).contiguous()
    lens = torch.full((batch,), L, device="cuda", dtype=torch.int32)
    out = torch.empty_like(q)
    d = dn.paged_attn_desc(batch, heads, 1, dim, page, pages, pages, io_type=io[1], cache_type=kind[1], scale=1.0)
    dn.check(dn.cuda_paged_attention(d, q, k, v, table, lens, out, stream=torch.cuda.current_stream()))
    off = float((out.double() - want).abs().max())
    drift = 192 if cache == "e4m3" or cache == "bf16" and dim > 128 else 0
    tol = r_of(torch, io[0]) * abs(want) + (6 * math.sqrt(L / 64) + drift) * U * size / 2
    assert off <= tol, (off / (U * size / 2), tol / (U * size / 2))


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("heads,kv,dim", [(2, 2, 64), (8, 1, 128), (8, 1, 256), (32, 2, 128), (16, 1, 256)])
@pytest.mark.parametrize("rise", [60.0, -60.0])
def test_attention_over_long_sequences_of_one_cta(gpu, dn, cache, heads, kv, dim, rise):
    """Scores that rise (or fall) by far more than the reference of exp tolerates while a CTA works on one
    sequence of ten runs of sums: what was put aside is brought to the new reference, item after item.

    Sums as in the tests of other lengths; the scores' products are exact but for their scaling."""
    torch = gpu
    t = types(torch, dn)
    pages, page, batch = 640, 64, 240
    io, kind = t["f32" if cache == "f32" else "bf16"], t[cache]
    g = torch.Generator(device="cuda").manual_seed(dim + heads)
    L = pages * page - 5
    k = torch.zeros(pages, page, kv, dim, device="cuda")
    k[..., 0] = torch.linspace(0, 1, pages * page, device="cuda").view(pages, page, 1) + 0.05 * torch.randn(
        pages, page, kv, device="cuda", generator=g)
    k = k.to(kind[0])
    v = torch.randn(pages, page, kv, dim, device="cuda", generator=g).to(kind[0])
    q = torch.zeros(batch, heads, dim, device="cuda", dtype=io[0])
    q[..., 0] = 1.0
    q[:, 1::2, 0] = 0.5
    table = torch.arange(pages, device="cuda", dtype=torch.int32).expand(batch, -1).contiguous()
    lens = torch.full((batch,), L, device="cuda", dtype=torch.int32)
    out, lse = torch.empty_like(q), torch.empty(batch, heads, device="cuda")
    d = dn.paged_attn_desc(batch, heads, kv, dim, page, pages, pages, io_type=io[1], cache_type=kind[1], scale=rise)
    dn.check(dn.cuda_paged_attention(d, q, k, v, table, lens, out, lse=lse, stream=torch.cuda.current_stream()))
    k64, v64 = k.view(-1, kv, dim)[:L].double(), v.view(-1, kv, dim)[:L].double()
    for h in range(heads):
        s = rise * float(q[0, h, 0]) * k64[:, h // (heads // kv), 0]
        total = torch.logsumexp(s, 0)
        p = torch.exp(s - total)
        values = v64[:, h // (heads // kv)]
        want, size = p @ values, p @ values.abs()
        score = 8 * U * float(s.abs().max())
        tol = r_of(torch, io[0]) * want.abs() + (2.2 * score + 2.0 ** -16) * size
        assert bool(((out[:, h].double() - want).abs() <= tol).all()), h
        assert bool(((lse[:, h].double() - total).abs() <= score + 2.0 ** -16).all()), h


# ------------------------------------------------------------------ gemm_w4
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(2, 127, 128), (8, 127, 128), (4, 8192, 4096), (8, 8192, 4096)])
def test_w4_activations_next_to_large_ones(gpu, dn, M, N, K, io):
    """Each column of C is one activation as it is held next to the largest of its 128: exact from 2^-14
    (BF16; 2^-6, FP32) of that, else within 2^-22 (2^-30) of it, or 2^-127.  What is held fits C's type.

    Row m's largest is a power of two, where the bound is sharp; it stands alone, so that nothing is summed."""
    torch = gpu
    f32 = io == "f32"
    tops = [0, 5, -90, 60, -20, 1, -97, 100] if f32 else [0, 5, -90, 60, -20, 1, -105, 100]
    T = types(torch, dn)[io][0]
    g = torch.Generator().manual_seed(M)
    A = torch.zeros(M, K, dtype=torch.float64)
    for m in range(M):
        down = torch.rand(127, generator=g, dtype=torch.float64) * 40 if f32 else torch.rand(127, generator=g, dtype=torch.float64) * 30
        A[m, 1:128] = 2.0 ** (tops[m] - down) * torch.where(torch.rand(127, generator=g) < 0.5, -1.0, 1.0)
        A[m, 0] = 2.0 ** tops[m]
    A = A.to(T).cuda()
    at = 1 + torch.arange(N) % 127
    codes = torch.full((N, K), 8, dtype=torch.uint8)
    codes[torch.arange(N), at] = 9
    W = (codes[:, 0::2] | codes[:, 1::2] << 4).cuda()
    C = w4_run(torch, dn, M, N, K, 128, A, W, torch.ones(N, -(-K // 128), device="cuda"), None, None)
    want = A.double().cpu()[:, at]
    top = A.double().cpu()[:, :1]
    held, low = (2.0 ** -30, 2.0 ** -6) if f32 else (2.0 ** -22, 2.0 ** -14)
    tol = torch.where(want.abs() >= low * top, torch.zeros(1, dtype=torch.float64), torch.clamp(held * top, min=2.0 ** -127))
    off = (C.double().cpu() - want).abs()
    assert bool((off <= tol).all()), float((off / top).max())


# Rows and groups that take each form of the kernels: digits of one or two rows side by side, digits apart
# with scales for 32, 64 and 128 weights, and codes in tensor memory for up to four and eight rows.
W4_FORMS = [(2, 70, 700, 32), (2, 70, 700, 64), (2, 70, 700, 128), (5, 70, 700, 32), (5, 70, 700, 64), (5, 70, 700, 128),
            (4, 8193, 4097, 128), (8, 8193, 4097, 128)]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", W4_FORMS)
def test_w4_scales_with_its_operands(gpu, dn, M, N, K, group, io, zeros):
    """Activations and scales times powers of two give the product times these, to the bit: every step
    is exact under them while nothing leaves FP32's normal numbers, as no result here does.

    The largest of 128 normal activations is between 1 and 8, so that its unit, 2^-30 (FP32) or 2^-22 of
    it, is a normal number down to activations of 2^-97 and 2^-104; results are above 2^-124 but where
    their terms cancel to 2^-24 of themselves."""
    torch = gpu
    A, W, scale, zero, _ = w4_inputs(torch, M, N, K, group, types(torch, dn)[io][0], torch.float32, zeros, False)
    want = w4_run(torch, dn, M, N, K, group, A, W, scale, zero, None)
    for a, s in ((-85, 0), (-60, -30), (-85, -10), (0, -60), (60, -30), (80, 20)):
        C = w4_run(torch, dn, M, N, K, group, A * 2.0 ** a, W, scale * 2.0 ** s, zero, None)
        assert torch.equal(C.double(), want.double() * 2.0 ** (a + s)), (a, s)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", W4_FORMS + [(2, 70, 28700, 128), (8, 70, 9000, 32), (7, 1009, 28700, 256), (9, 8192, 20000, 128)])
def test_w4_whole_numbers_are_exact(gpu, dn, M, N, K, group, io, zeros):
    """Every digit of an activation counts, at its worth: no rounding but C's own.

    A row of A is whole numbers |v| < 32 times 2^s, next to one 2^29 (BF16: 2^21) in each 128 whose weight
    is 0: so 1 is the unit in which the row is held, and v lies s bits above it, s going through all digits.
    Sums of (code - zero) v 2^s are below 2^(5 + 4 + 15 - 1) 2^s, scales 1, 2 or 4: multiples of 2^s with 24 bits
    for K <= 8192 and less for the random signs of longer rows.  With zero points the sums of all
    activations of 128, 2^29 among them, are also multiples of 2^s, with 24 bits from s = 12 (4) on."""
    torch = gpu
    f32 = io == "f32"
    T = types(torch, dn)[io][0]
    top = 29 if f32 else 21
    lowest = (12 if f32 else 4) if zeros else 0
    g = torch.Generator().manual_seed(K + M)
    G = -(-K // group)
    at = torch.arange(K) // group
    z = torch.randint(0, 16, (N, G), generator=g) if zeros else torch.full((N, G), 8)
    codes = torch.randint(0, 16, (N, K), generator=g)
    tops = torch.arange(0, K, 128) + torch.randint(0, 128, (-(-K // 128),), generator=g)
    tops = tops[tops < K]
    codes[:, tops] = z[:, at[tops]]
    padded = torch.zeros(N, -(-K // 32) * 32, dtype=torch.uint8)
    padded[:, :K] = codes.to(torch.uint8)
    W = (padded[:, 0::2] | padded[:, 1::2] << 4).cuda()
    scale = 2.0 ** torch.randint(0, 3, (N, G), generator=g)
    weight = ((codes - z[:, at]) * scale[:, at]).double()
    v = torch.randint(-31, 32, (M, K), generator=g).double()
    v[:, tops] = 0.0
    sums = v @ weight.t()
    assert float(sums.abs().max()) < 2.0 ** 24
    zt = z.float().cuda() if zeros else None
    for first in range(lowest, top - 5, M):
        s = torch.tensor([lowest + (first - lowest + m) % (top - 5 - lowest) for m in range(M)], dtype=torch.float64)[:, None]
        A = v * 2.0 ** s
        A[:, tops] = 2.0 ** top
        C = w4_run(torch, dn, M, N, K, group, A.to(T).cuda(), W, scale.cuda(), zt, None)
        want = (sums * 2.0 ** s).to(torch.float32).to(T)
        assert torch.equal(C.cpu(), want), first


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(2, 1009, 8192, 128), (5, 1009, 8192, 64), (4, 100, 28672, 32), (8, 4096, 4096, 128),
                                         (1, 33, 65000, 0), (9, 700, 20000, 96)])
def test_w4_infinities_across_parts(gpu, dn, M, N, K, group, io, zeros):
    """Infinities and NaN anywhere in K, where rows of W are cut into parts and K into ranges: they reach
    their own rows of C as the formula says, and no other."""
    torch = gpu
    A, W, scale, zero, _ = w4_inputs(torch, M, N, K, group, types(torch, dn)[io][0], torch.float32, zeros, False)
    clean = w4_run(torch, dn, M, N, K, group, A, W, scale, zero, None)
    codes = torch.stack((W & 15, W >> 4), 2).view(N, -1)[:, :K].double().cpu()
    at = torch.arange(K) // (group or K)
    sign = (codes - (zero.double().cpu()[:, at] if zeros else 8.0)) * scale.double().cpu()[:, at]
    inf, nan = float("inf"), float("nan")
    spots = [0, 1, 31, 127, 128, K // 2 - 1, K // 2, K // 2 + 1, K - 129, K - 2, K - 1] + list(range(500, K, 4097))
    for i, k in enumerate(spots):
        m, value = i % M, (inf, -inf, nan)[i % 3 if i % 7 == 2 else i % 2]
        B = A.clone()
        B[m, k] = value
        want = clean.clone()
        want[m] = (value * sign[:, k]).to(clean.dtype).cuda()      # inf * 0 is NaN
        if i % 5 == 4:      # two of them
            B[m, (k + 777) % K] = inf
            want[m] = (value * sign[:, k] + inf * sign[:, (k + 777) % K]).to(clean.dtype).cuda()
        C = w4_run(torch, dn, M, N, K, group, B, W, scale, zero, None)
        assert bool(((C == want) | (C.isnan() & want.isnan())).all()), (m, k, value)
