"""GPU tests of the decoder-step operators against plain 64-bit implementations.

Tolerances, with u = 2^-24 (half an FP32 ulp) and r = the output type's half
ulp (2^-24 for FP32, 2^-9 for BF16):

* A sum of n products accumulated in FP32 16 at a time, truncated at worst, is
  off by at most (n / 16) * 2u per unit of its sum of magnitudes S, plus
  roundings of random sign, six standard deviations of which are below
  6 sqrt(n) * 2u * S.  sum_tol(n) = (n / 16 + 6 sqrt(n)) * 2u.
* Attention: a score's error d = sum_tol(D) * sum |q k| * |scale| (plus its
  capping and scaling, 8u * |s|) changes each weight exp(s - lse) by at most a
  factor of 1 + 2.2 d, exp itself is good to 2^-20, and weights enter the
  product with the values as two BF16 parts (2^-17).  So out is off by at most
  r |out| + (2.2 max d + 2^-16 + sum_tol(L)) * sum p |v|, and lse by
  max d + 2^-20 + sum_tol(L) + 4u |lse|.
* Norms: a handful of FP32 operations on each element, and row sums whose
  relative error is below sum_tol(cols): h is off by at most r |h| +
  16u * (|rs x| + |bs g post|) + the post-norm's share, z likewise.

Outputs of BF16 type get r = 2^-8: a value within the computed error of a
rounding boundary may round the other way.
"""
from __future__ import annotations

import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def sum_tol(n):
    return (n / 16 + 6 * math.sqrt(n)) * 2 * U


def r_of(torch, t):
    return 2 * U if t == torch.float32 else 2.0 ** -8


@pytest.fixture(scope="module")
def gpu(torch_cuda, dn):
    return torch_cuda


def types(torch, dn):
    return {"f32": (torch.float32, dn.TYPE_F32), "bf16": (torch.bfloat16, dn.TYPE_BF16),
            "e4m3": (torch.float8_e4m3fn, dn.TYPE_E4M3)}


def within(got, want, tol, what=""):
    """|got - want| <= tol everywhere, infinities and NaN in the same places."""
    got, want = got.double().cpu(), want.double().cpu()
    tol = tol.double().cpu() if hasattr(tol, "cpu") else tol
    bad = ~((got == want) | ((got - want).abs() <= tol) | (got.isnan() & want.isnan()))
    if bad.any():
        i = bad.nonzero()[0].tolist()
        raise AssertionError(f"{what} {int(bad.sum())} of {bad.numel()} off, first at {i}: "
                             f"{got[tuple(i)]} for {want[tuple(i)]}")


# ------------------------------------------------------------------- gemm_w4
def w4_inputs(torch, M, N, K, group, io, st, zeros, bias, pad=0, seed=0, pitch=16, ldw=None):
    g = torch.Generator().manual_seed(seed)
    G = -(-K // group) if group else 1
    ldw = ldw or -(-((K + 1) // 2) // pitch) * pitch
    A = torch.randn(M, K + pad, generator=g).to(io).cuda()
    W = torch.randint(0, 256, (N, ldw), generator=g, dtype=torch.uint8).cuda()
    scale = (torch.rand(N, G + pad, generator=g) * 0.02 + 0.002).to(st).cuda()
    zero = (torch.rand(N, G + pad, generator=g) * 6 + 5).to(st).cuda() if zeros else None
    b = torch.randn(N, generator=g).cuda() if bias else None
    return A, W, scale, zero, b


def w4_exact(torch, A, W, scale, zero, bias, K, group):
    """(C, sum of magnitudes) in 64 bits."""
    A, W = A[:, :K].double().cpu(), W.cpu()
    code = torch.stack((W & 15, W >> 4), 2).reshape(W.shape[0], -1)[:, :K].double()
    at = torch.arange(K) // (group or K)
    z = zero.double().cpu()[:, at] if zero is not None else torch.full_like(code, 8.0)
    s = scale.double().cpu()[:, at]
    C = A @ ((code - z) * s).t()
    mag = A.abs() @ ((code + z.abs()) * s.abs()).t()
    if bias is not None:
        C = C + bias.double().cpu()
        mag = mag + bias.abs().double().cpu()
    return C, mag


def w4_run(torch, dn, M, N, K, group, A, W, scale, zero, bias, pad_c=0, stream=None, want=None):
    kinds = {torch.float32: dn.TYPE_F32, torch.bfloat16: dn.TYPE_BF16}
    C = torch.full((M, N + pad_c), float("nan"), device="cuda", dtype=A.dtype)
    d = dn.w4_desc(M, N, K, A.stride(0), W.stride(0), N + pad_c, group, scale.stride(0),
                   kinds[A.dtype], kinds[scale.dtype])
    dn.check(dn.cuda_gemm_w4(d, A, W, scale, zero, bias, C, stream or torch.cuda.current_stream()))
    return C


def w4_check(torch, dn, M, N, K, group, io="bf16", st="bf16", zeros=False, bias=False, pad=0, pitch=16,
             seed=0, ldw=None):
    t = types(torch, dn)
    ins = w4_inputs(torch, M, N, K, group, t[io][0], t[st][0], zeros, bias, pad, seed, pitch, ldw)
    C = w4_run(torch, dn, M, N, K, group, *ins, pad_c=pad)
    want, mag = w4_exact(torch, *ins, K, group)
    within(C[:, :N], want, r_of(torch, t[io][0]) * want.abs() + sum_tol(K) * mag, f"{M}x{N}x{K}")
    assert bool(C[:, N:].isnan().all())     # columns past N are left alone
    return ins, C


@pytest.mark.parametrize("io,st", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("M", [1, 2, 3, 5, 8, 9, 16, 33])
def test_w4_types_and_rows(gpu, dn, io, st, M):
    w4_check(gpu, dn, M, 257, 1024, 128, io, st, zeros=M % 2 == 0, bias=M % 3 == 0)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 160, 256, 512, 0])
@pytest.mark.parametrize("K", [1, 2, 31, 33, 127, 129, 1000, 2048, 4099])
def test_w4_groups_and_lengths(gpu, dn, K, group, zeros):
    w4_check(gpu, dn, 3, 97, K, group, "f32" if K % 2 else "bf16", "f32", zeros=zeros, bias=True)


@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 100, 1009, 4093])
def test_w4_widths(gpu, dn, N):
    w4_check(gpu, dn, 2, N, 640, 64, zeros=True)


@pytest.mark.parametrize("M,N,K,group,io", [(1, 4096, 8192, 128, "bf16"), (8, 640, 16384, 32, "bf16"),
                                            (8, 300, 28672, 128, "f32"), (64, 130, 4096, 128, "bf16"),
                                            (1, 16, 65536 + 64, 0, "f32"), (4, 20000, 512, 64, "bf16")])
def test_w4_long(gpu, dn, M, N, K, group, io):
    w4_check(gpu, dn, M, N, K, group, io, "f32" if io == "f32" else "bf16", zeros=True)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("K,pitch,pad", [(1023, 1, 0), (1024, 1, 3), (1000, 4, 1), (640, 16, 5), (640, 64, 8)])
def test_w4_pitches(gpu, dn, K, pitch, pad, io):
    w4_check(gpu, dn, 5, 77, K, 32, io, "f32", zeros=True, bias=True, pad=pad, pitch=pitch)


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K,group,io,pitch", [(3, 8195, 4099, 128, "bf16", 16), (4, 8192, 4096, 256, "f32", 16),
                                                  (5, 9000, 4000, 0, "bf16", 1), (8, 8321, 4225, 128, "f32", 16),
                                                  (9, 8192, 12289, 128, "bf16", 64), (8, 8200, 20000, 1024, "f32", 16),
                                                  (17, 65600, 513, 128, "bf16", 16), (4, 33000, 1025, 384, "f32", 1)])
def test_w4_long_products(gpu, dn, M, N, K, group, io, pitch, zeros):
    """Products of 2^25 weights and more: the first and last rows of W and some between."""
    torch = gpu
    t = types(torch, dn)
    A, W, scale, zero, bias = w4_inputs(torch, M, N, K, group, t[io][0], torch.float32 if zeros else torch.bfloat16,
                                        zeros, True, pitch=pitch)
    C = w4_run(torch, dn, M, N, K, group, A, W, scale, zero, bias, pad_c=3)
    rows = torch.cat((torch.arange(140), torch.randint(0, N, (200,), generator=torch.Generator().manual_seed(1)),
                      torch.arange(N - 140, N))).cuda()
    want, mag = w4_exact(torch, A, W[rows], scale[rows], None if zero is None else zero[rows], bias[rows], K, group)
    within(C[:, rows], want, r_of(torch, t[io][0]) * want.abs() + sum_tol(K) * mag, f"{M}x{N}x{K}")
    assert bool(C[:, N:].isnan().all())
    assert bool(C[:, :N].isfinite().all())
    assert torch.equal(C[:, :N], w4_run(torch, dn, M, N, K, group, A, W, scale, zero, bias))
    # An infinity and a NaN reach their own rows.
    clean = C[:, :N].clone()
    A[1, K - 1], A[2, 700 % K] = float("inf"), float("nan")
    C = w4_run(torch, dn, M, N, K, group, A, W, scale, zero, bias)
    keep = [m for m in range(M) if m not in (1, 2)]
    assert torch.equal(C[keep], clean[keep])
    last = (W[:, (K - 1) // 2] >> (4 * ((K - 1) % 2))) & 15
    sign = last.float() - (8.0 if zero is None else zero[:, (K - 1) // group if group else 0].float())
    some = sign != 0
    assert torch.equal(C[1, some].float(), torch.where(sign > 0, float("inf"), -float("inf"))[some])
    assert bool(C[1, ~some].isnan().all()) and bool(C[2].isnan().all())


def test_w4_unaligned_bases(gpu, dn):
    """Operands that start one element into their allocation."""
    torch = gpu
    M, N, K = 4, 130, 512
    A, W, scale, zero, bias = w4_inputs(torch, M, N, K, 64, torch.bfloat16, torch.bfloat16, True, True)
    want, mag = w4_exact(torch, A, W, scale, zero, bias, K, 64)

    def moved(t):
        flat = torch.empty(t.numel() + 1, device="cuda", dtype=t.dtype)
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    for which in range(5):
        ops = [A, W, scale, zero, bias]
        ops[which] = moved(ops[which])
        C = w4_run(torch, dn, M, N, K, 64, *ops)
        within(C, want, 2.0 ** -8 * want.abs() + sum_tol(K) * mag, f"operand {which}")


def test_w4_same_bits_each_time(gpu, dn):
    torch = gpu
    for M, N, K, io in ((1, 1009, 8192, torch.bfloat16), (5, 4096, 4096, torch.float32)):
        ins = w4_inputs(torch, M, N, K, 128, io, torch.float32, True, False)
        first = w4_run(torch, dn, M, N, K, 128, *ins)
        for _ in range(3):
            assert torch.equal(first, w4_run(torch, dn, M, N, K, 128, *ins))


def test_w4_infinite_and_nan_activations(gpu, dn):
    """Infinities and NaN reach their own row of C and no other."""
    torch = gpu
    M, N, K = 4, 64, 256
    for io in (torch.bfloat16, torch.float32):
        A, W, scale, zero, bias = w4_inputs(torch, M, N, K, 32, io, torch.float32, True, False)
        clean = w4_run(torch, dn, M, N, K, 32, A, W, scale, zero, bias)
        A[1, 7], A[2, 100] = float("inf"), float("nan")
        C = w4_run(torch, dn, M, N, K, 32, A, W, scale, zero, bias)
        assert torch.equal(C[0], clean[0]) and torch.equal(C[3], clean[3])
        code = (W[:, 3] >> 4).float() - zero[:, 0]
        want = torch.where(code > 0, float("inf"), -float("inf"))
        assert torch.equal(C[1].float(), want)
        assert bool(C[2].isnan().all())


def test_w4_extreme_activations(gpu, dn):
    """FP32 activations over the whole range keep all their bits."""
    torch = gpu
    K = 64
    A = torch.zeros(3, K)
    A[0, 5], A[1, 6], A[2, 7] = 3.4e38, 1.17e-30, 1.0 + 2.0 ** -23
    A = A.cuda()
    W = torch.full((16, 32), 0x99, dtype=torch.uint8, device="cuda")     # every weight is 1
    scale = torch.ones(16, 2, device="cuda")
    C = w4_run(torch, dn, 3, 16, K, 32, A, W, scale, None, None)
    for m, k in ((0, 5), (1, 6), (2, 7)):
        assert bool((C[m] == A[m, k]).all()), m


def test_w4_offsets_past_32_bits(gpu, dn):
    """Rows of W that start beyond 2^31 bytes."""
    torch = gpu
    N, K, ldw = 70000, 64, 32768
    W = torch.empty(N, ldw, dtype=torch.uint8, device="cuda")
    W[:, :32] = torch.randint(0, 256, (N, 32), device="cuda", dtype=torch.uint8)
    A = torch.randn(2, K, device="cuda").bfloat16()
    scale = torch.rand(N, 2, device="cuda")
    C = w4_run(torch, dn, 2, N, K, 32, A, W, scale, None, None)
    rows = torch.tensor([0, 1, 65535, 65536, 69999])
    want, mag = w4_exact(torch, A, W[rows.cuda(), :32], scale[rows.cuda()], None, None, K, 32)
    within(C[:, rows.cuda()], want, 2.0 ** -8 * want.abs() + sum_tol(K) * mag)


def test_w4_other_stream_and_graph(gpu, dn):
    torch = gpu
    M, N, K = 4, 1009, 2048
    ins = w4_inputs(torch, M, N, K, 64, torch.bfloat16, torch.bfloat16, False, True)
    want = w4_run(torch, dn, M, N, K, 64, *ins)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        C = w4_run(torch, dn, M, N, K, 64, *ins, stream=side)
    side.synchronize()
    assert torch.equal(C, want)
    g = torch.cuda.CUDAGraph()
    out = torch.empty_like(want)
    d = dn.w4_desc(M, N, K, K, ins[1].stride(0), N, 64, ins[2].stride(0))
    with torch.cuda.graph(g, stream=side):
        dn.check(dn.cuda_gemm_w4(d, ins[0], ins[1], ins[2], None, ins[4], out, side))
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


# ------------------------------------------------------- paged attention
class Paged:
    """A random paged cache and its 64-bit attention.

    Everything outside the sequences' tokens is poisoned with NaN or infinities,
    and unused table entries point nowhere."""

    def __init__(self, torch, dn, lens, heads, kv_heads, dim, page, cache="bf16", layout="token", seed=0,
                 append=False, window=0, softcap=0.0, k_scale=1.0, v_scale=1.0, scale=None, poison="nan",
                 spare=3, wide=2, share=None):
        self.torch, self.dn, self.lens = torch, dn, list(lens)
        self.io = "f32" if cache == "f32" else "bf16"
        self.heads, self.kv, self.dim, self.page, self.cache = heads, kv_heads, dim, page, cache
        self.window, self.softcap, self.ks, self.vs = window, softcap, k_scale, v_scale
        self.scale = dim ** -0.5 if scale is None else scale
        g = torch.Generator().manual_seed(seed)
        t = types(torch, dn)
        iot, ct = t[self.io][0], t[cache][0]
        B = len(self.lens)
        need = [-(-n // page) for n in self.lens]
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g).tolist()
        self.width = max(need + [0]) + wide
        table = torch.full((B, self.width), -7, dtype=torch.int32)
        bad = {"nan": float("nan"), "inf": float("inf"), "low": torch.finfo(torch.float32).min}[poison]
        if cache == "e4m3":
            bad = float("nan") if poison == "nan" else -448.0
        elif cache == "bf16" and poison == "low":
            bad = torch.finfo(torch.bfloat16).min
        k = torch.full((pages, page, kv_heads, dim), bad)
        v = torch.full((pages, page, kv_heads, dim), bad)
        if poison == "inf":
            v.neg_()
        self.rows, at = [], 0
        for b, n in enumerate(self.lens):
            kr = torch.randn(n, kv_heads, dim, generator=g).to(ct)
            vr = torch.randn(n, kv_heads, dim, generator=g).to(ct)
            for i in range(need[b]):
                table[b, i] = order[at + i]
                m = min(page, n - i * page)
                k[order[at + i], :m] = kr[i * page:i * page + m].float()
                v[order[at + i], :m] = vr[i * page:i * page + m].float()
            at += need[b]
            self.rows.append([kr.double() * k_scale, vr.double() * v_scale])
        self.q = torch.randn(B, heads, dim, generator=g).to(iot)
        self.new = None
        if append:
            self.new = [torch.randn(B, kv_heads, dim, generator=g).to(iot) for _ in range(2)]
            for b, n in enumerate(self.lens):
                if n == 0:
                    continue
                p, slot = table[b, (n - 1) // page].item(), (n - 1) % page
                for i, (cache_t, sc) in enumerate(((k, k_scale), (v, v_scale))):
                    cache_t[p, slot] = bad      # what was there before is not used
                    stored = (self.new[i][b].float() / sc)
                    stored = (stored.clamp(-448, 448) if cache == "e4m3" else stored).to(ct)
                    self.rows[b][i][n - 1] = stored.double() * sc
        if layout == "head":
            k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
        self.layout = layout
        self.k, self.v = k.to(ct).cuda(), v.to(ct).cuda()
        self.table = table.cuda()
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32).cuda()

    def desc(self, **kw):
        dn, t = self.dn, types(self.torch, self.dn)
        token, head = (1, 2) if self.layout == "token" else (2, 1)
        args = dict(io_type=t[self.io][1], cache_type=t[self.cache][1], page_stride=self.k.stride(0),
                    token_stride=self.k.stride(token), head_stride=self.k.stride(head), scale=self.scale,
                    softcap=self.softcap, window=self.window, k_scale=self.ks, v_scale=self.vs)
        args.update(kw)
        return dn.paged_attn_desc(len(self.lens), self.heads, self.kv, self.dim, self.page,
                                  self.k.shape[0], self.width, **args)

    def run(self, stream=None, lse=True, **kw):
        torch = self.torch
        q = self.q.cuda()
        out = torch.full_like(q, float("nan"))
        ls = torch.full(q.shape[:2], float("nan"), device="cuda") if lse else None
        new = [n.cuda() for n in self.new] if self.new else [None, None]
        s = stream or torch.cuda.current_stream()
        self.dn.check(self.dn.cuda_paged_attention(self.desc(**kw), q, self.k, self.v, self.table, self.lens_t,
                                                   out, lse=ls, k_new=new[0], v_new=new[1], stream=s))
        self.keep = (q, new)
        return out, ls

    def exact(self):
        """out, lse and their tolerances."""
        torch = self.torch
        B, G = len(self.lens), self.heads // self.kv
        out = torch.zeros(B, self.heads, self.dim, dtype=torch.float64)
        lse = torch.full((B, self.heads), -math.inf, dtype=torch.float64)
        tol, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
        r = r_of(torch, self.q.dtype)
        for b, n in enumerate(self.lens):
            first = max(0, n - self.window) if self.window else 0
            if n == 0:
                continue
            for h in range(self.heads):
                k, v = self.rows[b][0][first:, h // G], self.rows[b][1][first:, h // G]
                q = self.q[b, h].double()
                raw = k @ q * self.scale
                s = self.softcap * torch.tanh(raw / self.softcap) if self.softcap else raw
                d = float((sum_tol(self.dim) * (k.abs() @ q.abs()) * abs(self.scale) + 8 * U * raw.abs()).max())
                if self.softcap:
                    d += self.softcap * 2.0 ** -21      # tanh itself
                lse[b, h] = torch.logsumexp(s, 0)
                p = torch.exp(s - lse[b, h])
                out[b, h] = p @ v
                tol[b, h] = r * out[b, h].abs() + (2.2 * d + 2.0 ** -16 + sum_tol(n)) * (p @ v.abs())
                tol_lse[b, h] = d + 2.0 ** -20 + sum_tol(n) + 4 * U * lse[b, h].abs()
        return out, lse, tol, tol_lse

    def check(self, **kw):
        torch = self.torch
        before = [c.view(torch.uint8).clone() for c in (self.k, self.v)]
        out, lse = self.run(**kw)
        want, want_lse, tol, tol_lse = self.exact()
        within(out, want, tol, "out")
        if lse is not None:
            within(lse, want_lse, tol_lse, "lse")
        # The cache: the new rows as stored, every other byte as it was.
        t = types(torch, self.dn)[self.cache][0]
        for i, (old, now) in enumerate(zip(before, (self.k, self.v))):
            old = old.view(t).reshape(now.shape)
            if self.new:
                for b, n in enumerate(self.lens):
                    if n == 0:
                        continue
                    p, slot = self.table[b, (n - 1) // self.page].item(), (n - 1) % self.page
                    sc = (self.ks, self.vs)[i]
                    row = (self.rows[b][i][n - 1] / sc).to(torch.float32).to(t).cuda()
                    where = (p, slot) if self.layout == "token" else (p, slice(None), slot)
                    old.view(torch.uint8)[where] = row.view(torch.uint8).reshape(old.view(torch.uint8)[where].shape)
            assert torch.equal(old.view(torch.uint8), now.view(torch.uint8)), "cache"
        assert self.dn.stream_status(torch.cuda.current_stream()) == self.dn.SUCCESS
        return out, lse


LENS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 200, 0, 301]


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("page", [1, 12, 16, 64])
def test_attention_pages(gpu, dn, cache, layout, page, append):
    Paged(gpu, dn, LENS, 8, 2, 128, page, cache, layout, seed=page, append=append).check()


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 256])
def test_attention_dims(gpu, dn, cache, dim):
    Paged(gpu, dn, [1, 37, 130], 4, 2, dim, 16, cache, seed=dim, append=True).check()


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (7, 1), (8, 1), (9, 1), (16, 1), (17, 1), (40, 2),
                                      (64, 1), (12, 4), (32, 8), (128, 1)])
def test_attention_head_groups(gpu, dn, cache, heads, kv):
    Paged(gpu, dn, [70, 0, 129], heads, kv, 64, 16, cache, seed=heads, append=True).check()


@pytest.mark.parametrize("cache,poison", [("bf16", "inf"), ("bf16", "low"), ("f32", "inf"), ("f32", "low"),
                                          ("e4m3", "low")])
def test_attention_poisoned_slots(gpu, dn, cache, poison):
    for layout in ("token", "head"):
        Paged(gpu, dn, LENS, 4, 2, 64, 24, cache, layout, poison=poison, append=True).check()


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("window,softcap", [(1, 0.0), (16, 0.0), (50, 5.0), (1000, 0.0), (0, 2.0), (64, 30.0)])
def test_attention_window_and_softcap(gpu, dn, cache, window, softcap):
    p = Paged(gpu, dn, LENS, 8, 2, 64, 16, cache, window=window, softcap=softcap, seed=window)
    if window:
        # What lies before the window is not read: poison it.
        for b, n in enumerate(p.lens):
            for j in range(max(0, n - window)):
                page, slot = p.table[b, j // 16].item(), j % 16
                for c in (p.k, p.v):
                    c[page, slot] = gpu.full(c[page, slot].shape, float("nan"), device="cuda").to(c.dtype)
            for i in range(max(0, n - window) // 16):
                p.table[b, i] = -1
    p.check()


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3])
def test_attention_scales(gpu, dn, scale):
    Paged(gpu, dn, [100, 1], 4, 1, 64, 16, "bf16", scale=scale).check()
    Paged(gpu, dn, [100, 1], 4, 1, 64, 16, "e4m3", scale=scale, k_scale=0.37, v_scale=2.5, append=True).check()


def test_attention_large_scores(gpu, dn):
    """Scores in the thousands: one token takes it all, nothing overflows."""
    for cache in ("bf16", "e4m3", "f32"):
        p = Paged(gpu, dn, [333, 64], 8, 2, 64, 16, cache, scale=60.0)
        out, lse = p.run()
        want, want_lse, _, _ = p.exact()
        assert bool(out.isfinite().all()) and bool(lse.isfinite().all())
        assert float(((lse.double().cpu() - want_lse).abs() / want_lse.abs()).max()) < 1e-5


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("batch,longest", [(1, 5000), (1, 40000), (3, 20000), (40, 700)])
def test_attention_split_over_length(gpu, dn, cache, batch, longest):
    rng = np.random.default_rng(longest)
    lens = [longest] + [int(v) for v in rng.integers(0, longest // 4, batch - 1)]
    Paged(gpu, dn, lens, 4, 2, 64, 64, cache, append=True, layout="head").check()


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("batch", [1, 2, 31, 32, 33, 400])
@pytest.mark.parametrize("heads,kv", [(4, 4), (16, 1)])
def test_attention_among_empty_sequences(gpu, dn, cache, batch, heads, kv):
    """Sequences without a token first, last, in runs and everywhere; the others of one to many tiles."""
    rng = np.random.default_rng(batch)
    lens = rng.choice([1, 15, 64, 65, 200, 1000 if batch <= 33 else 129], batch)
    lens[rng.random(batch) < 0.6] = 0
    lens[:batch // 4] = 0
    lens[batch - batch // 8:] = 0
    Paged(gpu, dn, lens.tolist(), heads, kv, 64, 32, cache).check()
    Paged(gpu, dn, lens[::-1].tolist(), heads, kv, 64, 32, cache, window=70).check()
    Paged(gpu, dn, [0] * batch, heads, kv, 64, 32, cache).check()


def test_attention_same_bits_each_time(gpu, dn):
    for cache in ("bf16", "e4m3", "f32"):
        p = Paged(gpu, dn, [9000, 10, 0, 777], 8, 2, 128, 16, cache, append=True)
        out, lse = p.run()
        for _ in range(4):
            again, lse2 = p.run()
            assert gpu.equal(out, again) and gpu.equal(lse, lse2)


def test_attention_strides(gpu, dn):
    """q, out and new rows inside a fused projection's output; a table wider than it needs; K and V interleaved."""
    torch = gpu
    for cache in ("bf16", "f32"):
        p = Paged(torch, dn, [100, 33, 1], 8, 2, 64, 16, cache, append=True)
        want, want_lse, tol, tol_lse = p.exact()
        B, D = 3, 64
        fused = torch.full((B, 8 + 2 + 2 + 1, D), float("nan"), dtype=p.q.dtype, device="cuda")
        fused[:, :8], fused[:, 8:10], fused[:, 10:12] = p.q.cuda(), p.new[0].cuda(), p.new[1].cuda()
        both = torch.stack((p.k, p.v), 1).contiguous()       # [page][k, v][slot][head][dim]
        out = torch.full((8, B, D + 16), float("nan"), dtype=p.q.dtype, device="cuda")
        table = torch.full((B, p.width + 5), -3, dtype=torch.int32, device="cuda")
        table[:, :p.width] = p.table
        d = p.desc(q_strides=(13 * D, D), new_strides=(13 * D, D), out_strides=(D + 16, B * (D + 16)),
                   page_stride=both.stride(0), table_stride=p.width + 5)
        lse = torch.empty(B, 8, device="cuda")
        dn.check(dn.cuda_paged_attention(d, fused, both[:, 0], both[:, 1], table, p.lens_t, out, lse=lse,
                                         k_new=fused[:, 8:], v_new=fused[:, 10:],
                                         stream=torch.cuda.current_stream()))
        within(out[:, :, :D].transpose(0, 1), want, tol)
        within(lse, want_lse, tol_lse)
        assert bool(out[:, :, D:].isnan().all())


def test_attention_without_lse_on_another_stream(gpu, dn):
    torch = gpu
    p = Paged(torch, dn, [3000, 5, 0], 8, 2, 128, 16, "bf16")
    want, _ = p.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out, none = p.run(stream=side, lse=False)
    side.synchronize()
    assert none is None and torch.equal(out, want)


def test_attention_in_a_graph_with_growing_lengths(gpu, dn):
    """A captured call reads the lengths of each replay and takes one token in each time."""
    torch = gpu
    p = Paged(torch, dn, [90, 17], 8, 2, 64, 16, "bf16", append=True, wide=8, spare=16)
    p.run()
    full = Paged(torch, dn, [90, 17], 8, 2, 64, 16, "bf16", append=True, wide=8, spare=16)
    # Give both sequences the pages for more tokens.
    used = set(full.table.flatten().tolist())
    free = [i for i in range(full.k.shape[0]) if i not in used]
    full.table[0, 6], full.table[1, 2] = free[0], free[1]
    q, new = full.q.cuda(), [n.cuda() for n in full.new]
    out, lens = torch.empty_like(q), full.lens_t
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    d = full.desc()

    def call(stream):
        dn.check(dn.cuda_paged_attention(d, q, full.k, full.v, full.table, lens, out, k_new=new[0], v_new=new[1],
                                         stream=stream))
    call(side)
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call(side)
    for step in range(8):
        lens += 1
        for i in range(2):
            new[i].copy_(torch.randn(new[i].shape))
        g.replay()
        torch.cuda.synchronize()
        full.lens = lens.tolist()
        for b in range(2):
            for i in range(2):
                full.rows[b][i] = torch.cat((full.rows[b][i], new[i][b].double().cpu()[None]))
        want, _, tol, _ = full.exact()
        within(out, want, tol, f"step {step}")


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
def test_attention_bad_indexes_are_reported(gpu, dn, cache):
    """Lengths and page numbers out of range are not followed, and do not touch other sequences."""
    torch = gpu
    s = torch.cuda.current_stream()
    p = Paged(torch, dn, [40, 40, 40, 40], 4, 2, 64, 16, cache, append=True)
    want, want_lse, tol, _ = p.exact()
    cap = p.width * 16
    for lens in ([40, -1, 40, 40], [40, cap + 1, 40, 40], [40, 2 ** 31 - 1, 40, 40]):
        p.lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
        out, lse = p.run()
        assert dn.stream_status(s) == dn.INVALID_VALUE
        for b in (0, 2, 3):
            within(out[b], want[b], tol[b])
        assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())
    assert dn.stream_status(s) == dn.SUCCESS
    p.lens_t.fill_(40)
    for page in (-1, p.k.shape[0], 2 ** 31 - 1):
        table = p.table.clone()
        p.table[1, 1] = page
        out, lse = p.run()
        assert dn.stream_status(s) == dn.INVALID_VALUE
        # Sequence 1 is left with the tokens of its other pages.
        rows = [torch.cat((c[:16], c[32:])) for c in p.rows[1]]
        kept, p.rows[1], p.lens[1] = p.rows[1], rows, 24
        want1, _, tol1, _ = p.exact()
        p.rows[1], p.lens[1] = kept, 40
        within(out, want1, tol1)
        p.table.copy_(table)
    p.check()


def test_attention_offsets_past_32_bits(gpu, dn):
    """Pages that start beyond 2^31 elements."""
    torch = gpu
    stride = (1 << 31) + 64
    p = Paged(torch, dn, [40, 21], 4, 2, 64, 16, "bf16", spare=0)
    pages = p.k.shape[0]
    big = torch.empty(stride * (pages - 1) // 2 + 2 * p.k[0].numel(), dtype=torch.bfloat16, device="cuda")
    # K and V share the allocation: page i of K starts at i * stride2, V just after it.
    stride2 = big.numel() // (pages - 1) // 16 * 16 - 2 * p.k[0].numel()
    n = p.k[0].numel()
    for i in range(pages):
        big[i * stride2:i * stride2 + n] = p.k[i].reshape(-1)
        big[i * stride2 + n:i * stride2 + 2 * n] = p.v[i].reshape(-1)
    assert stride2 * (pages - 1) > 1 << 31
    out = torch.empty(2, 4, 64, dtype=torch.bfloat16, device="cuda")
    q = p.q.cuda()
    dn.check(dn.cuda_paged_attention(p.desc(page_stride=stride2), q, big, big[n:], p.table, p.lens_t, out,
                                     stream=torch.cuda.current_stream()))
    want, _, tol, _ = p.exact()
    within(out, want, tol)


def test_attention_nothing_to_do(gpu, dn):
    """No sequences; sequences without a token and a cache without a page."""
    torch = gpu
    s = torch.cuda.current_stream()
    d = dn.paged_attn_desc(0, 4, 2, 64, 16, 10, 4)
    assert dn.cuda_paged_attention(d, None, None, None, None, None, None, stream=s) == dn.SUCCESS
    q = torch.randn(3, 4, 64, device="cuda").bfloat16()
    out, lse = torch.full_like(q, 7.0), torch.full((3, 4), 7.0, device="cuda")
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    d = dn.paged_attn_desc(3, 4, 2, 64, 16, 0, 0)
    dn.check(dn.cuda_paged_attention(d, q, None, None, None, lens, out, lse=lse, stream=s))
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


# ------------------------------------------------------------- block norm
NORMS = {"none": 0, "rms": 1, "layer": 2}


def norm64(v, kind, w, b, off, eps):
    if kind == "none":
        return v
    mean = v.mean(1, keepdim=True) if kind == "layer" else 0.0
    v = (v - mean) / ((v - mean) ** 2).mean(1, keepdim=True).add(eps).sqrt()
    if w is not None:
        v = v * (w.double().cpu() + off)
    return v if b is None else v + b.double().cpu()


def norm_check(torch, dn, rows, cols, io="bf16", wt="bf16", post="rms", pre="rms", gate="none", weights=True,
               biases=False, off=0.0, rs=1.0, bs=1.0, eps=1e-5, pad=0, y=True, gate_rows=1, alias=None,
               shift=0.0, seed=0, h=True, z=True):
    t = types(torch, dn)
    g = torch.Generator().manual_seed(seed)
    T, W = t[io][0], t[wt][0]

    def mat(r=rows):
        return (torch.randn(r, cols + pad, generator=g) + shift).to(T).cuda()

    X, Y = mat(), mat() if y else None
    Gt = {"none": None, "channel": mat(1), "row": mat(-(-rows // gate_rows))}[gate]
    vec = lambda on, at: (torch.randn(cols, generator=g) * 0.2 + at).to(W).cuda() if on else None  # noqa: E731
    pw, pb, qw, qb = vec(weights, 1.0 - off), vec(biases, 0), vec(weights, 1.0 - off), vec(biases, 0)
    x64 = X.double().cpu()[:, :cols]
    want = rs * x64
    scale = want.abs()
    if y:
        block = norm64(Y.double().cpu()[:, :cols], post, pw, pb, off, eps)
        bmag = block.abs() + (pb.double().cpu().abs() if pb is not None and post != "none" else 0.0)
        if post == "layer":     # the mean's rounding, against the values it is taken from
            std = Y.double().cpu()[:, :cols].std(1, unbiased=False, keepdim=True).clamp(min=math.sqrt(eps))
            bmag = bmag + Y.double().cpu()[:, :cols].abs().mean(1, keepdim=True) / std * 2.0
        if Gt is not None:
            at = torch.arange(rows) // gate_rows if gate == "row" else torch.zeros(rows, dtype=torch.long)
            G64 = Gt.double().cpu()[at, :cols]
            block, bmag = block * G64, bmag * G64.abs()
        want, scale = want + bs * block, scale + abs(bs) * bmag
    want_z = norm64(want, pre, qw, qb, off, eps)
    H = torch.full((rows, cols + pad), float("nan"), dtype=T, device="cuda") if h else None
    Z = torch.full((rows, cols + pad), float("nan"), dtype=T, device="cuda") if z else None
    x_in, y_in = X.clone(), Y.clone() if y else None
    if alias:
        H = {"x": x_in, "y": y_in}.get(alias[0], H)
        Z = {"x": x_in, "y": y_in}.get(alias[1], Z)
    d = dn.block_norm_desc(rows, cols, post=NORMS[post], pre=NORMS[pre], io_type=t[io][1], weight_type=t[wt][1],
                           eps=eps, weight_offset=off, residual_scale=rs, block_scale=bs, ldx=cols + pad,
                           ldy=cols + pad, ldh=cols + pad, ldz=cols + pad, ldg=cols + pad if gate == "row" else 0,
                           gate_rows=gate_rows)
    dn.check(dn.cuda_block_norm(d, x_in, y_in, Gt, pw, pb, qw, qb, H, Z, torch.cuda.current_stream()))
    r = r_of(torch, T)
    err_h = (16 * U + sum_tol(cols)) * scale
    if h:
        within(H[:, :cols], want, r * want.abs() + err_h, "h")
    if z:
        # h's error over its deviation, then the row statistics' own.
        c = want - want.mean(1, keepdim=True) if pre == "layer" else want
        dev = (c ** 2).mean(1, keepdim=True).add(eps).sqrt() if pre != "none" else torch.ones(rows, 1).double()
        w = (qw.double().cpu() + off).abs() if qw is not None and pre != "none" else 1.0
        big = err_h + err_h.mean(1, keepdim=True) + (sum_tol(cols) * want.abs().mean(1, keepdim=True) if pre == "layer" else 0)
        tol = r * want_z.abs() + big / dev * w + (16 * U + sum_tol(cols)) * (c.abs() / dev * w + 1e-30)
        if qb is not None and pre != "none":
            tol = tol + 4 * U * qb.double().cpu().abs()
        within(Z[:, :cols], want_z, tol, "z")
    for m, src in ((H, X), (Z, X)):
        if m is not None and pad and m is not x_in and (not y or m is not y_in):
            assert bool(m[:, cols:].isnan().all())
    return H, Z


@pytest.mark.parametrize("io,wt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("pre", ["none", "rms", "layer"])
@pytest.mark.parametrize("gate", ["none", "channel", "row"])
def test_norm_forms(gpu, dn, io, wt, post, pre, gate):
    norm_check(gpu, dn, 5, 264, io, wt, post, pre, gate, biases=True, rs=0.7, bs=-1.3)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [1, 2, 7, 8, 31, 64, 100, 256, 257, 1000, 1024, 2039, 4093, 4096, 8192, 11008, 16384,
                                  28672, 49152])
def test_norm_widths(gpu, dn, cols, io):
    norm_check(gpu, dn, 3, cols, io, io, "rms", "layer", "channel", biases=True, seed=cols)


@pytest.mark.parametrize("rows", [1, 2, 147, 149, 1000, 5000])
@pytest.mark.parametrize("cols", [64, 200, 1009])
def test_norm_rows(gpu, dn, rows, cols):
    norm_check(gpu, dn, rows, cols, "bf16", "bf16", "layer", "rms", "row", seed=rows, gate_rows=3)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("cols,pad", [(256, 1), (256, 8), (1001, 7), (4096, 3), (4096, 16)])
def test_norm_pitches(gpu, dn, cols, pad, io):
    norm_check(gpu, dn, 7, cols, io, "f32", gate="row", pad=pad)


@pytest.mark.parametrize("io,wt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,cols,pad", [(700, 1100, 0), (700, 1099, 1), (700, 1099, 0), (700, 5001, 1), (700, 2999, 3),
                                           (3, 334, 0), (3, 333, 1), (2, 12002, 0), (700, 602, 0), (700, 601, 1),
                                           (700, 768, 0), (650, 1536, 0), (650, 3071, 1), (5, 20002, 0), (700, 6146, 0)])
def test_norm_pairs_and_sizes(gpu, dn, rows, cols, pad, io, wt):
    """Rows at multiples of one, two and eight elements, whose last pair may have one."""
    norm_check(gpu, dn, rows, cols, io, wt, post="layer", gate="row", pad=pad, biases=True)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("cols", [96, 4096, 20000])
@pytest.mark.parametrize("alias", ["x-", "y-", "-x", "-y", "xy", "yx"])
def test_norm_in_place(gpu, dn, cols, alias, io):
    norm_check(gpu, dn, 9, cols, io, "f32", "rms", "rms", "row", alias=alias)


def test_norm_optional_parts(gpu, dn):
    for io in ("bf16", "f32"):
        norm_check(gpu, dn, 6, 300, io, y=False)
        norm_check(gpu, dn, 6, 300, io, y=False, pre="layer", h=False)
        norm_check(gpu, dn, 6, 300, io, h=False)
        norm_check(gpu, dn, 6, 300, io, z=False)
        norm_check(gpu, dn, 6, 300, io, weights=False, biases=True)
        norm_check(gpu, dn, 6, 300, io, off=1.0, eps=0.0)


def test_norm_means_far_from_zero(gpu, dn):
    """A layer norm of values around 100 does not lose its variance."""
    norm_check(gpu, dn, 4, 4096, "f32", "f32", "layer", "layer", shift=100.0)


def test_norm_constant_and_zero_rows(gpu, dn):
    torch = gpu
    for kind, want in ((dn.NORM_RMS, 0.0), (dn.NORM_LAYER, 0.0)):
        x = torch.zeros(3, 512, device="cuda")
        z = torch.empty_like(x)
        dn.check(dn.cuda_block_norm(dn.block_norm_desc(3, 512, pre=kind, io_type=dn.TYPE_F32), x, None, None, None,
                                    None, None, None, None, z, torch.cuda.current_stream()))
        assert bool((z == want).all())
    x = torch.full((3, 512), 3.0, device="cuda")
    dn.check(dn.cuda_block_norm(dn.block_norm_desc(3, 512, pre=dn.NORM_LAYER, io_type=dn.TYPE_F32), x, None, None,
                                None, None, None, None, None, z, torch.cuda.current_stream()))
    assert bool((z == 0).all())


def test_norm_nan_stays_in_its_row(gpu, dn):
    torch = gpu
    for cols in (64, 4096, 20000):
        x = torch.randn(4, cols, device="cuda").bfloat16()
        z = torch.empty_like(x)
        d = dn.block_norm_desc(4, cols)
        dn.check(dn.cuda_block_norm(d, x, None, None, None, None, None, None, None, z, torch.cuda.current_stream()))
        clean = z.clone()
        x[1, 5], x[2, 6] = float("nan"), float("inf")
        dn.check(dn.cuda_block_norm(d, x, None, None, None, None, None, None, None, z, torch.cuda.current_stream()))
        assert torch.equal(z[0], clean[0]) and torch.equal(z[3], clean[3])
        assert bool(z[1].isnan().all())
        assert bool(z[2, 6].isnan()) and bool((z[2, :6] == 0).all())


def test_norm_offsets_past_32_bits(gpu, dn):
    torch = gpu
    rows, cols, pitch = 3, 200, (1 << 30) + 8
    big = torch.empty(2 * pitch + cols, dtype=torch.bfloat16, device="cuda")
    view = big.as_strided((rows, cols), (pitch, 1))
    view.copy_(torch.randn(rows, cols))
    z = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    d = dn.block_norm_desc(rows, cols, ldx=pitch, ldh=pitch)
    want = norm64(view.double().cpu(), "rms", None, None, 0.0, 1e-5)
    dn.check(dn.cuda_block_norm(d, view, None, None, None, None, None, None, view, z, torch.cuda.current_stream()))
    within(z, want, 2.0 ** -8 * want.abs() + sum_tol(cols) * want.abs())


# ------------------------------------------------------------- failure paths
def test_injected_launch_failure_leaves_outputs(gpu, dn):
    torch = gpu
    ins = w4_inputs(torch, 2, 64, 128, 32, torch.bfloat16, torch.bfloat16, False, False)
    C = torch.full((2, 64), 7.0, device="cuda").bfloat16()
    d = dn.w4_desc(2, 64, 128, 128, 64, 64, 32, 4)
    dn.lib.dnnopt_debug_inject_fault(2, 1)
    s = torch.cuda.current_stream()
    assert dn.cuda_gemm_w4(d, ins[0], ins[1], ins[2], None, None, C, s) == dn.INJECTED_FAULT
    torch.cuda.synchronize()
    assert bool((C == 7).all())
    assert dn.cuda_gemm_w4(d, ins[0], ins[1], ins[2], None, None, C, s) == dn.SUCCESS
