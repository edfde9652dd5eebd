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
@pytest.mark.parametrize("lens", [[5], [5, 0, 0], [0, 5, 0], [0] * 40 + [64, 1]])
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


def test_graphs_outlive_a_grown_workspace(gpu, dn):
    """A step captured for few rows replays after larger calls on its stream, whose workspace has grown,
    and after other memory was taken and written."""
    from test_decode_ops import Paged, w4_inputs
    torch = gpu
    side = torch.cuda.Stream()
    M, N, K = 2, 1009, 20000        # digits made before the product, tiles in several parts
    A, W, scale, _, _ = w4_inputs(torch, M, N, K, 128, torch.bfloat16, torch.bfloat16, False, False)
    C = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
    d = dn.w4_desc(M, N, K, K, W.stride(0), N, 128, scale.stride(0))
    p = Paged(torch, dn, [3000, 40], 8, 2, 64, 16, "bf16")
    q, out = p.q.cuda(), torch.empty_like(p.q, device="cuda")
    torch.cuda.synchronize()

    def step():
        dn.check(dn.cuda_gemm_w4(d, A, W, scale, None, None, C, side))
        dn.check(dn.cuda_paged_attention(p.desc(), q, p.k, p.v, p.table, p.lens_t, out, stream=side))

    step()
    side.synchronize()
    want = C.clone(), out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    kept = []
    for rows in (9, 40, 200):
        big = w4_inputs(torch, rows, 9000, K, 128, torch.bfloat16, torch.bfloat16, False, False)
        Cb = torch.empty(rows, 9000, device="cuda", dtype=torch.bfloat16)
        db = dn.w4_desc(rows, 9000, K, K, big[1].stride(0), 9000, 128, big[2].stride(0))
        pb = Paged(torch, dn, [70] * (4 * rows), 16, 4, 64, 16, "bf16")
        torch.cuda.synchronize()
        dn.check(dn.cuda_gemm_w4(db, big[0], big[1], big[2], None, None, Cb, side))
        with torch.cuda.stream(side):
            pb.run(stream=side)
        side.synchronize()
        torch.cuda.empty_cache()
        kept.append(torch.full((1 << 28,), 0xFF, device="cuda", dtype=torch.uint8))
        for t in (C, out):
            t.zero_()
        torch.cuda.synchronize()
        for _ in range(2):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(C, want[0]) and torch.equal(out, want[1]), rows
    assert dn.stream_status(side) == dn.SUCCESS


def test_bad_lengths_are_not_another_calls(gpu, dn):
    """A product of host operands on the same stream succeeds, and leaves the report where it is."""
    import numpy as np
    from test_decode_ops import Paged
    torch = gpu
    side = torch.cuda.Stream()
    p = Paged(torch, dn, [40, 40], 4, 2, 64, 16, "bf16")
    p.lens_t.copy_(torch.tensor([40, -1], dtype=torch.int32))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        p.run(stream=side)
    a, b, c = np.ones((4, 8), np.float32), np.ones((8, 16), np.float32), np.zeros((4, 16), np.float32)
    dn.set_stream(side)
    try:
        assert dn.gemm_f32_desc(dn.desc(4, 16, 8, 8, 16, 16), a, b, c) == dn.SUCCESS
    finally:
        dn.set_stream(None)
    assert (c == 8).all()
    assert dn.stream_status(side) == dn.INVALID_VALUE
    assert dn.stream_status(side) == dn.SUCCESS


@pytest.mark.parametrize("M,N,K,pitch,pad", [(511, 70, 300, 16, 0), (512, 70, 300, 16, 0), (513, 70, 300, 1, 5), (1100, 33, 129, 16, 1),
                                             (1538, 8192, 4096, 16, 0)])
def test_w4_many_rows(gpu, dn, M, N, K, pitch, pad):
    """Rows past those of one launch, the last launch of one, two or more of them."""
    from test_decode_ops import sum_tol, w4_exact, w4_inputs, w4_run, within
    torch = gpu
    ins = w4_inputs(torch, M, N, K, 128, torch.bfloat16, torch.bfloat16, True, True, pad, pitch=pitch)
    C = w4_run(torch, dn, M, N, K, 128, *ins, pad_c=pad)
    rows = sorted({*range(0, M, 37), *range(505, min(M, 520)), *range(M - 4, M)})
    want, mag = w4_exact(torch, ins[0][rows], *ins[1:], K, 128)
    within(C[rows][:, :N], want, 2.0 ** -8 * want.abs() + sum_tol(K) * mag)
    assert bool(C[:, N:].isnan().all()) and bool(C[:, :N].isfinite().all())


def test_w4_rows_without_end(gpu, dn):
    """More rows than a grid has blocks; a workspace that does not grow with them."""
    torch = gpu
    M, N, K = 530000, 32, 32
    A = torch.randint(-8, 9, (M, K), device="cuda").bfloat16()
    W = torch.randint(0, 256, (N, 16), device="cuda", dtype=torch.uint8)
    scale = torch.ones(N, 1, device="cuda").bfloat16()
    codes = torch.stack((W & 15, W >> 4), 2).view(N, K).float() - 8
    C = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    free = torch.cuda.mem_get_info()[0]
    dn.check(dn.cuda_gemm_w4(dn.w4_desc(M, N, K, K, 16, N, 0, 1), A, W, scale, None, None, C, side))
    side.synchronize()
    assert free - torch.cuda.mem_get_info()[0] < 1 << 28
    assert torch.equal(C, (A.float() @ codes.t()).bfloat16())      # whole numbers below 2^24


@pytest.mark.parametrize("cache", ["bf16", "e4m3", "f32"])
@pytest.mark.parametrize("lens", [[0, -1, 40], [0, -1, 0], [0, 0, 10 ** 6, 5], [-1], [40, 0, 0, -5], [0] * 31 + [-1],
                                  [0] * 32 + [-1], [0] * 200 + [-1] + [0] * 100, [7] * 31 + [1 << 30]])
def test_bad_lengths_after_empty_sequences(gpu, dn, cache, lens):
    """A length out of range is reported wherever it stands, and only its sequence counts as empty."""
    from test_decode_ops import Paged, within
    torch = gpu
    s = torch.cuda.current_stream()
    assert dn.stream_status(s) == dn.SUCCESS
    p = Paged(torch, dn, [n if 0 <= n < 1000 else 0 for n in lens], 4, 2, 64, 16, cache)
    want, want_lse, tol, tol_lse = p.exact()
    p.lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
    for window in (0, 16):
        out, lse = p.run(window=window)
        assert dn.stream_status(s) == dn.INVALID_VALUE
        assert dn.stream_status(s) == dn.SUCCESS
        if not window:
            within(out, want, tol)
            within(lse, want_lse, tol_lse)
