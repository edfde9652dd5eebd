"""Refusals of the decoder-step operators: argument checks that need no GPU.

Every call here must be answered before the device is touched: the pointers
are host addresses that are never followed."""
from __future__ import annotations

import ctypes

import pytest

P = 1 << 20     # an address that is 16-byte aligned and never read


def w4(dn, change=None, A=P, W=P, scale=P, zero=None, bias=None, C=P):
    d = dn.w4_desc(2, 64, 128, 128, 64, 64, 32, 4)
    for k, v in (change or {}).items():
        setattr(d, k, v)
    return dn.cuda_gemm_w4(d, A, W, scale, zero, bias, C)


@pytest.mark.parametrize("change", [
    {"M": -1}, {"N": -1}, {"K": -1}, {"lda": 127}, {"ldw": 63}, {"ldc": 63}, {"lds": 3}, {"group": 16},
    {"group": 33}, {"group": -32}, {"io_type": 2}, {"io_type": 7}, {"scale_type": 2}, {"K": 129, "lda": 129}])
def test_w4_refuses(dn, change):
    assert w4(dn, change) == dn.INVALID_VALUE


def test_w4_refuses_pointers(dn):
    for name in ("A", "W", "scale", "C"):
        assert w4(dn, **{name: None}) == dn.INVALID_VALUE, name
    for name in ("A", "scale", "zero", "C", "bias"):
        assert w4(dn, **{name: P + 1}) == dn.INVALID_VALUE, name
    assert dn.lib.dnnopt_cuda_gemm_w4(None, P, P, P, None, None, P, None) == dn.INVALID_VALUE


def test_w4_nothing_to_do(dn):
    for name in ("M", "N", "K"):
        assert w4(dn, {name: 0}, A=None, W=None, scale=None, C=None) == dn.SUCCESS
    assert w4(dn, {"K": 2 ** 31 - 1, "lda": 2 ** 31 - 1, "ldw": 2 ** 30, "group": 0}) == dn.NOT_SUPPORTED


def attn(dn, change=None, q=P, k=P, v=P, table=P, lens=P, k_new=None, v_new=None, out=P, lse=None):
    d = dn.paged_attn_desc(2, 8, 2, 64, 16, 10, 4)
    for key, value in (change or {}).items():
        setattr(d, key, value)
    return dn.cuda_paged_attention(d, q, k, v, table, lens, out, lse=lse, k_new=k_new, v_new=v_new)


@pytest.mark.parametrize("change", [
    {"batch": -1}, {"heads": 0}, {"kv_heads": 0}, {"heads": 9}, {"head_dim": 0}, {"page_size": 0},
    {"num_pages": -1}, {"max_pages": -1}, {"window": -1}, {"io_type": 2}, {"cache_type": 3}, {"cache_type": -1},
    {"scale": float("nan")}, {"scale": float("inf")}, {"softcap": -1.0}, {"softcap": float("nan")},
    {"k_scale": 0.0, "cache_type": 2}, {"v_scale": -1.0, "cache_type": 2}, {"k_scale": 2.0}, {"v_scale": 0.5},
    {"table_stride": 3}, {"table_stride": -1}, {"max_pages": 2 ** 28, "table_stride": 2 ** 28, "page_size": 2 ** 10}])
def test_attention_refuses(dn, change):
    assert attn(dn, change) == dn.INVALID_VALUE


@pytest.mark.parametrize("change", [
    {"head_dim": 72}, {"head_dim": 272}, {"io_type": 0}, {"cache_type": 0}, {"io_type": 0, "cache_type": 2},
    {"token_stride": 129}, {"head_stride": 68}, {"page_stride": 2049}, {"q_head_stride": 65}, {"q_batch_stride": 513},
    {"out_head_stride": 65}, {"out_batch_stride": 513}])
def test_attention_has_no_path(dn, change):
    assert attn(dn, change) == dn.NOT_SUPPORTED


def test_attention_refuses_pointers(dn):
    for name in ("q", "k", "v", "table", "lens", "out"):
        assert attn(dn, **{name: None}) == dn.INVALID_VALUE, name
    assert attn(dn, k_new=P) == dn.INVALID_VALUE
    assert attn(dn, v_new=P) == dn.INVALID_VALUE
    for name in ("q", "k", "v", "out"):
        assert attn(dn, **{name: P + 8}) == dn.NOT_SUPPORTED, name
    for name in ("table", "lens", "lse"):
        assert attn(dn, **{name: P + 2}) == dn.INVALID_VALUE, name
    assert attn(dn, k_new=P + 8, v_new=P) == dn.NOT_SUPPORTED
    assert attn(dn, {"new_head_stride": 63}, k_new=P, v_new=P) == dn.NOT_SUPPORTED
    assert dn.lib.dnnopt_cuda_paged_attention(*([None] * 11)) == dn.INVALID_VALUE
    assert attn(dn, {"batch": 0}, q=None, k=None, v=None, table=None, lens=None, out=None) == dn.SUCCESS


def norm(dn, change=None, x=P, y=P, gate=None, post_w=None, post_b=None, pre_w=None, pre_b=None, h=2 * P, z=3 * P):
    d = dn.block_norm_desc(4, 256, post=dn.NORM_RMS)
    for key, value in (change or {}).items():
        setattr(d, key, value)
    return dn.cuda_block_norm(d, x, y, gate, post_w, post_b, pre_w, pre_b, h, z)


@pytest.mark.parametrize("change", [
    {"rows": -1}, {"cols": -1}, {"post": 3}, {"pre": -1}, {"io_type": 2}, {"weight_type": 2}, {"eps": -1.0},
    {"eps": float("nan")}, {"gate_rows": 0}, {"ldx": 255}, {"ldy": 255}, {"ldh": 255}, {"ldz": 0}])
def test_norm_refuses(dn, change):
    assert norm(dn, change) == dn.INVALID_VALUE


def test_norm_refuses_pointers(dn):
    assert norm(dn, x=None) == dn.INVALID_VALUE
    assert norm(dn, h=None, z=None) == dn.INVALID_VALUE
    assert norm(dn, h=P * 4, z=P * 4) == dn.INVALID_VALUE
    for name in ("x", "y", "gate", "post_w", "post_b", "pre_w", "pre_b", "h", "z"):
        assert norm(dn, **{name: P + 1}) == dn.INVALID_VALUE, name
    assert norm(dn, {"ldg": 255}, gate=P) == dn.INVALID_VALUE
    # A row written over another row's input.
    assert norm(dn, {"ldh": 512}, h=P) == dn.INVALID_VALUE
    assert norm(dn, {"ldz": 512}, z=P) == dn.INVALID_VALUE
    assert norm(dn, {"cols": 49153, "ldx": 49153, "ldy": 49153, "ldh": 49153, "ldz": 49153}) == dn.NOT_SUPPORTED
    assert dn.lib.dnnopt_cuda_block_norm(*([None] * 11)) == dn.INVALID_VALUE
    for name in ("rows", "cols"):
        assert norm(dn, {name: 0}, x=None, y=None, h=None, z=None) == dn.SUCCESS


def test_descriptors_match_the_header(dn):
    """The ctypes mirrors have the C structs' sizes (compiled from the public header)."""
    import os
    import subprocess
    import tempfile
    names = {"dnnopt_w4_desc": dn.W4Desc, "dnnopt_paged_attn_desc": dn.PagedAttnDesc,
             "dnnopt_block_norm_desc": dn.BlockNormDesc}
    lines = []
    for c, mirror in names.items():
        lines.append(f'printf("%zu\\n", sizeof({c}));')
        lines += [f'printf("%zu\\n", offsetof({c}, {f[0]}));' for f in mirror._fields_]
    with tempfile.TemporaryDirectory() as tmp:
        src, exe = os.path.join(tmp, "t.c"), os.path.join(tmp, "t")
        with open(src, "w") as f:
            f.write('#include <stdio.h>\n#include "dnnopt_b200.h"\nint main(void) {' + "".join(lines) + "return 0;}\n")
        subprocess.run(["gcc", "-I", os.path.dirname(dn.HEADER_PATH), src, "-o", exe], check=True)
        got = [int(v) for v in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for mirror in names.values():
        want.append(ctypes.sizeof(mirror))
        want += [getattr(mirror, f[0]).offset for f in mirror._fields_]
    assert got == want
