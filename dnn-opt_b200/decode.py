"""One decoder layer's step for one new token per sequence, on the C ABI.

What a caller of the small-M products runs to generate a token, end to end:

    q, k, v = W_qkv z                      4-bit weights      dnnopt_cuda_gemm_w4
    a       = attention(q; cache + k, v)   paged cache        dnnopt_cuda_paged_attention
    h, z    = norms(h, W_o a)              post, gate, pre    dnnopt_cuda_block_norm
    u       = W_up z ; g = W_gate z        4-bit weights      dnnopt_cuda_gemm_w4
    h, z    = norms(h, W_down (silu(g) u)) post, gate, pre    dnnopt_cuda_block_norm

Eight calls of the library and two elementwise torch operations a layer, all on
the caller's stream, nothing synchronised: a step can be captured in a CUDA
graph once the cache's pages are assigned.

``python decode.py`` runs a small random-weight stack and compares a step with
the same computation in 32-bit torch operations.
"""
from __future__ import annotations

import sys
from dataclasses import dataclass

import torch


def _package():
    """The package this file belongs to (its folder's name is no identifier)."""
    if "dnnopt_b200" in sys.modules:
        return sys.modules["dnnopt_b200"]
    import importlib.util
    import os
    here = os.path.dirname(os.path.abspath(__file__))
    spec = importlib.util.spec_from_file_location("dnnopt_b200", os.path.join(here, "__init__.py"),
                                                  submodule_search_locations=[here])
    module = importlib.util.module_from_spec(spec)
    sys.modules["dnnopt_b200"] = module
    spec.loader.exec_module(module)
    return module


# ---- 4-bit weights -----------------------------------------------------------
def quantize_w4(w: torch.Tensor, group: int, symmetric: bool = True):
    """(packed, scale, zero) of a weight [N, K]: codes 0..15, two per byte with the even k in the
    low four bits, rows padded to 16 bytes; scale and zero are bf16, zero is None when symmetric.
    group: a multiple of 32 (the last group of a row may be short)."""
    N, K = w.shape
    G = -(-K // group)
    padded = torch.zeros(N, G * group, device=w.device)
    padded[:, :K] = w.float()
    g = padded.view(N, G, group)
    if symmetric:
        scale = (g.abs().amax(2) / 7.0).clamp(min=1e-8).bfloat16()
        zero = None
        codes = (g / scale.float()[..., None]).round().clamp(-8, 7) + 8
    else:
        lo, hi = g.amin(2).clamp(max=0.0), g.amax(2).clamp(min=0.0)
        scale = ((hi - lo) / 15.0).clamp(min=1e-8).bfloat16()
        zero = (-lo / scale.float()).round().clamp(0, 15).bfloat16()
        codes = ((g / scale.float()[..., None]).round() + zero.float()[..., None]).clamp(0, 15)
    codes = codes.view(N, -1)[:, :K].to(torch.uint8)
    pitch = (-(-K // 2) + 15) // 16 * 16
    bytes_ = torch.zeros(N, pitch, 2, device=w.device, dtype=torch.uint8)
    bytes_.view(N, -1)[:, :K] = codes
    return (bytes_[..., 0] | (bytes_[..., 1] << 4)).contiguous(), scale, zero


def dequantize_w4(packed: torch.Tensor, scale: torch.Tensor, zero, K: int, group: int) -> torch.Tensor:
    """The FP32 weight [N, K] that a packed one stands for."""
    codes = torch.stack((packed & 15, packed >> 4), 2).view(packed.shape[0], -1)[:, :K].float()
    at = torch.arange(K, device=packed.device) // group
    return (codes - (8.0 if zero is None else zero.float()[:, at])) * scale.float()[:, at]


class W4Linear:
    """y = x W^T with a 4-bit weight; x and y bf16, any number of rows (few are fast).  x has its
    rows' elements side by side, rows any pitch apart."""

    def __init__(self, w: torch.Tensor, group: int = 128, symmetric: bool = True):
        self.N, self.K = w.shape
        self.group = group
        self.packed, self.scale, self.zero = quantize_w4(w, group, symmetric)

    def __call__(self, x: torch.Tensor, stream=None) -> torch.Tensor:
        dn = _package()
        if x.dtype != torch.bfloat16 or x.dim() != 2 or x.shape[1] != self.K:
            raise ValueError(f"rows of {self.K} bf16 elements are wanted: got {x.dtype} {tuple(x.shape)}")
        if x.shape[1] > 1 and x.stride(1) != 1 or x.shape[0] > 1 and x.stride(0) < self.K:
            raise ValueError(f"rows' elements have to lie side by side: got strides {x.stride()}")
        y = torch.empty(x.shape[0], self.N, device=x.device, dtype=x.dtype)
        d = dn.w4_desc(x.shape[0], self.N, self.K, max(x.stride(0), self.K), self.packed.stride(0), self.N, self.group,
                       self.scale.stride(0))
        dn.check(dn.cuda_gemm_w4(d, x, self.packed, self.scale, self.zero, None, y,
                                 stream or torch.cuda.current_stream()), "cuda_gemm_w4")
        return y

    def plain(self, x: torch.Tensor) -> torch.Tensor:
        """The same in 32-bit torch operations, rounded once."""
        return (x.float() @ dequantize_w4(self.packed, self.scale, self.zero, self.K, self.group).t()).to(x.dtype)


# ---- paged cache --------------------------------------------------------------
class PagedCache:
    """Key and value pages of the layers, bf16 or E4M3, and the pages that sequences share out.

    Pages are assigned on the host (`grow`), one page table for all layers; the
    step reads lengths and table on the device."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, pages: int, page_size: int, max_pages: int,
                 layers: int = 1, dtype=torch.bfloat16, device="cuda"):
        if dtype not in (torch.bfloat16, torch.float8_e4m3fn):
            raise ValueError(f"the cache of a bf16 layer holds bfloat16 or float8_e4m3fn, not {dtype}")
        self.page_size, self.max_pages = page_size, max_pages
        shape = (pages, page_size, kv_heads, head_dim)
        self.k = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(layers)]
        self.v = [torch.zeros(shape, device=device, dtype=dtype) for _ in range(layers)]
        self.table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.free = list(range(pages - 1, -1, -1))
        self.held = [[] for _ in range(batch)]

    def grow(self, tokens: int = 1, slots=None) -> None:
        """Makes every sequence, or those of `slots` alone, `tokens` longer, assigning the pages that
        this takes.  Where they are not there nothing changes.  A slot that is left out keeps its
        length: an ended one (`release`) stays empty, and the step answers zeros for its attention."""
        lens = self.lens.tolist()
        grown = range(len(lens)) if slots is None else sorted(set(slots))
        if any(not 0 <= b < len(lens) for b in grown):
            raise IndexError(f"slots are 0 to {len(lens) - 1}: got {list(grown)}")
        want = {b: max(0, -(-(lens[b] + tokens) // self.page_size) - len(self.held[b])) for b in grown}
        if sum(want.values()) > len(self.free) or any(len(self.held[b]) + n > self.max_pages for b, n in want.items()):
            raise RuntimeError("the cache has no page left for a longer sequence")
        for b, n in want.items():
            for _ in range(n):
                page = self.free.pop()
                self.table[b, len(self.held[b])] = page
                self.held[b].append(page)
        if slots is None:
            self.lens += tokens
        elif want:
            self.lens[list(want)] += tokens

    def release(self, b: int) -> None:
        """Ends sequence b: its pages are free again."""
        self.free += self.held[b][::-1]
        self.held[b] = []
        self.table[b] = -1
        self.lens[b] = 0


# ---- the layer ------------------------------------------------------------------
@dataclass
class LayerConfig:
    hidden: int
    heads: int
    kv_heads: int
    head_dim: int
    ffn: int
    group: int = 128
    eps: float = 1e-5


class DecoderLayer:
    """Attention and a gated FFN, each with a norm before and after it and a learnt gate per channel."""

    def __init__(self, c: LayerConfig, seed: int = 0, device="cuda"):
        g = torch.Generator(device=device)
        g.manual_seed(seed)

        def weight(n, k, symmetric=True):
            return W4Linear(torch.randn(n, k, device=device, generator=g) * k ** -0.5, c.group, symmetric)

        def vector(at):
            return (torch.rand(c.hidden, device=device, generator=g) * 0.2 + at).bfloat16()

        self.c = c
        self.qkv = weight((c.heads + 2 * c.kv_heads) * c.head_dim, c.hidden)
        self.o = weight(c.hidden, c.heads * c.head_dim)
        self.up, self.gate = weight(c.ffn, c.hidden, False), weight(c.ffn, c.hidden, False)
        self.down = weight(c.hidden, c.ffn)
        self.post = [vector(0.9), vector(0.9)]          # after attention, after the FFN
        self.pre = [vector(0.9), vector(0.9)]           # before the FFN, before the next layer
        self.scale = [vector(0.5), vector(0.5)]         # gates of the two residual additions

    def _norms(self, which, h, y):
        """h + gate * rms(y), in place of h; and the next block's rms of it."""
        dn, c = _package(), self.c
        z = torch.empty_like(h)
        d = dn.block_norm_desc(h.shape[0], c.hidden, post=dn.NORM_RMS, pre=dn.NORM_RMS, eps=c.eps)
        dn.check(dn.cuda_block_norm(d, h, y, self.scale[which], self.post[which], None, self.pre[which], None, h, z,
                                    torch.cuda.current_stream()), "cuda_block_norm")
        return z

    def step(self, h, z, cache: PagedCache, layer: int):
        """h: residual stream [B, hidden], updated in place; z: its norm, this layer's input.
        Returns the next layer's input.  cache.lens counts the new token."""
        dn, c = _package(), self.c
        B, D = cache.lens.shape[0], c.head_dim
        for name, t in (("h", h), ("z", z)):
            if t.dtype != torch.bfloat16 or tuple(t.shape) != (B, c.hidden) or not t.is_contiguous():
                raise ValueError(f"{name} has to be contiguous bf16 [{B}, {c.hidden}]: got {t.dtype} {tuple(t.shape)}")
        if cache.k[layer].shape[2:] != (c.kv_heads, D):
            raise ValueError(f"the cache has rows of {tuple(cache.k[layer].shape[2:])}, the layer {(c.kv_heads, D)}")
        qkv = self.qkv(z)
        row = qkv.stride(0)
        q, k, v = qkv, qkv[:, c.heads * D:], qkv[:, (c.heads + c.kv_heads) * D:]
        a = torch.empty(B, c.heads * D, device=h.device, dtype=h.dtype)
        keys, values = cache.k[layer], cache.v[layer]
        kind = dn.TYPE_BF16 if keys.dtype == torch.bfloat16 else dn.TYPE_E4M3
        d = dn.paged_attn_desc(B, c.heads, c.kv_heads, D, cache.page_size, keys.shape[0], cache.max_pages,
                               cache_type=kind, q_strides=(row, D), new_strides=(row, D))
        dn.check(dn.cuda_paged_attention(d, q, keys, values, cache.table, cache.lens, a, k_new=k, v_new=v,
                                         stream=torch.cuda.current_stream()), "cuda_paged_attention")
        z = self._norms(0, h, self.o(a))
        y = self.down(torch.nn.functional.silu(self.gate(z)) * self.up(z))
        return self._norms(1, h, y)

    def plain_step(self, h, z, keys, values):
        """The same step in 32-bit torch operations on dense keys and values [B, L, kv_heads, dim],
        which end with room for the new token; returns (h, z)."""
        c, B = self.c, h.shape[0]

        def rms(x, w):
            return x * torch.rsqrt((x * x).mean(1, keepdim=True) + c.eps) * w.float()

        def norms(which, h, y):
            h = h.float() + self.scale[which].float() * rms(y.float(), self.post[which])
            return h.to(torch.bfloat16), rms(h, self.pre[which]).to(torch.bfloat16)

        q, k, v = self.qkv.plain(z).split([c.heads * c.head_dim, c.kv_heads * c.head_dim, c.kv_heads * c.head_dim], 1)
        keys[:, -1], values[:, -1] = k.view(B, c.kv_heads, -1), v.view(B, c.kv_heads, -1)
        qh = q.float().view(B, c.kv_heads, c.heads // c.kv_heads, c.head_dim)
        p = torch.softmax(qh @ keys.float().permute(0, 2, 3, 1) * c.head_dim ** -0.5, 3)
        a = (p @ values.float().permute(0, 2, 1, 3)).reshape(B, -1).to(h.dtype)
        h, z = norms(0, h, self.o.plain(a))
        y = torch.nn.functional.silu(self.gate.plain(z)) * self.up.plain(z)
        return norms(1, h, self.down.plain(y))


def main() -> None:
    """Generates a few tokens' worth of steps on two layers and prints how far the plain form is."""
    c = LayerConfig(hidden=1024, heads=16, kv_heads=4, head_dim=64, ffn=2048)
    B, layers = 4, 2
    stack = [DecoderLayer(c, seed=i) for i in range(layers)]
    cache = PagedCache(B, c.kv_heads, c.head_dim, pages=32, page_size=16, max_pages=8, layers=layers)
    dense = [[torch.zeros(B, 0, c.kv_heads, c.head_dim, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
             for _ in range(layers)]
    torch.manual_seed(0)
    for step in range(20):
        x = torch.randn(B, c.hidden, device="cuda").bfloat16()
        cache.grow()
        h, z, hp, zp = x.clone(), x.clone(), x.clone(), x.clone()
        for i, layer in enumerate(stack):
            z = layer.step(h, z, cache, i)
            room = torch.zeros(B, 1, c.kv_heads, c.head_dim, device="cuda", dtype=torch.bfloat16)
            dense[i] = [torch.cat((t, room), 1) for t in dense[i]]
            hp, zp = layer.plain_step(hp, zp, *dense[i])
        off = float((z.float() - zp.float()).norm() / zp.float().norm())
        print(f"token {step + 1}: off the plain form by {off:.4f}")


if __name__ == "__main__":
    main()
