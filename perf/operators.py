"""Cases, plain forms and exact values of the decoder-step operators.

Three operators are measured: products of few rows with 4-bit weights
(`gemm_w4`), attention of one new token over a paged key-value cache
(`paged_attention`) and the norms around a block with its gate and residual
scale (`block_norm`).  A case is a dict of plain values; `prepare` makes what a
user's program holds before the call, `run` makes one call (or, where `own` is
false, computes the same thing from elementary torch operations in 32 bits) and
`exact` computes it from the definition in 64 bits.
"""
from __future__ import annotations

import importlib.util
import math
import os
import random
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "e4m3": 1}


def _package():
    """The framework's Python package (its folder's name is no identifier)."""
    if "dnnopt_b200" not in sys.modules:
        where = os.path.join(ROOT, "dnn-opt_b200")
        spec = importlib.util.spec_from_file_location(
            "dnnopt_b200", os.path.join(where, "__init__.py"), submodule_search_locations=[where])
        module = importlib.util.module_from_spec(spec)
        sys.modules["dnnopt_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["dnnopt_b200"]


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _w4(name, M, N, K, group, io="bf16", scale="bf16", zeros=False, bias=False, pitch=16):
    """group 0: one scale a row.  pitch: packed rows start at multiples of so many bytes."""
    return {"name": name, "op": "gemm_w4", "M": M, "N": N, "K": K, "group": group, "io": io,
            "scale": scale, "zeros": zeros, "bias": bias, "pitch": pitch}


def _attn(name, batch, heads, kv_heads, dim, page, max_len, lens, io="bf16", cache="bf16",
          layout="token", append=False, window=0, softcap=0.0):
    """lens: "full" (every sequence max_len long) or "ragged" (1 .. max_len, some slots empty).
    layout: a page holds [page, kv_heads, dim] ("token") or [kv_heads, page, dim] ("head")."""
    return {"name": name, "op": "paged_attention", "batch": batch, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "max_len": max_len, "lens": lens,
            "io": io, "cache": cache, "layout": layout, "append": append, "window": window,
            "softcap": softcap}


def _norm(name, rows, cols, io="bf16", weight="bf16", post="rms", pre="rms", gate="none",
          bias=False, offset=0.0, residual=1.0, block=1.0, pad=0):
    """gate: "none", "channel" (one row for all) or "row" (one for each row)."""
    return {"name": name, "op": "block_norm", "rows": rows, "cols": cols, "io": io,
            "weight": weight, "post": post, "pre": pre, "gate": gate, "bias": bias,
            "offset": offset, "residual": residual, "block": block, "pad": pad}


def listed():
    return [
        # Smallest product: the irregular-N sweep's two-row, prime-N shape in 32 bits; latency counts.
        _w4("w4 2x1009x1024 f32 g32", 2, 1009, 1024, 32, io="f32", scale="f32"),
        # One token through a square projection (the single-row GEMV shape), symmetric codes.
        _w4("w4 1x4096x4096 g128", 1, 4096, 4096, 128),
        # Four tokens through an up-projection with zero points and a bias (the int8 GEMV's shape).
        _w4("w4 4x11008x4096 g64 zeros", 4, 11008, 4096, 64, zeros=True, bias=True),
        # Eight tokens through the decode FFN's wide projection: the largest weights.
        _w4("w4 8x28672x8192 g128", 8, 28672, 8192, 128),
        # Odd sizes in 32 bits: a ragged last group and an odd K, prime N.
        _w4("w4 5x4093x4099 f32 g96 zeros", 5, 4093, 4099, 96, io="f32", scale="f32", zeros=True),
        # Smallest attention: one sequence that has just begun; latency counts.
        _attn("attn b1 17 tokens", 1, 32, 8, 128, 16, 17, "full", append=True),
        # One long sequence: all of the GPU shares each head's cache.
        _attn("attn b1 131072 tokens", 1, 32, 8, 128, 64, 131072, "full"),
        # A served batch of uneven lengths, empty slots among them, taking its new tokens in.
        _attn("attn b64 ragged 8192", 64, 64, 8, 128, 16, 8192, "ragged", append=True),
        # An 8-bit cache, pages by head, a window over the last 4096 tokens and capped scores.
        _attn("attn b16 e4m3 window", 16, 16, 4, 256, 32, 10000, "ragged", cache="e4m3",
              layout="head", append=True, window=4096, softcap=30.0),
        # 32-bit cache with a key-value head for each head, small odd pages.
        _attn("attn b8 f32 mha", 8, 16, 16, 64, 12, 2039, "ragged", io="f32", cache="f32"),
        # One token between two blocks: latency counts.
        _norm("norm 1x4096", 1, 4096),
        # A long prompt's rows, gated, with layer norms, odd width, 32 bits.
        _norm("norm 16384x4093 f32 layer", 16384, 4093, io="f32", weight="f32", post="layer",
              pre="layer", gate="row", bias=True, residual=0.5, block=1.5),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["gemm_w4", "paged_attention", "block_norm"])
    if op == "gemm_w4":
        io = rng.choice(["bf16", "bf16", "f32"])
        c = _w4("", _log(rng, 1, 16), _log(rng, 33, 28672), _log(rng, 64, 8192),
                rng.choice([32, 64, 128, 128, 96, 256, 0]), io=io,
                scale="f32" if io == "f32" else rng.choice(["bf16", "f32"]),
                zeros=rng.random() < 0.5, bias=rng.random() < 0.5,
                pitch=rng.choice([16, 16, 16, 1]))
    elif op == "paged_attention":
        cache = rng.choice(["bf16", "bf16", "e4m3", "f32"])
        kv = rng.choice([1, 2, 3, 4, 8, 16])
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        group = rng.choice([1, 2, 4, 5, 7, 8, 16])
        page = rng.choice([1, 8, 12, 16, 32, 64, 128])
        longest = _log(rng, 1, 131072)
        # Batch and length together stay within the ragged batch's bytes.
        most = 64 * 8192 * 8 * 128 // (kv * dim * SIZE[cache])
        longest = min(longest, most)
        c = _attn("", max(1, min(_log(rng, 1, 128), most // longest)), kv * group, kv, dim, page, longest,
                  rng.choice(["full", "ragged"]), io="f32" if cache == "f32" else "bf16",
                  cache=cache, layout=rng.choice(["token", "head"]), append=rng.random() < 0.5,
                  window=rng.choice([0, 0, 0, 1000]), softcap=rng.choice([0.0, 0.0, 30.0]))
    else:
        rows, cols = _log(rng, 1, 16384), _log(rng, 64, 11008)
        rows = max(1, min(rows, 16384 * 4093 // cols))
        if rng.random() < 0.6:
            cols = max(64, cols // 64 * 64)
        io = rng.choice(["bf16", "f32"])
        c = _norm("", rows, cols, io=io, weight=rng.choice([io, "f32"]),
                  post=rng.choice(["rms", "layer", "none"]), pre=rng.choice(["rms", "layer"]),
                  gate=rng.choice(["none", "channel", "row"]), bias=rng.random() < 0.5,
                  offset=rng.choice([0.0, 1.0]), residual=rng.choice([1.0, 0.5]),
                  block=rng.choice([1.0, 0.25]), pad=rng.choice([0, 0, 8, 3]))
    del c["name"]
    return c


def _lengths(c):
    """The batch's lengths, the same for every seed up to their order."""
    if c["lens"] == "full":
        return [c["max_len"]] * c["batch"]
    rng = random.Random("%d %d %d" % (c["batch"], c["max_len"], c["kv_heads"]))
    got = [rng.randint(1, c["max_len"]) for _ in range(c["batch"])]
    got[0] = c["max_len"]
    for i in range(7, c["batch"], 16):
        got[i] = 0
    return got


def _groups(c):
    return -(-c["K"] // c["group"]) if c["group"] else 1


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, dtype="f32", std=1.0):
        return (torch.randn(*shape, device=DEV, generator=g) * std).to(TYPES[dtype])

    def uniform(*shape, lo=0.0, hi=1.0, dtype="f32"):
        return (torch.rand(*shape, device=DEV, generator=g) * (hi - lo) + lo).to(TYPES[dtype])

    s = {"case": dict(case)}
    if case["op"] == "gemm_w4":
        M, N, K, G = case["M"], case["N"], case["K"], _groups(case)
        pitch = -(-((K + 1) // 2) // case["pitch"]) * case["pitch"]
        s["A"] = normal(M, K, dtype=case["io"])
        s["W"] = torch.randint(0, 256, (N, pitch), device=DEV, dtype=torch.uint8, generator=g)
        s["scale"] = uniform(N, G, lo=0.002, hi=0.02, dtype=case["scale"])
        # Zero points of asymmetric codes: whole numbers near the middle.
        s["zero"] = (torch.randint(5, 11, (N, G), device=DEV, generator=g).to(TYPES[case["scale"]])
                     if case["zeros"] else None)
        s["bias"] = normal(N) if case["bias"] else None
        return s
    if case["op"] == "paged_attention":
        B, H, KV, D, page = (case[k] for k in ("batch", "heads", "kv_heads", "dim", "page"))
        lens = _lengths(case)
        random.Random(seed).shuffle(lens)
        need = [-(-n // page) for n in lens]
        width = max(1, max(need))
        pages = sum(need) + 8       # some pages are free
        order = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)
        lens_t = torch.tensor(lens, device=DEV, dtype=torch.int32)
        need_t = torch.tensor(need, device=DEV)
        column = torch.arange(width, device=DEV)[None, :]
        first = (need_t.cumsum(0) - need_t)[:, None]
        table = torch.where(column < need_t[:, None],
                            order[(first + column).clamp(max=pages - 1)], -1)
        shape = (pages, page, KV, D) if case["layout"] == "token" else (pages, KV, page, D)
        s["k"] = normal(*shape, dtype=case["cache"])
        s["v"] = normal(*shape, dtype=case["cache"])
        s["q"] = normal(B, H, D, dtype=case["io"])
        s["table"], s["lens"] = table.to(torch.int32).contiguous(), lens_t
        if case["append"]:
            s["k_new"], s["v_new"] = normal(B, KV, D, dtype=case["io"]), normal(B, KV, D, dtype=case["io"])
        return s
    R, C, pad = case["rows"], case["cols"], case["pad"]
    # The residual stream carries a few large channels; the block's output is smaller.
    loud = 1.0 + 20.0 * (torch.rand(C + pad, device=DEV, generator=g) < 0.01)
    s["x"] = (normal(R, C + pad) * loud).to(TYPES[case["io"]])[:, :C]
    s["y"] = normal(R, C + pad, dtype=case["io"], std=0.5)[:, :C]
    s["gate"] = {"none": lambda: None, "channel": lambda: uniform(1, C, dtype=case["io"]),
                 "row": lambda: uniform(R, C, dtype=case["io"])}[case["gate"]]()
    for which in ("post", "pre"):
        on = case[which] != "none"
        w = uniform(C, lo=0.5, hi=1.5) - case["offset"]
        s[which + "_w"] = w.to(TYPES[case["weight"]]) if on else None
        s[which + "_b"] = normal(C, dtype=case["weight"], std=0.1) if on and case["bias"] else None
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
EPS = 1e-5


def run(state):
    c = state["case"]
    if own:
        return {"gemm_w4": _own_w4, "paged_attention": _own_attention, "block_norm": _own_norm}[c["op"]](state, c)
    return {"gemm_w4": _plain_w4, "paged_attention": _plain_attention, "block_norm": _plain_norm}[c["op"]](state, c)


def _own_w4(s, c):
    dn = _package()
    A, W, scale = s["A"], s["W"], s["scale"]
    C = torch.empty(c["M"], c["N"], device=DEV, dtype=A.dtype)
    d = dn.w4_desc(c["M"], c["N"], c["K"], c["K"], W.stride(0), c["N"], c["group"], scale.stride(0),
                   io_type=dn.TYPE_F32 if c["io"] == "f32" else dn.TYPE_BF16,
                   scale_type=dn.TYPE_F32 if c["scale"] == "f32" else dn.TYPE_BF16)
    dn.check(dn.cuda_gemm_w4(d, A, W, scale, s["zero"], s["bias"], C, torch.cuda.current_stream()),
             "cuda_gemm_w4")
    return {"C": C}


def _own_attention(s, c):
    dn = _package()
    q, k = s["q"], s["k"]
    kinds = {"f32": dn.TYPE_F32, "bf16": dn.TYPE_BF16, "e4m3": dn.TYPE_E4M3}
    token, head = (1, 2) if c["layout"] == "token" else (2, 1)
    out = torch.empty_like(q)
    lse = torch.empty(c["batch"], c["heads"], device=DEV)
    d = dn.paged_attn_desc(
        c["batch"], c["heads"], c["kv_heads"], c["dim"], c["page"], k.shape[0], s["table"].shape[1],
        io_type=kinds[c["io"]], cache_type=kinds[c["cache"]], page_stride=k.stride(0),
        token_stride=k.stride(token), head_stride=k.stride(head), scale=c["dim"] ** -0.5,
        softcap=c["softcap"], window=c["window"])
    dn.check(dn.cuda_paged_attention(d, q, k, s["v"], s["table"], s["lens"], out, lse=lse,
                                     k_new=s.get("k_new"), v_new=s.get("v_new"),
                                     stream=torch.cuda.current_stream()), "cuda_paged_attention")
    return {"out": out, "lse": lse, **({"k": k, "v": s["v"]} if c["append"] else {})}


def _own_norm(s, c):
    dn = _package()
    x, y, gate = s["x"], s["y"], s["gate"]
    kinds = {"none": dn.NORM_NONE, "rms": dn.NORM_RMS, "layer": dn.NORM_LAYER}
    h = torch.empty(c["rows"], c["cols"], device=DEV, dtype=x.dtype)
    z = torch.empty_like(h)
    d = dn.block_norm_desc(
        c["rows"], c["cols"], post=kinds[c["post"]], pre=kinds[c["pre"]],
        io_type=dn.TYPE_F32 if c["io"] == "f32" else dn.TYPE_BF16,
        weight_type=dn.TYPE_F32 if c["weight"] == "f32" else dn.TYPE_BF16, eps=EPS,
        weight_offset=c["offset"], residual_scale=c["residual"], block_scale=c["block"],
        ldx=x.stride(0), ldy=y.stride(0), ldh=c["cols"], ldz=c["cols"],
        ldg=c["cols"] if c["gate"] == "row" else 0)
    dn.check(dn.cuda_block_norm(d, x, y, gate, s["post_w"], s["post_b"], s["pre_w"], s["pre_b"], h, z,
                                torch.cuda.current_stream()), "cuda_block_norm")
    return {"h": h, "z": z}


def _plain_w4(s, c):
    K, W = c["K"], s["W"]
    code = torch.stack((W & 15, W >> 4), dim=2).reshape(W.shape[0], -1)[:, :K].float()
    group = c["group"] or K
    at = torch.arange(K, device=DEV) // group
    zero = 8.0 if s["zero"] is None else s["zero"].float()[:, at]
    out = s["A"].float() @ ((code - zero) * s["scale"].float()[:, at]).t()
    if s["bias"] is not None:
        out = out + s["bias"]
    return {"C": out.to(s["A"].dtype)}


def _plain_attention(s, c):
    B, H, KV, D, page = (c[k] for k in ("batch", "heads", "kv_heads", "dim", "page"))
    lens, table, k, v = s["lens"].long(), s["table"].long(), s["k"], s["v"]
    if c["append"]:
        live = (lens > 0).nonzero()[:, 0]
        at = lens[live] - 1
        where, slot = table[live, at // page], at % page
        for cache, new in ((k, s["k_new"]), (v, s["v_new"])):
            new = new[live].float()
            if c["cache"] == "e4m3":
                new = new.clamp(-448.0, 448.0)
            # The stored bytes are indexed: 8-bit floats have no indexed store.
            bits = torch.uint8 if c["cache"] == "e4m3" else cache.dtype
            rows = new.to(cache.dtype).view(bits)
            if c["layout"] == "token":
                cache.view(bits)[where, slot] = rows
            else:
                cache.view(bits)[where, :, slot] = rows

    def rows_of(cache):
        bits = torch.uint8 if c["cache"] == "e4m3" else cache.dtype
        got = cache.view(bits)[table.clamp(min=0)].view(cache.dtype).float()
        order = (0, 3, 1, 2, 4) if c["layout"] == "token" else (0, 2, 1, 3, 4)
        return got.permute(*order).reshape(B, KV, -1, D)

    keys, values = rows_of(k), rows_of(v)
    score = s["q"].float().reshape(B, KV, H // KV, D) @ keys.transpose(2, 3) * D ** -0.5
    if c["softcap"]:
        score = c["softcap"] * torch.tanh(score / c["softcap"])
    pos = torch.arange(score.shape[3], device=DEV)[None, :]
    seen = pos < lens[:, None]
    if c["window"]:
        seen = seen & (pos >= lens[:, None] - c["window"])
    score = torch.where(seen[:, None, None, :], score, -math.inf)
    top = score.amax(3, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(score - top)
    total = p.sum(3, keepdim=True)
    out = (p @ values) / torch.where(total == 0, torch.ones_like(total), total)
    lse = (top + torch.log(total)).reshape(B, H)
    out = out.reshape(B, H, D).to(s["q"].dtype)
    return {"out": out, "lse": lse, **({"k": k, "v": v} if c["append"] else {})}


def _plain_norm(s, c):
    def norm(v, kind, w, b):
        if kind == "none":
            return v
        if kind == "layer":
            v = v - v.mean(1, keepdim=True)
        v = v * torch.rsqrt((v * v).mean(1, keepdim=True) + EPS) * (w.float() + c["offset"])
        return v if b is None else v + b.float()

    block = norm(s["y"].float(), c["post"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        block = block * s["gate"].float()
    h = s["x"].float() * c["residual"] + block * c["block"]
    z = norm(h, c["pre"], s["pre_w"], s["pre_b"])
    return {"h": h.to(s["x"].dtype), "z": z.to(s["x"].dtype)}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "gemm_w4":
        M, N, K, io = c["M"], c["N"], c["K"], SIZE[c["io"]]
        b = N * ((K + 1) // 2) + N * _groups(c) * SIZE[c["scale"]] * (2 if c["zeros"] else 1)
        return {"bytes": b + io * (M * K + M * N) + (4 * N if c["bias"] else 0), "flops": 2 * M * N * K}
    if c["op"] == "paged_attention":
        lens = _lengths(c)
        seen = sum(min(n, c["window"]) if c["window"] else n for n in lens)
        row = c["kv_heads"] * c["dim"]
        b = 2 * seen * row * SIZE[c["cache"]] + c["batch"] * c["heads"] * (2 * c["dim"] * SIZE[c["io"]] + 4)
        if c["append"]:     # the new rows come from their own tensors and are stored once
            b += 2 * sum(n > 0 for n in lens) * row * SIZE[c["io"]]
        b += 4 * (c["batch"] + sum(-(-n // c["page"]) for n in lens))
        return {"bytes": b, "flops": 4 * seen * c["heads"] * c["dim"]}
    n, io = c["rows"] * c["cols"], SIZE[c["io"]]
    vectors = sum((c[k] != "none") * (2 if c["bias"] else 1) for k in ("post", "pre")) * SIZE[c["weight"]] * c["cols"]
    gates = {"none": 0, "channel": c["cols"], "row": n}[c["gate"]]
    return {"bytes": (4 * n + gates) * io + vectors, "flops": 12 * n}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "gemm_w4":
        # Group by group: sum over a group of a * code, less zero * the sum of a.
        A = s["A"].double()
        out = torch.zeros(c["M"], c["N"], device=DEV, dtype=torch.float64)
        if s["bias"] is not None:
            out += s["bias"].double()
        group = c["group"] or c["K"]
        for g in range(_groups(c)):
            lo, hi = g * group, min(c["K"], (g + 1) * group)
            part = torch.empty(c["N"], hi - lo, device=DEV, dtype=torch.float64)
            packed = s["W"][:, lo // 2:(hi + 1) // 2]
            part[:, 0::2] = (packed % 16).double()
            part[:, 1::2] = (packed // 16).double()[:, :(hi - lo) // 2]
            zero = s["zero"][:, g].double() if s["zero"] is not None else torch.full_like(part[:, 0], 8.0)
            a = A[:, lo:hi]
            out += (a @ part.t() - a.sum(1, keepdim=True) * zero) * s["scale"][:, g].double()
        return {"C": out}
    if c["op"] == "paged_attention":
        B, H, KV, D, page = (c[k] for k in ("batch", "heads", "kv_heads", "dim", "page"))
        out = torch.zeros(B, H, D, device=DEV, dtype=torch.float64)
        lse = torch.full((B, H), -math.inf, device=DEV, dtype=torch.float64)
        for b, n in enumerate(s["lens"].tolist()):
            first = max(0, n - c["window"]) if c["window"] else 0
            if n == 0:
                continue
            pages = s["table"][b, first // page:-(-n // page)].long()
            skip = first - first // page * page
            got = []
            for cache, new in ((s["k"], s.get("k_new")), (s["v"], s.get("v_new"))):
                rows = cache.view(torch.uint8)[pages].view(cache.dtype).float()
                rows = rows if c["layout"] == "token" else rows.transpose(1, 2)
                rows = rows.reshape(-1, KV, D)[skip:skip + n - first].double()
                if new is not None:
                    last = new[b].float().clamp(-448.0, 448.0) if c["cache"] == "e4m3" else new[b]
                    rows[-1] = last.to(cache.dtype).double()
                got.append(rows)
            for h in range(KV):
                q = s["q"][b, h * (H // KV):(h + 1) * (H // KV)].double()
                score = q @ got[0][:, h].t() / math.sqrt(D)
                if c["softcap"]:
                    score = c["softcap"] * torch.tanh(score / c["softcap"])
                total = torch.logsumexp(score, 1)
                at = slice(h * (H // KV), (h + 1) * (H // KV))
                lse[b, at] = total
                out[b, at] = torch.exp(score - total[:, None]) @ got[1][:, h]
        # The cache itself holds stored numbers, not computed ones.
        return {"out": out, "lse": lse, **({"k": None, "v": None} if c["append"] else {})}

    def norm(v, kind, w, b):
        if kind == "none":
            return v
        mean = v.mean(1, keepdim=True) if kind == "layer" else 0.0
        v = (v - mean) / torch.sqrt(((v - mean) ** 2).mean(1, keepdim=True) + EPS)
        return v * (w.double() + c["offset"]) + (b.double() if b is not None else 0.0)

    gate = s["gate"].double() if s["gate"] is not None else 1.0
    h = c["residual"] * s["x"].double() + c["block"] * gate * norm(s["y"].double(), c["post"], s["post_w"], s["post_b"])
    return {"h": h, "z": norm(h, c["pre"], s["pre_w"], s["pre_b"])}
