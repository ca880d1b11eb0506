"""The attention side of a decoder layer over a quantised paged cache, as measurable cases.

Five kinds of call, each through the entry point that a program uses:

* ``rope``: RMS norm of each query and key head and the rotation by position, from the views of a
  fused qkv projection (``qk_norm_rope``).
* ``rope_bwd``: its gradients for q, k and both norm weights (``qk_norm_rope_bwd``).
* ``write``: keys and values quantised into the pages of a cache (``kv_cache_write``).
* ``read``: the pages of a ragged batch gathered and dequantised (``kv_cache_read``).
* ``attn``: attention of the newest tokens of each sequence over its pages, and over the pages of a
  prefix that the whole batch shares (``paged_attention``).

With ``own`` false ``run`` computes the same in elementary torch operations in 32 bits.
"""
import functools
import math
import random

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "fp8": FP8,
          "int8": torch.int8}
SIZE = {"bf16": 2, "f16": 2, "f32": 4, "ue8m0": 1}
QMAX = {"fp8": 448.0, "int8": 127.0}
EPS = 1e-6
TABLE_ROWS = 32768       # positions of the rotation tables
MOST_BYTES = 1.0e9       # a drawn case moves no more than this, and multiplies no more than
MOST_FLOPS = 6.0e10      # this (the largest listed cases: 1.1e9 bytes, 6.9e10 operations)


# ------------------------------------------------------------------------------------ the cases

def _rope(name, T, Hq, Hk, D, R, act="bf16", interleaved=False, bwd=False):
    return {"name": name, "kind": "rope_bwd" if bwd else "rope", "T": T, "Hq": Hq, "Hk": Hk,
            "D": D, "R": R, "act": act, "interleaved": interleaved}


def _write(name, T, H, D, G, page, act="bf16", scale="f32", latent=False):
    return {"name": name, "kind": "write", "T": T, "H": H, "D": D, "G": G, "page": page,
            "act": act, "q": "fp8", "scale": scale, "latent": latent}


def _read(name, B, L, H, D, G, page, q="fp8", scale="f32", act="bf16", ragged=False):
    return {"name": name, "kind": "read", "B": B, "L": L, "H": H, "D": D, "G": G, "page": page,
            "q": q, "scale": scale, "act": act, "ragged": ragged}


def _attn(name, B, S, Hq, H, D, L, page, prefix=0, q="fp8", scale="f32", act="bf16", ragged=False):
    return {"name": name, "kind": "attn", "B": B, "S": S, "Hq": Hq, "H": H, "D": D, "G": D, "L": L,
            "page": page, "prefix": prefix, "q": q, "scale": scale, "act": act, "ragged": ragged}


def listed():
    return [
        # One decode step of 16 sequences: the smallest call, where the launch counts.
        _rope("rope_decode_16x32+8x128", 16, 32, 8, 128, 128),
        # One layer's prefill of the benchmark's 16384 tokens, 64 query heads.
        _rope("rope_prefill_16384x64+8x128", 16384, 64, 8, 128, 128),
        # A training step's backward over 8192 tokens.
        _rope("rope_bwd_8192x32+8x128", 8192, 32, 8, 128, 128, bwd=True),
        # A ragged one in 32 bits: 96-wide heads, a third of them rotated, in adjacent pairs.
        _rope("rope_bwd_777x12+12x96", 777, 12, 12, 96, 32, "f32", True, bwd=True),
        # A decode step of 128 sequences writes one token of each.
        _write("write_decode_128x8x128", 128, 8, 128, 128, 64),
        # A prefill of 16384 tokens writes its latents: 512 wide in groups of 128, UE8M0 scales.
        _write("write_latent_16384x1x512", 16384, 1, 512, 128, 64, scale="ue8m0", latent=True),
        # A chunk of a short ragged batch reads its context back, int8 codes.
        _read("read_ragged_5x613x8x128", 5, 613, 8, 128, 64, 16, q="int8", act="f16", ragged=True),
        # Eight contexts of 16384 tokens in 16 bits for a prefill that continues them.
        _read("read_long_8x16384x8x128", 8, 16384, 8, 128, 128, 64),
        # A decode step of four short sequences: latency counts.
        _attn("attn_decode_4x32+8x128_l1000", 4, 1, 32, 8, 128, 1000, 16, ragged=True, q="int8",
              act="f16"),
        # A decode step of a full batch with long contexts: the cache is read once.
        _attn("attn_decode_64x64+8x128_l8192", 64, 1, 64, 8, 128, 8192, 64),
        # Eight candidates behind one prompt, four tokens each to verify, 64-wide heads.
        _attn("attn_prefix_8x4x16+4x64_p2047", 8, 4, 16, 4, 64, 129, 32, prefix=2047, ragged=True,
              scale="ue8m0"),
        # A batch of 64 behind a prompt of 32768 tokens, each some hundred tokens on.
        _attn("attn_prefix_64x64+8x128_p32768", 64, 1, 64, 8, 128, 512, 64, prefix=32768,
              ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(("rope", "rope", "rope_bwd", "write", "read", "attn", "attn", "attn"))
    act16 = rng.choice(("bf16", "bf16", "f16"))
    page = rng.choice((16, 32, 64, 128))
    if kind in ("rope", "rope_bwd"):
        D = rng.choice((64, 80, 96, 128, 128, 192, 256))
        Hk = rng.choice((1, 2, 4, 8, 12))
        R = rng.choice((D, D, 32, 64))
        return _rope("", _log_int(rng, 1, 16384), Hk * rng.choice((1, 3, 4, 8)), Hk, D, R,
                     rng.choice((act16, act16, "f32")), rng.random() < 0.4, kind == "rope_bwd")
    if kind == "write":
        D = rng.choice((64, 128, 128, 192, 256, 512))
        G = rng.choice([g for g in (64, 128, 256) if D % g == 0])
        return _write("", _log_int(rng, 1, 16384), rng.choice((1, 2, 4, 8, 12)), D, G, page, act16,
                      rng.choice(("f32", "ue8m0")), rng.random() < 0.3)
    if kind == "read":
        D = rng.choice((64, 128, 128, 192, 256, 512))
        G = rng.choice([g for g in (64, 128, 256) if D % g == 0])
        return _read("", rng.randint(1, 48), _log_int(rng, 1, 16384), rng.choice((1, 2, 4, 8)), D,
                     G, page, rng.choice(("fp8", "int8")), rng.choice(("f32", "ue8m0")),
                     rng.choice((act16, "f32")), rng.random() < 0.7)
    H = rng.choice((1, 2, 4, 8))
    S = rng.choice((1, 1, 1, 2, 5, 16))
    prefix = rng.choice((0, 0, _log_int(rng, 64, 32768)))
    return _attn("", _log_int(rng, 1, 96), S, H * rng.choice((1, 4, 5, 8, 16)), H,
                 rng.choice((64, 128, 128, 256)), _log_int(rng, S, 2048 if prefix else 16384), page,
                 prefix, rng.choice(("fp8", "fp8", "int8")), rng.choice(("f32", "ue8m0")), act16,
                 rng.random() < 0.7)


def draw(rng):
    while True:
        case = _draw_once(rng)
        del case["name"]
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


# ------------------------------------------------------------------------------------ inputs

def _lens(case):
    """Tokens of each sequence's own pages.  A ragged batch spreads from the longest to a sixth of
    it, in mixed order; without a prefix its last slot is a padding one, of no tokens."""
    B, L, S = case["B"], case["L"], case.get("S", 1)
    if not case["ragged"]:
        return [L] * B
    lens = [max(S, L - (5 * L * b) // (6 * max(1, B - 1))) for b in range(B)]
    random.Random(B * 7919 + L).shuffle(lens)
    if B > 2 and not case.get("prefix"):
        lens[-1] = 0
    return lens


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _outliers(g, x):
    """x with the few large channels that keys and hidden states have in earnest."""
    channels = torch.randperm(x.shape[-1], generator=g, device=DEV)[:2]
    x[..., channels] *= 8.0
    return x


def _tables(R):
    """cos and sin of the angles, computed in 64 bits (far positions)."""
    freq = 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
    angle = torch.arange(TABLE_ROWS, device=DEV, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _scale_of(absmax, q, scale):
    """(scale as stored, its value): max(|x|) / QMAX, as UE8M0 the next power of two."""
    s = (absmax * (1.0 / QMAX[q])).clamp_min(1e-12)
    if scale == "f32":
        return s, s
    m, e = torch.frexp(s)
    e = torch.where(m == 0.5, e - 1, e)                 # ceil(log2 s), exactly
    return (e + 127).to(torch.uint8), torch.ldexp(torch.ones_like(s), e)


def _codes_of(t, q):
    return t.to(FP8) if q == "fp8" else torch.round(t).to(torch.int8)


def _value(stored):
    """The scale that a stored one stands for."""
    if stored.dtype == torch.float32:
        return stored
    return torch.ldexp(torch.ones(stored.shape, device=DEV), stored.to(torch.int32) - 127)


def _empty_cache(case, pages):
    H, D, G, page = (case[n] for n in ("H", "D", "G", "page"))
    codes = torch.zeros(pages, H, page, D, device=DEV, dtype=torch.int8).view(DTYPES[case["q"]])
    scale = torch.zeros(pages, H, D // G, page, device=DEV,
                        dtype=torch.uint8 if case["scale"] == "ue8m0" else torch.float32)
    return codes, scale


def _filled_cache(g, case, pages):
    """Codes and scales of normal rows with a few large channels."""
    H, D, G, page = (case[n] for n in ("H", "D", "G", "page"))
    x = _outliers(g, _randn(g, pages, H, page, D)).view(pages, H, page, D // G, G)
    stored, s = _scale_of(x.abs().amax(-1), case["q"], case["scale"])
    codes = _codes_of(x * (1.0 / s)[..., None], case["q"]).view(pages, H, page, D)
    return codes, stored.transpose(2, 3).contiguous()


def _page_table(order, lens, page):
    """int32 [B, most pages]: the next pages of `order` for each sequence, -1 behind its last."""
    width = max(1, max(-(-n // page) for n in lens))
    rows, at = [], 0
    for n in lens:
        need = -(-n // page)
        rows.append(order[at:at + need] + [-1] * (width - need))
        at += need
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    act = DTYPES[case["act"]]
    st = {"case": case}
    if kind in ("rope", "rope_bwd"):
        T, Hq, Hk, D, R = (case[n] for n in ("T", "Hq", "Hk", "D", "R"))
        qkv = _outliers(g, _randn(g, T, Hq + 2 * Hk, D)).to(act)
        st["q"], st["k"] = qkv[:, :Hq], qkv[:, Hq:Hq + Hk]
        st["q_weight"] = (1.0 + 0.1 * _randn(g, D)).to(act)
        st["k_weight"] = (1.0 + 0.1 * _randn(g, D)).to(act)
        st["cos"], st["sin"] = _tables(R)
        first = torch.randint(0, TABLE_ROWS - T, (1,), generator=g, device=DEV)
        st["positions"] = first + torch.arange(T, device=DEV)
        if kind == "rope_bwd":
            st["dq_out"] = _randn(g, T, Hq, D).to(act)
            st["dk_out"] = _randn(g, T, Hk, D).to(act)
        return st
    H, D, page = (case[n] for n in ("H", "D", "page"))
    if kind == "write":
        T = case["T"]
        pages = -(-T // page) + 3
        st["k"] = _outliers(g, _randn(g, T, H, D)).to(act)
        st["v"] = None if case["latent"] else _randn(g, T, H, D).to(act)
        st["slots"] = torch.randperm(pages * page, generator=g, device=DEV)[:T] if T <= 512 else \
            (torch.randperm(pages, generator=g, device=DEV)[:, None] * page
             + torch.arange(page, device=DEV)).view(-1)[:T].contiguous()
        st["k_cache"], st["k_scale"] = _empty_cache(case, pages)
        st["v_cache"], st["v_scale"] = (None, None) if case["latent"] else _empty_cache(case, pages)
        return st
    lens = _lens(case)
    prefix = case.get("prefix", 0)
    own_pages, prefix_pages = sum(-(-n // page) for n in lens), -(-prefix // page)
    pages = own_pages + prefix_pages + 3
    order = torch.randperm(pages, generator=g, device=DEV).tolist()
    st["k_cache"], st["k_scale"] = _filled_cache(g, case, pages)
    st["v_cache"], st["v_scale"] = _filled_cache(g, case, pages)
    st["page_table"] = _page_table(order, lens, page)
    if kind == "read":
        total = sum(lens)
        ends = torch.tensor(lens, dtype=torch.int32).cumsum(0, dtype=torch.int32)
        st["cu_seqlens"] = torch.cat([torch.zeros(1, dtype=torch.int32), ends]).to(DEV)
        st["k_out"] = torch.empty(total, H, D, dtype=act, device=DEV)
        st["v_out"] = torch.empty(total, H, D, dtype=act, device=DEV)
        return st
    B, S, Hq = case["B"], case["S"], case["Hq"]
    st["q"] = (2.0 * _randn(g, B, S, Hq, D)).to(act)
    st["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["prefix_pages"] = torch.tensor(order[own_pages:own_pages + prefix_pages], dtype=torch.int32,
                                      device=DEV) if prefix else None
    return st


# ------------------------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    return (_own if own else _PLAIN[case["kind"]])(state)


@functools.lru_cache(maxsize=None)
def _framework():
    from __graft_entry__ import load_package
    return load_package()


def _own(st):
    pkg = _framework()
    case, kind = st["case"], st["case"]["kind"]
    if kind == "rope":
        return pkg.qk_norm_rope(st["q"], st["k"], st["q_weight"], st["k_weight"], st["cos"],
                                st["sin"], st["positions"], EPS, interleaved=case["interleaved"])
    if kind == "rope_bwd":
        return pkg.qk_norm_rope_bwd(st["dq_out"], st["dk_out"], st["q"], st["k"], st["q_weight"],
                                    st["k_weight"], st["cos"], st["sin"], st["positions"], EPS,
                                    interleaved=case["interleaved"])
    if kind == "write":
        pkg.kv_cache_write(st["k"], st["v"], st["slots"], st["k_cache"], st["v_cache"],
                           st["k_scale"], st["v_scale"])
        return st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"]
    if kind == "read":
        return pkg.kv_cache_read(st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"],
                                 st["page_table"], st["cu_seqlens"], st["k_out"], st["v_out"])
    return pkg.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"],
                               st["page_table"], st["kv_lens"], case["D"] ** -0.5,
                               prefix_pages=st["prefix_pages"], prefix_len=case["prefix"])


# ------------------------------------------------------------------------------------ plain forms

def _rotate(n, cos, sin, interleaved, back=False):
    """The first R dims of n [T, H, D] rotated by cos, sin [T, R/2]; `back`: the other way."""
    half = cos.shape[-1]
    cos, sin = cos[:, None], -sin[:, None] if back else sin[:, None]
    r, rest = n[..., :2 * half], n[..., 2 * half:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :half], r[..., half:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((r, rest), -1)


def _plain_rope(st):
    cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]

    def one(x, w):
        f = x.float()
        n = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS) * w.float()
        return _rotate(n, cos, sin, st["case"]["interleaved"]).to(x.dtype)

    return one(st["q"], st["q_weight"]), one(st["k"], st["k_weight"])


def _plain_rope_bwd(st):
    cos, sin = st["cos"][st["positions"]], st["sin"][st["positions"]]

    def one(dy, x, w):
        f = x.float()
        rstd = torch.rsqrt(f.square().mean(-1, keepdim=True) + EPS)
        dn = _rotate(dy.float(), cos, sin, st["case"]["interleaved"], back=True)
        xh = f * rstd
        a = dn * w.float()
        dx = rstd * (a - xh * (a * xh).mean(-1, keepdim=True))
        return dx.to(x.dtype), (dn * xh).sum((0, 1))

    dq, dwq = one(st["dq_out"], st["q"], st["q_weight"])
    dk, dwk = one(st["dk_out"], st["k"], st["k_weight"])
    return dq, dk, dwq, dwk


def _plain_write_one(x, slots, cache, scale, case):
    if x is None:
        return
    T, H, D, G, page = (case[n] for n in ("T", "H", "D", "G", "page"))
    f = x.float().view(T, H, D // G, G)
    stored, s = _scale_of(f.abs().amax(-1), case["q"], case["scale"])
    codes = _codes_of(f * (1.0 / s)[..., None], case["q"]).view(T, H, D)
    at, off = slots // page, slots % page
    cache.view(torch.int8)[at, :, off] = codes.view(torch.int8)
    scale[at, :, :, off] = stored


def _plain_write(st):
    case = st["case"]
    _plain_write_one(st["k"], st["slots"], st["k_cache"], st["k_scale"], case)
    _plain_write_one(st["v"], st["slots"], st["v_cache"], st["v_scale"], case)
    return st["k_cache"], st["v_cache"], st["k_scale"], st["v_scale"]


def _pages_in_32_bits(cache, scale, pages):
    """codes * scale of pages [..., n] as float32 [..., n * page, H, D]."""
    c = cache.view(torch.int8)[pages].view(cache.dtype).float()
    s = _value(scale[pages]).transpose(-1, -2)                      # [..., n, H, page, D/G]
    c = c.view(*s.shape, -1) * s[..., None]
    return c.flatten(-2).transpose(-2, -3).flatten(-4, -3)


def _plain_read(st):
    case = st["case"]
    cu, page = st["cu_seqlens"].long(), case["page"]
    i = torch.arange(st["k_out"].shape[0], device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), i, right=True)
    j = i - cu[b]
    at, off = st["page_table"][b, j // page].long(), j % page
    for n in ("k", "v"):
        codes = st[n + "_cache"].view(torch.int8)[at, :, off].view(DTYPES[case["q"]]).float()
        s = _value(st[n + "_scale"][at, :, :, off])
        f = codes.view(*s.shape, -1) * s[..., None]
        st[n + "_out"].copy_(f.view(st[n + "_out"].shape))
    return st["k_out"], st["v_out"]


def _plain_attn(st):
    case = st["case"]
    B, S, Hq, H, D, P = (case[n] for n in ("B", "S", "Hq", "H", "D", "prefix"))
    g = Hq // H
    # Queries [B, H, D, S * g], each kv head's group together.
    q = st["q"].float().view(B, S, H, g, D).permute(0, 2, 4, 1, 3).reshape(B, H, D, S * g)
    q = q * D ** -0.5
    table = st["page_table"].clamp_min(0).long()
    k = _pages_in_32_bits(st["k_cache"], st["k_scale"], table).transpose(1, 2).contiguous()
    v = _pages_in_32_bits(st["v_cache"], st["v_scale"], table).transpose(1, 2).contiguous()
    s = torch.matmul(k, q)                                          # [B, H, L, S * g]
    L = s.shape[2]
    # Token s of the S newest sees the cache up to itself.
    seen = st["kv_lens"].long()[:, None] - S + 1 + torch.arange(S, device=DEV)
    mask = torch.arange(L, device=DEV)[None, :, None] < seen.repeat_interleave(g, 1)[:, None]
    s = s.masked_fill(~mask[:, None], float("-inf"))
    if P:
        kp = _pages_in_32_bits(st["k_cache"], st["k_scale"], st["prefix_pages"].long())
        vp = _pages_in_32_bits(st["v_cache"], st["v_scale"], st["prefix_pages"].long())
        kp, vp = (t[:P].transpose(0, 1).contiguous() for t in (kp, vp))     # [H, P, D]
        rows = q.permute(1, 2, 0, 3).reshape(H, D, B * S * g)
        sp = torch.matmul(kp, rows).view(H, P, B, S * g).permute(2, 0, 1, 3)
        s = torch.cat((sp, s), 2)
    top = s.amax(2, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    total = p.sum(2)
    p, own_p = p[:, :, :P], p[:, :, P:]
    o = torch.matmul(own_p.transpose(2, 3).contiguous(), v)         # [B, H, S * g, D]
    if P:
        rows = p.permute(1, 0, 3, 2).reshape(H, B * S * g, P)
        o = o + torch.matmul(rows, vp).view(H, B, S * g, D).transpose(0, 1)
    o = torch.where(total[..., None] > 0, o / total[..., None], 0.0)
    return o.view(B, H, S, g, D).transpose(1, 2).reshape(B, S, Hq, D).to(st["q"].dtype)


_PLAIN = {"rope": _plain_rope, "rope_bwd": _plain_rope_bwd, "write": _plain_write,
          "read": _plain_read, "attn": _plain_attn}


# ------------------------------------------------------------------------------------ its work

def work(case):
    kind = case["kind"]
    if kind in ("rope", "rope_bwd"):
        T, D, R, e = case["T"], case["D"], case["R"], SIZE[case["act"]]
        n = T * (case["Hq"] + case["Hk"]) * D
        table = T * (R * 4 + 8) + 2 * D * e
        if kind == "rope":
            return {"bytes": 2 * n * e + table, "flops": 8 * n}
        return {"bytes": 3 * n * e + table + 8 * D, "flops": 16 * n}
    H, D = case["H"], case["D"]
    row = H * (D + D // case["G"] * SIZE[case["scale"]])            # a token's codes and scales
    e = SIZE[case["act"]]
    if kind == "write":
        T, n = case["T"], 1 if case["latent"] else 2
        return {"bytes": n * T * (H * D * e + row) + 8 * T, "flops": n * T * H * D * 3}
    lens, page = _lens(case), case["page"]
    pages = 4 * sum(-(-n // page) for n in lens)
    if kind == "read":
        total = sum(lens)
        return {"bytes": 2 * total * (row + H * D * e) + pages, "flops": 2 * total * H * D}
    B, S, Hq, P = case["B"], case["S"], case["Hq"], case["prefix"]
    seen = sum(min(n, max(0, n - S + 1 + s)) for n in lens for s in range(S)) + B * S * P
    return {"bytes": 2 * (sum(lens) + P) * row + 2 * B * S * Hq * D * e + pages + 4 * B
            + 4 * -(-P // page), "flops": 4 * seen * Hq * D}


# ------------------------------------------------------------------------------------ in 64 bits

def _rope_in_64_bits(x, w, cos, sin, interleaved):
    """The norm and the rotation as products of complex numbers."""
    n = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * w
    R = 2 * cos.shape[-1]
    turn = torch.complex(cos, sin)[:, None]
    pairs = n[..., :R].unflatten(-1, (-1, 2) if interleaved else (2, -1))
    z = torch.complex(*pairs.unbind(-1 if interleaved else -2)) * turn
    return torch.cat((torch.stack((z.real, z.imag), -1 if interleaved else -2).flatten(-2),
                      n[..., R:]), -1)


def _dequantized(codes, stored):
    """codes [H, page, D] of one page or [n, H, page, D], times their scales, in 64 bits."""
    s = stored.double() if stored.dtype == torch.float32 else torch.exp2(stored.double() - 127.0)
    G = codes.shape[-1] // s.shape[-2]
    return codes.float().double() * s.transpose(-1, -2).repeat_interleave(G, -1)


def _sequence(st, n, pages, count):
    """The first `count` rows [H, count, D] of a list of pages, in 64 bits."""
    codes, scale = st[n + "_cache"], st[n + "_scale"]
    f = _dequantized(codes.view(torch.int8)[pages].view(codes.dtype), scale[pages])
    return f.transpose(0, 1).flatten(1, 2)[:, :count].contiguous()


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind in ("rope", "rope_bwd"):
        cos, sin = (st[n][st["positions"]].double() for n in ("cos", "sin"))
        leaves = [st[n].double() for n in ("q", "k", "q_weight", "k_weight")]
        grad = kind == "rope_bwd"
        leaves = [t.requires_grad_() for t in leaves] if grad else leaves
        y = [_rope_in_64_bits(leaves[i], leaves[2 + i], cos, sin, case["interleaved"])
             for i in (0, 1)]
        if not grad:
            return tuple(y)
        return torch.autograd.grad(y, leaves, [st["dq_out"].double(), st["dk_out"].double()])
    if kind == "write":
        # The codes are real numbers here.  No largest magnitude of 16-bit values lies so near a
        # power of two times QMAX that 32 and 64 bits would take different UE8M0 steps.
        got = []
        for n in ("k", "v"):
            if st[n] is None:
                got.append((None, None))
                continue
            x = st[n].double().unflatten(-1, (-1, case["G"]))
            s = (x.abs().amax(-1) / QMAX[case["q"]]).clamp_min(1e-12)
            ue8m0 = case["scale"] == "ue8m0"
            if ue8m0:
                s = torch.exp2(torch.ceil(torch.log2(s)))
            codes, scale = st[n + "_cache"].float().double(), st[n + "_scale"].double()
            at, off = st["slots"] // case["page"], st["slots"] % case["page"]
            codes[at, :, off] = (x / s[..., None]).flatten(-2)
            scale[at, :, :, off] = s
            got.append((codes, None if ue8m0 else scale))
        (kc, ks), (vc, vs) = got
        return kc, vc, ks, vs
    lens, table = _lens(case), st["page_table"].long()
    page = case["page"]
    if kind == "read":
        return tuple(torch.cat([_sequence(st, n, table[b, :-(-c // page)], c).transpose(0, 1)
                                for b, c in enumerate(lens)]) for n in ("k", "v"))
    B, S, Hq, H, D, P = (case[n] for n in ("B", "S", "Hq", "H", "D", "prefix"))
    if P:
        front = [_sequence(st, n, st["prefix_pages"].long(), P) for n in ("k", "v")]
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64, device=DEV)
    for b, c in enumerate(lens):
        k, v = (_sequence(st, n, table[b, :-(-c // page)], c) for n in ("k", "v"))
        if P:
            k, v = torch.cat((front[0], k), 1), torch.cat((front[1], v), 1)
        for s in range(S):
            seen = P + max(0, c - S + 1 + s)
            if seen == 0:
                continue
            q = st["q"][b, s].double().view(H, Hq // H, D)
            a = torch.softmax(torch.matmul(q, k[:, :seen].transpose(1, 2).contiguous())
                              / math.sqrt(D), -1)
            out[b, s] = torch.matmul(a, v[:, :seen].contiguous()).view(Hq, D)
    return out
