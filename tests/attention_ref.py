"""Plain implementations, in 64 bits, of the attention-side operators, for their GPU tests, with
the error bounds that go with them."""
from __future__ import annotations

import torch

U = 2.0 ** -24                                            # half a step of fp32
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def rounding(ref: torch.Tensor, dtype) -> torch.Tensor:
    """How far rounding to dtype may move ref."""
    return ref.abs() * HALF[dtype] + TINY[dtype]


def tables(P: int, R: int, base: float = 10000.0):
    freq = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    angle = torch.arange(P, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _turn(n, cos, sin, interleaved, back=False, absolute=False):
    """n [T, H, D] rotated; absolute: the sum of the terms' magnitudes."""
    h = cos.shape[-1]
    c, s = cos[:, None].double(), sin[:, None].double()
    s = -s if back else s
    if absolute:
        n, c, s = n.abs(), c.abs(), s.abs()
    a, b = (n[..., 0:2 * h:2], n[..., 1:2 * h:2]) if interleaved else (n[..., :h], n[..., h:2 * h])
    x, y = (a * c + b * s, b * c + a * s) if absolute else (a * c - b * s, b * c + a * s)
    r = torch.stack((x, y), -1).flatten(-2) if interleaved else torch.cat((x, y), -1)
    return torch.cat((r, n[..., 2 * h:]), -1)


def rope(x, w, cos, sin, positions, eps, interleaved):
    """(y, bound of fp32 arithmetic's error) of one of q and k; padding rows are zeros.

    A kernel's sum of D squares of 16 elements a lane errs by at most (16 + 5) U of itself, rstd
    by half of that and its own 4 roundings; norm and rotation add 2 + 2: 19 U, rounded to 24."""
    x, w = x.double(), w.double()
    real = (positions >= 0) & (positions < cos.shape[0])
    at = positions.clamp(0, max(0, cos.shape[0] - 1)).long()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    y = _turn(n, cos[at], sin[at], interleaved)
    off = 24 * U * _turn(n, cos[at], sin[at], interleaved, absolute=True)
    keep = real[:, None, None]
    return torch.where(keep, y, 0.0), torch.where(keep, off, 0.0)


def rope_bwd(dy, x, w, cos, sin, positions, eps, interleaved):
    """(dx, its bound, dw, its bound).

    dn errs by 2 U of its terms' magnitudes M; a = dn w by one more; the mean of a x by 24 U of
    the magnitudes' mean, and rstd by 15 U: all within 48 U of the magnitudes.  A weight's sum
    over n rows adds at most n + 16 roundings of the partial sums."""
    dy, x, w = dy.double(), x.double(), w.double()
    real = ((positions >= 0) & (positions < cos.shape[0]))[:, None, None]
    at = positions.clamp(0, max(0, cos.shape[0] - 1)).long()
    rstd = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    dn = _turn(dy, cos[at], sin[at], interleaved, back=True)
    mn = _turn(dy, cos[at], sin[at], interleaved, back=True, absolute=True)
    a, ma = dn * w, mn * w.abs()
    dx = rstd * (a - x * rstd ** 2 * (a * x).mean(-1, keepdim=True))
    mx = rstd * (ma + x.abs() * rstd ** 2 * (ma * x.abs()).mean(-1, keepdim=True))
    rows = x.shape[0] * x.shape[1]
    zero = torch.zeros((), dtype=torch.float64)
    dw = torch.where(real, dn * x * rstd, zero).sum((0, 1))
    mw = torch.where(real, mn * (x * rstd).abs(), zero).sum((0, 1))
    return (torch.where(real, dx, zero), torch.where(real, 48 * U * mx, zero), dw,
            (rows + 16 + 24) * U * mw)


QMAX = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def quantize(x, G, qdt, ue8m0):
    """Codes and scales of rows x [..., D], by the operator's own fp32 steps: amax * fp32(1/QMAX)
    (at least 1e-12), code = encode(x * (1 / s)), or 2^ceil(log2 s) and encode(x / s)."""
    f = x.float().unflatten(-1, (-1, G))
    s = f.abs().amax(-1) * torch.tensor(1.0 / QMAX[qdt], dtype=torch.float32)
    s = s.clamp_min(torch.tensor(1e-12, dtype=torch.float32))
    if ue8m0:
        m, e = torch.frexp(s)
        e = torch.where(m == 0.5, e - 1, e)
        t, stored = torch.ldexp(f, -e[..., None]), (e + 127).to(torch.uint8)
    else:
        t, stored = f * (1.0 / s)[..., None], s
    t = t.flatten(-2)
    return (t.to(qdt) if qdt != torch.int8 else torch.round(t).to(qdt)), stored


def scale_value(stored):
    return stored if stored.dtype == torch.float32 else torch.exp2(stored.double() - 127).float()


def dequantize(codes, scales):
    """[P, H, page, D] codes and [P, H, D/G, page] scales -> fp32 values (one rounding)."""
    s = scale_value(scales).transpose(-1, -2)
    return (codes.float().unflatten(-1, (s.shape[-1], -1)) * s[..., None]).flatten(-2)


def token_rows(values, pages, tokens, num_pages):
    """(rows [tokens, H, D], whether each has a page) of a list of pages of [P, H, page, D]."""
    page = values.shape[2]
    j = torch.arange(tokens)
    p = j // page
    has = p < len(pages)
    at = torch.tensor([int(pages[i]) if i < len(pages) else -1 for i in p.tolist()], dtype=torch.long)
    has &= (at >= 0) & (at < num_pages)
    rows = values[at.clamp(0, max(0, num_pages - 1)), :, j % page]
    return rows, has


def attention(q, kc, vc, ks, vs, table, lens, sm_scale, prefix_pages=None, prefix_len=0, most=None):
    """(out, bound) in 64 bits.

    x = q . k errs by (D + 4) U of its terms' magnitudes X (times log2 e and the scales' two
    roundings), which moves a probability by a factor e^(2 X (D + 4) U); probabilities are
    rounded to fp16 times their value scales (half a step each, and 2^-24 of the largest scale);
    n terms are summed in fp32 (n + 40 U)."""
    B, S, Hq, D = q.shape
    P, H, page, _ = kc.shape
    g = Hq // H
    kd = kc.float().double() * scale_value(ks).double().transpose(-1, -2)
    vd = vc.float().double() * scale_value(vs).double().transpose(-1, -2)
    sv = scale_value(vs).double()[:, :, 0, :, None].expand(vd.shape)
    room = table.shape[1] * page
    most = room if most is None else min(most, room)
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    off = torch.zeros_like(out)
    half = HALF[torch.float16]
    front = [token_rows(t, prefix_pages.tolist() if prefix_len else [], prefix_len, P)
             for t in (kd, vd, sv)]
    for b in range(B):
        n = max(0, min(int(lens[b]), most))
        own = [token_rows(t, table[b].tolist(), n, P) for t in (kd, vd, sv)]
        for s in range(S):
            seen = max(0, min(int(lens[b]), most) - S + s + 1)
            has = torch.cat((front[0][1], own[0][1][:seen]))
            k, v, w = (torch.cat((f[0], o[0][:seen]))[has] for f, o in zip(front, own))
            if k.shape[0] == 0:
                continue
            for h in range(H):
                qq = q[b, s, h * g:(h + 1) * g].double()
                x = qq @ k[:, h].T * sm_scale
                mx = (qq.abs() @ k[:, h].abs().T * abs(sm_scale)).amax(-1, keepdim=True)
                p = torch.softmax(x, -1)
                o, mo = p @ v[:, h], p @ v[:, h].abs()
                top = torch.exp(x - x.amax(-1, keepdim=True)).sum(-1, keepdim=True)
                spread = 2.0 ** -24 * w[:, h].amax() * (v[:, h].abs() / w[:, h].clamp_min(1e-300)).sum(0)
                out[b, s, h * g:(h + 1) * g] = o
                off[b, s, h * g:(h + 1) * g] = mo * (half + 4 * mx * (D + 4) * U
                                                    + (k.shape[0] + 40) * U) + spread / top
    return out, off


def outside(got, ref, bound, dtype):
    """How many values of got are further from ref than bound and a rounding to dtype."""
    d = (got.double().cpu() - ref).abs()
    return int((~(d <= bound + rounding(ref.abs() + bound, dtype))).sum())
