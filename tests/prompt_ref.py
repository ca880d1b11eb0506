"""Plain implementations, in 64 bits, of the attention of prompts, its gradients, draft trees over the
cache and a step's index tensors, for their GPU tests, with the error bounds that go with them."""
from __future__ import annotations

import torch

from tests import attention_ref as ref
from tests.attention_ref import HALF, U

# What 16 bits lose of a value however small it is (fp16's subnormals; bf16 has fp32's range).
LOST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}


def spans(cu, cu_k):
    """(q rows, k rows) of each sequence."""
    cu_k = cu if cu_k is None else cu_k
    return [(slice(int(cu[b]), int(cu[b + 1])), slice(int(cu_k[b]), int(cu_k[b + 1])))
            for b in range(len(cu) - 1)]


def hidden(n, m):
    """bool [n, m]: keys that a query does not see."""
    return torch.ones(n, m, dtype=torch.bool).triu(m - n + 1)


def forward(q, k, v, cu, sm_scale, cu_k=None):
    """(out, its bound, lse, its bound).

    x = scale q . k errs by (D + 4) U of its terms' magnitudes X, which moves e^x by a factor
    e^(2 X (D + 4) U); p, at most 2^8 and at least 1 for the largest, is rounded to 16 bits (half a
    step, and what fp16 loses of small ones, relative to the largest's); n terms are summed in
    fp32 (n + 40 U, exponential and division among them)."""
    T, Hq, D = q.shape
    g = Hq // k.shape[1]
    out, off = (torch.zeros(T, Hq, D, dtype=torch.float64) for _ in range(2))
    lse = torch.full((Hq, T), float("-inf"), dtype=torch.float64)
    lse_off = torch.zeros(Hq, T, dtype=torch.float64)
    for rows, keys in spans(cu, cu_k):
        n, m = rows.stop - rows.start, keys.stop - keys.start
        if n <= 0 or m <= 0:
            continue
        hide = hidden(n, m)
        some = ~hide.all(1)
        for h in range(Hq):
            qq, kk, vv = q[rows, h].double(), k[keys, h // g].double(), v[keys, h // g].double()
            x = (qq @ kk.T * sm_scale).masked_fill(hide, float("-inf"))
            mx = (qq.abs() @ kk.abs().T * abs(sm_scale)).masked_fill(hide, 0.0).amax(1)
            s = torch.logsumexp(x, 1)
            p = torch.exp(x - torch.where(some, s, 0.0)[:, None])
            top = torch.exp(x - torch.where(some, x.amax(1), 0.0)[:, None]).sum(1)
            rel = 4 * mx * (D + 4) * U + (m + 40) * U
            out[rows, h] = p @ vv
            lost = LOST[q.dtype] * ((~hide).double() @ vv.abs()) / top.clamp_min(1.0)[:, None]
            off[rows, h] = (p @ vv.abs()) * (HALF[q.dtype] + rel)[:, None] + lost
            lse[h, rows] = s
            lse_off[h, rows] = torch.where(some, rel + 8 * U * (s.abs() + 1), 0.0)
    return out, off, lse, lse_off


def backward(dout, q, k, v, out, lse, cu, sm_scale, cu_k=None):
    """((dq, bound), (dk, bound), (dv, bound)) for the out and lse that are given.

    P = e^(x - lse) errs by (4 X (D + 4) + 8 |lse| + 16) U of itself, dP and delta by (D + 8) U of
    their terms' magnitudes; P and dS are rounded to 16 bits; sums of n terms add (n + 8) U."""
    Hq, D, H = q.shape[1], q.shape[2], k.shape[1]
    g, half, lost = Hq // H, HALF[q.dtype], LOST[q.dtype]
    grads = [[torch.zeros(t.shape, dtype=torch.float64) for _ in range(2)] for t in (q, k, v)]
    (dq, dq_off), (dk, dk_off), (dv, dv_off) = grads
    for rows, keys in spans(cu, cu_k):
        n, m = rows.stop - rows.start, keys.stop - keys.start
        if n <= 0 or m <= 0:
            continue
        seen = ~hidden(n, m)
        for h in range(Hq):
            qq, do, oo = (t[rows, h].double() for t in (q, dout, out))
            kk, vv = k[keys, h // g].double(), v[keys, h // g].double()
            s = torch.where(seen.any(1), lse[h, rows].double(), 0.0)[:, None]
            x = qq @ kk.T * sm_scale
            mx = qq.abs() @ kk.abs().T * abs(sm_scale)
            p = torch.where(seen, torch.exp(x - s), 0.0)
            rel = (4 * mx * (D + 4) + 8 * s.abs() + 16) * U
            p_off = p * (rel + half) + lost * seen
            y = do @ vv.T - (do * oo).sum(1)[:, None]
            my = do.abs() @ vv.abs().T + (do * oo).abs().sum(1)[:, None]
            t = p * y
            t_off = p * (rel * y.abs() + (D + 8) * U * my) + half * t.abs() + lost * seen
            sums = (n * g + 24) * U
            dv[keys, h // g] += p.T @ do
            dv_off[keys, h // g] += (p_off + sums * p).T @ do.abs()
            dq[rows, h] = t @ kk * sm_scale
            dq_off[rows, h] = (t_off + (m + 24) * U * t.abs()) @ kk.abs() * abs(sm_scale)
            dk[keys, h // g] += t.T @ qq * sm_scale
            dk_off[keys, h // g] += (t_off + sums * t.abs()).T @ qq.abs() * abs(sm_scale)
    return tuple(map(tuple, grads))


def tree(q, kc, vc, ks, vs, table, lens, mask, sm_scale, prefix_pages=None, prefix_len=0, most=None):
    """(out, bound): `attention_ref.attention` with a mask; its bounds hold as they stand."""
    B, S, Hq, D = q.shape
    room = table.shape[1] * kc.shape[2]
    most = room if most is None else min(most, room)
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    off = torch.zeros_like(out)
    P, H, page, _ = kc.shape
    g = Hq // H
    kd = kc.float().double() * ref.scale_value(ks).double().transpose(-1, -2)
    vd = vc.float().double() * ref.scale_value(vs).double().transpose(-1, -2)
    sv = ref.scale_value(vs).double()[:, :, 0, :, None].expand(vd.shape)
    half = HALF[torch.float16]
    front = [ref.token_rows(t, prefix_pages.tolist() if prefix_len else [], prefix_len, P)
             for t in (kd, vd, sv)]
    for b in range(B):
        n = max(0, min(int(lens[b]), most))
        own = [ref.token_rows(t, table[b].tolist(), n, P) for t in (kd, vd, sv)]
        for s in range(S):
            row = mask[s] if mask.dim() == 2 else mask[b, s]
            j = torch.arange(n)
            seen = (j < n - S) | ((j >= n - S) & (row.bool()[(j - (n - S)).clamp(0, S - 1)]))
            has = torch.cat((front[0][1], own[0][1] & seen))
            k, v, w = (torch.cat((f[0], o[0]))[has] for f, o in zip(front, own))
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


def tables(context, new, free, table, page, rows, start=0):
    """What batch_tables returns, and the table, by a loop over the requests."""
    most = 2 ** 31 - 1
    table = table.clone()
    F, width = len(free), table.shape[1]
    positions, slots = torch.full((rows,), -1, dtype=torch.int32), torch.full((rows,), -1, dtype=torch.int64)
    cu, cu_k, lens = [0], [0], []
    start = max(0, int(start))
    at, total = start, 0
    for b in range(len(context)):
        ctx = min(max(0, int(context[b])), most)
        mine = min(max(0, int(new[b])), rows - cu[-1])
        n = min(ctx + mine, most)
        have, need = (min(width, -(-x // page)) for x in (ctx, n))
        for i in range(have, need):
            table[b, i] = free[at] if at < F else -1
            at += 1
        for j in range(mine):
            pos, r = ctx + j, cu[-1] + j
            i = pos // page
            p = int(table[b, i]) if i < width else -1
            positions[r] = min(pos, most)
            slots[r] = -1 if p < 0 else p * page + pos % page
        lens.append(n)
        total += n
        cu.append(cu[-1] + mine)
        cu_k.append(min(total, most))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32)
    return i32(cu), i32(cu_k), i32(lens), positions, slots, i32([min(at, most)]), table
