"""Attention of whole prompts and of drafted tokens, and a step's index tensors, as measurable cases.

Four kinds of call, each through the entry point that a program uses:

* ``prompt``: causal attention of packed sequences with grouped heads, their keys as long as their
  queries or longer (``prompt_attention``).
* ``prompt_bwd``: its gradients (``prompt_attention_bwd``).
* ``tree``: attention of a tree of drafted tokens over a quantised paged cache
  (``paged_tree_attention``).
* ``tables``: page table, slots, positions and cumulative lengths of a step from the requests'
  lengths (``batch_tables``).

With ``own`` false ``run`` computes the same in elementary torch operations in 32 bits.
"""
import functools
import math
import random

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": FP8, "int8": torch.int8}
QMAX = {"fp8": 448.0, "int8": 127.0}
SCORES = 1 << 28         # scores that the plain forms hold at a time
MOST_FLOPS = 1.3e12      # a drawn case multiplies no more than this and moves no more than that
MOST_BYTES = 5.0e8       # (the largest listed ones: 4.4e12 operations, 6.0e8 bytes)


# ------------------------------------------------------------------------------------ the cases

def _prompt(name, B, L, Hq, H, D, ctx=0, act="bf16", ragged=False, lse=False, bwd=False):
    """B sequences of L new tokens behind contexts of ctx."""
    return {"name": name, "kind": "prompt_bwd" if bwd else "prompt", "B": B, "L": L, "Hq": Hq,
            "H": H, "D": D, "ctx": ctx, "act": act, "ragged": ragged, "lse": lse}


def _tree(name, B, S, Hq, H, D, L, page, prefix=0, q="fp8", scale="f32", act="bf16", ragged=False):
    """B sequences of L tokens in the cache, the newest S of them drafts."""
    return {"name": name, "kind": "tree", "B": B, "S": S, "Hq": Hq, "H": H, "D": D, "L": L,
            "page": page, "prefix": prefix, "q": q, "scale": scale, "act": act, "ragged": ragged}


def _tables(name, B, new, ctx, page, spare, idx="i32", ragged=False):
    """B requests of `new` tokens behind ctx cached ones; `spare` rows behind the last."""
    return {"name": name, "kind": "tables", "B": B, "L": new, "ctx": ctx, "page": page,
            "spare": spare, "idx": idx, "ragged": ragged}


def listed():
    return [
        # A few short requests join a running batch: the smallest prefill, where latency counts.
        _prompt("prompt_short_4x200_32+8x128", 4, 200, 32, 8, 128, ragged=True),
        # One prompt of the benchmark's 16384 tokens, 64 query heads.
        _prompt("prompt_16384_64+8x128", 1, 16384, 64, 8, 128),
        # The forward of a training step over 16 packed documents, with what its backward needs.
        _prompt("prompt_packed_16x1000_32+8x128", 16, 1000, 32, 8, 128, ragged=True, lse=True),
        # Chunks of 512 tokens that continue contexts of 4096, wide heads.
        _prompt("prompt_chunk_4x512_c4096_16+4x256", 4, 512, 16, 4, 256, ctx=4096, act="f16"),
        # A small ragged training batch, as many kv heads as query heads, 64 wide.
        _prompt("bwd_5x77_12+12x64", 5, 77, 12, 12, 64, act="f16", ragged=True, bwd=True),
        # The backward of the packed documents.
        _prompt("bwd_packed_16x1000_32+8x128", 16, 1000, 32, 8, 128, ragged=True, bwd=True),
        # The backward of one long sequence.
        _prompt("bwd_8192_32+8x128", 1, 8192, 32, 8, 128, bwd=True),
        # Sixteen drafts behind four short contexts: latency counts.
        _tree("tree_4x16_32+8x128_l1000", 4, 16, 32, 8, 128, 1000, 16, q="int8", act="f16",
              ragged=True),
        # A full batch with long contexts, 32 drafts each: the cache is read once.
        _tree("tree_32x32_64+8x128_l8192", 32, 32, 64, 8, 128, 8192, 64),
        # Eight candidates behind one prompt, 63 drafts each, 64-wide heads.
        _tree("tree_8x63_16+4x64_p2047", 8, 63, 16, 4, 64, 129, 32, prefix=2047, scale="ue8m0",
              ragged=True),
        # A decode step of 256 requests.
        _tables("tables_decode_256", 256, 1, 8192, 64, 0, ragged=True),
        # Prompts of a full batch are admitted at once, into pages of 16.
        _tables("tables_admit_64x16384", 64, 16384, 0, 16, 1000, "i64", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    kind = rng.choice(("prompt", "prompt", "prompt", "prompt_bwd", "prompt_bwd", "tree", "tree",
                       "tables"))
    act = rng.choice(("bf16", "bf16", "f16"))
    ragged = rng.random() < 0.7
    page = rng.choice((16, 32, 64, 128))
    if kind == "tables":
        return _tables("", _log_int(rng, 1, 512), _log_int(rng, 1, 4096),
                       rng.choice((0, _log_int(rng, 1, 16384))), page, rng.choice((0, 1, 777)),
                       rng.choice(("i32", "i64")), ragged)
    H = rng.choice((1, 2, 4, 8))
    D = rng.choice((64, 128, 128, 256))
    if kind == "tree":
        S = _log_int(rng, 2, 128)
        prefix = rng.choice((0, 0, _log_int(rng, 64, 16384)))
        return _tree("", _log_int(rng, 1, 48), S, H * rng.choice((1, 4, 5, 8)), H, D,
                     S + _log_int(rng, 1, 1024 if prefix else 8192), page, prefix,
                     rng.choice(("fp8", "int8")), rng.choice(("f32", "ue8m0")), act, ragged)
    bwd = kind == "prompt_bwd"
    return _prompt("", _log_int(rng, 1, 32), _log_int(rng, 1, 8192), H * rng.choice((1, 3, 4, 8)),
                   H, D, rng.choice((0, 0, 0, _log_int(rng, 1, 8192))), act, ragged,
                   rng.random() < 0.3 and not bwd, bwd)


def draw(rng):
    while True:
        case = _draw_once(rng)
        del case["name"]
        w = work(case)
        if w["bytes"] <= MOST_BYTES and w["flops"] <= MOST_FLOPS:
            return case


# ------------------------------------------------------------------------------------ inputs

def _spread(n, B, least, seed):
    """Lengths from n down to a sixth of it, in mixed order."""
    lens = [max(least, n - (5 * n * b) // (6 * max(1, B - 1))) for b in range(B)]
    random.Random(seed).shuffle(lens)
    return lens


def _lens(case):
    """(new tokens, tokens of the context before them) of each sequence; a ragged batch of more than
    two holds a padding slot, of no tokens at all."""
    B, n, ctx, kind = case["B"], case["L"], case.get("ctx", 0), case["kind"]
    if not case["ragged"]:
        return [n] * B, [ctx] * B
    if kind == "tree":
        return _spread(n, B, case["S"], B * 7919 + n), [0] * B
    new = _spread(n, B, 1, B * 7919 + n)
    old = _spread(ctx, B, 0, B * 104729 + ctx)
    if B > 2:
        new[-1] = old[-1] = 0
    return new, old


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _outliers(g, x):
    """x with the few large channels that keys and hidden states have in earnest."""
    channels = torch.randperm(x.shape[-1], generator=g, device=DEV)[:2]
    x[..., channels] *= 4.0
    return x


def _cumulative(lens):
    return torch.tensor([0] + lens).cumsum(0, dtype=torch.int32).to(DEV)


def _value(stored):
    """The scale that a stored one stands for."""
    if stored.dtype == torch.float32:
        return stored
    return torch.ldexp(torch.ones(stored.shape, device=DEV), stored.to(torch.int32) - 127)


def _filled_cache(g, case, pages):
    """Codes and scales of normal rows with a few large channels, a scale for each row."""
    x = _outliers(g, _randn(g, pages, case["H"], case["page"], case["D"]))
    s = (x.abs().amax(-1) / QMAX[case["q"]]).clamp_min(1e-12)
    if case["scale"] == "ue8m0":
        m, e = torch.frexp(s)
        e = torch.where(m == 0.5, e - 1, e)                 # ceil(log2 s), exactly
        stored, s = (e + 127).to(torch.uint8), torch.ldexp(torch.ones_like(s), e)
    else:
        stored = s
    x = x / s[..., None]
    codes = x.to(FP8) if case["q"] == "fp8" else torch.round(x).to(torch.int8)
    return codes, stored[:, :, None].contiguous()


def _draft_masks(g, B, S):
    """bool [B, S, S]: a draft sees itself and what its parent sees; a parent is one of the eight
    drafts before it, or the context."""
    back = torch.randint(1, 9, (B, S), generator=g, device=DEV).cpu().tolist()
    mask = torch.zeros(B, S, S, dtype=torch.bool)
    for b in range(B):
        for s in range(S):
            parent = s - back[b][s]
            if parent >= 0:
                mask[b, s] = mask[b, parent]
            mask[b, s, s] = True
    return mask.to(DEV)


def _prepare_prompt(g, case, st):
    new, old = _lens(case)
    Hq, H, D, act = case["Hq"], case["H"], case["D"], DTYPES[case["act"]]
    T = sum(new)
    st["new"], st["both"] = new, [a + b for a, b in zip(new, old)]
    st["cu"] = _cumulative(new)
    st["cu_k"] = _cumulative(st["both"]) if case["ctx"] else None
    # Without a context q, k and v are views of one projection; with one, k and v were gathered.
    if case["ctx"]:
        st["q"] = (1.5 * _outliers(g, _randn(g, T, Hq, D))).to(act)
        Tk = sum(st["both"])
        st["k"] = _outliers(g, _randn(g, Tk, H, D)).to(act)
        st["v"] = _randn(g, Tk, H, D).to(act)
    else:
        qkv = _randn(g, T, Hq + 2 * H, D)
        qkv[:, :Hq] *= 1.5
        qkv = _outliers(g, qkv).to(act)
        st["q"], st["k"], st["v"] = qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:]
    if case["kind"] == "prompt_bwd":
        st["out"], st["lse"] = _plain_prompt(st, True)
        st["dout"] = _randn(g, T, Hq, D).to(act)


def _prepare_tables(g, case, st):
    new, old = _lens(case)
    B, page = case["B"], case["page"]
    have = [-(-n // page) for n in old]
    need = [-(-(n + c) // page) for n, c in zip(new, old)]
    width = max(need) + 1
    pages = sum(need) + 5
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    before = torch.tensor([0] + have[:-1], device=DEV).cumsum(0)
    i = torch.arange(width, device=DEV)
    st["page_table"] = torch.where(i < torch.tensor(have, device=DEV)[:, None],
                                   order[(before[:, None] + i).clamp_max(pages - 1)],
                                   -1).to(torch.int32)
    st["free_pages"] = order[sum(have):].contiguous()
    dtype = torch.int32 if case["idx"] == "i32" else torch.int64
    st["new_lens"] = torch.tensor(new, dtype=dtype, device=DEV)
    st["context_lens"] = torch.tensor(old, dtype=dtype, device=DEV)
    st["rows"] = sum(new) + case["spare"]


def _prepare_tree(g, case, st):
    B, S, page, prefix = (case[n] for n in ("B", "S", "page", "prefix"))
    lens, _ = _lens(case)
    need = [-(-n // page) for n in lens]
    own_pages, prefix_pages = sum(need), -(-prefix // page)
    order = torch.randperm(own_pages + prefix_pages + 3, generator=g, device=DEV).to(torch.int32)
    st["k_cache"], st["k_scale"] = _filled_cache(g, case, len(order))
    st["v_cache"], st["v_scale"] = _filled_cache(g, case, len(order))
    before = torch.tensor([0] + need[:-1], device=DEV).cumsum(0)
    i = torch.arange(max(need), device=DEV)
    st["page_table"] = torch.where(i < torch.tensor(need, device=DEV)[:, None],
                                   order[(before[:, None] + i).clamp_max(len(order) - 1)],
                                   -1).to(torch.int32)
    st["prefix_pages"] = order[own_pages:own_pages + prefix_pages].contiguous() if prefix else None
    st["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st["tree_mask"] = _draft_masks(g, B, S)
    st["q"] = (2.0 * _randn(g, B, S, case["Hq"], case["D"])).to(DTYPES[case["act"]])


def prepare(case, seed):
    st = {"case": case}
    kind = "prompt" if case["kind"] == "prompt_bwd" else case["kind"]
    {"prompt": _prepare_prompt, "tree": _prepare_tree, "tables": _prepare_tables}[kind](
        _gen(seed), case, st)
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
    if kind == "prompt":
        return pkg.prompt_attention(st["q"], st["k"], st["v"], st["cu"], case["D"] ** -0.5,
                                    cu_seqlens_k=st["cu_k"], return_lse=case["lse"])
    if kind == "prompt_bwd":
        return pkg.prompt_attention_bwd(st["dout"], st["q"], st["k"], st["v"], st["out"], st["lse"],
                                        st["cu"], case["D"] ** -0.5, cu_seqlens_k=st["cu_k"])
    if kind == "tree":
        return pkg.paged_tree_attention(st["q"], st["k_cache"], st["v_cache"], st["k_scale"],
                                        st["v_scale"], st["page_table"], st["kv_lens"],
                                        st["tree_mask"], case["D"] ** -0.5,
                                        prefix_pages=st["prefix_pages"], prefix_len=case["prefix"])
    return (*pkg.batch_tables(st["context_lens"], st["new_lens"], st["free_pages"],
                              st["page_table"], case["page"], st["rows"]), st["page_table"])


# ------------------------------------------------------------------------------------ plain forms

def _pieces(st):
    """Each sequence's (rows of q, rows of k), and its queries in pieces of so many scores:
    (sequence's first q row, first k row, first and last query, keys that they see)."""
    Hq, at, at_k = st["case"]["Hq"], 0, 0
    for n, m in zip(st["new"], st["both"]):
        step = max(1, SCORES // (Hq * max(1, m)))
        for i in range(0, n, step):
            stop = min(n, i + step)
            yield at, at_k, i, stop, m - n + stop, m - n
        at, at_k = at + n, at_k + m


def _heads_first(x, H):
    """[n, H * g, D] -> [H, g * n, D] in 32 bits."""
    n, Hq, D = x.shape
    return x.float().view(n, H, Hq // H, D).permute(1, 2, 0, 3).reshape(H, -1, D)


def _tokens_first(x, n):
    """[H, g * n, D] -> [n, H * g, D]"""
    H, _, D = x.shape
    return x.view(H, -1, n, D).permute(2, 0, 1, 3).reshape(n, -1, D)


def _scores(q, k, n, first):
    """Scores [H, g * n, m] of queries [H, g * n, D]; what a query does not see is -inf."""
    s = torch.matmul(q, k.permute(1, 2, 0).contiguous())
    m = s.shape[-1]
    hidden = torch.arange(m, device=DEV) > first + torch.arange(n, device=DEV)[:, None]
    return s.view(s.shape[0], -1, n, m).masked_fill_(hidden, float("-inf")).view(s.shape)


def _plain_prompt(st, lse=None):
    case = st["case"]
    H, scale = case["H"], case["D"] ** -0.5
    q, k, v = st["q"], st["k"], st["v"]
    out = torch.zeros(q.shape, dtype=q.dtype, device=DEV)
    sums = torch.full((q.shape[1], q.shape[0]), float("-inf"), device=DEV)
    for at, at_k, i, stop, m, ahead in _pieces(st):
        n = stop - i
        s = _scores(_heads_first(q[at + i:at + stop], H) * scale, k[at_k:at_k + m].float(), n,
                    ahead + i)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s.sub_(top))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, v[at_k:at_k + m].float().transpose(0, 1).contiguous()) / total
        out[at + i:at + stop] = _tokens_first(o, n).to(q.dtype)
        sums[:, at + i:at + stop] = (top + torch.log(total)).view(-1, n)
    return (out, sums) if (case["lse"] if lse is None else lse) else out


def _plain_prompt_bwd(st):
    case = st["case"]
    H, D = case["H"], case["D"]
    q, k, v = st["q"], st["k"], st["v"]
    dq = torch.zeros(q.shape, device=DEV)
    dk, dv = torch.zeros(k.shape, device=DEV), torch.zeros(v.shape, device=DEV)
    for at, at_k, i, stop, m, ahead in _pieces(st):
        n, rows = stop - i, slice(at + i, at + stop)
        qs, do = _heads_first(q[rows], H), _heads_first(st["dout"][rows], H)
        ks, vs = k[at_k:at_k + m].float(), v[at_k:at_k + m].float()
        s = _scores(qs * D ** -0.5, ks, n, ahead + i)
        p = torch.exp(s.sub_(st["lse"][:, rows].reshape(H, -1, 1)))
        delta = (do * _heads_first(st["out"][rows], H)).sum(-1, keepdim=True)
        ds = torch.matmul(do, vs.permute(1, 2, 0).contiguous()).sub_(delta).mul_(p).mul_(D ** -0.5)
        dq[rows] = _tokens_first(torch.matmul(ds, ks.transpose(0, 1).contiguous()), n)
        dk[at_k:at_k + m] += torch.matmul(ds.transpose(1, 2), qs).transpose(0, 1)
        dv[at_k:at_k + m] += torch.matmul(p.transpose(1, 2), do).transpose(0, 1)
    return dq.to(q.dtype), dk.to(q.dtype), dv.to(q.dtype)


def _pages_in_32_bits(cache, scale, pages):
    """codes * scale of pages [..., n] as float32 [..., n * page, H, D]."""
    c = cache.view(torch.int8)[pages].view(cache.dtype).float() * _value(scale[pages])[..., 0, :, None]
    return c.transpose(-2, -3).flatten(-4, -3)


def _plain_tree(st):
    case = st["case"]
    B, S, Hq, H, D, P = (case[n] for n in ("B", "S", "Hq", "H", "D", "prefix"))
    g = Hq // H
    q = st["q"].float().view(B, S, H, g, D).permute(0, 2, 4, 3, 1).reshape(B, H, D, g * S)
    q = q * D ** -0.5
    lens = st["kv_lens"].long()
    out = torch.empty(B, H, g * S, D, device=DEV)
    if P:
        kp = _pages_in_32_bits(st["k_cache"], st["k_scale"], st["prefix_pages"].long())
        vp = _pages_in_32_bits(st["v_cache"], st["v_scale"], st["prefix_pages"].long())
        kp, vp = (t[:P].transpose(0, 1).contiguous() for t in (kp, vp))
    L = st["page_table"].shape[1] * case["page"]
    step = max(1, SCORES // (Hq * S * (L + P)))
    for b in range(0, B, step):
        at = slice(b, b + step)
        table = st["page_table"][at].clamp_min(0).long()
        k = _pages_in_32_bits(st["k_cache"], st["k_scale"], table).transpose(1, 2).contiguous()
        v = _pages_in_32_bits(st["v_cache"], st["v_scale"], table).transpose(1, 2).contiguous()
        # Key j of a sequence is draft j - (len - S); the ones before are its context.
        draft = torch.arange(L, device=DEV) - (lens[at, None] - S)          # [b, L]
        seen = st["tree_mask"][at].gather(2, draft.clamp(0, S - 1)[:, None].expand(-1, S, -1))
        seen = torch.where((draft >= 0)[:, None], seen & (draft < S)[:, None], True)
        if P:
            k, v = (torch.cat((f.expand(k.shape[0], -1, -1, -1), own_), 2)
                    for f, own_ in ((kp, k), (vp, v)))
            seen = torch.cat((torch.ones(*seen.shape[:2], P, dtype=torch.bool, device=DEV), seen), 2)
        s = torch.matmul(k, q[at]).view(-1, H, P + L, g, S)
        s = s.masked_fill(~seen.transpose(1, 2)[:, None, :, None], float("-inf")).flatten(-2)
        p = torch.exp(s - s.amax(2, keepdim=True))
        out[at] = torch.matmul(p.transpose(2, 3).contiguous(), v) / p.sum(2)[..., None]
    return out.view(B, H, g, S, D).permute(0, 3, 1, 2, 4).reshape(B, S, Hq, D).to(st["q"].dtype)


def _plain_tables(st):
    case, page, rows = st["case"], st["case"]["page"], st["rows"]
    new, ctx, table = st["new_lens"].long(), st["context_lens"].long(), st["page_table"]
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    cu, kv = torch.cat((zero, new.cumsum(0))), ctx + new
    have, need = (ctx + page - 1) // page, (kv + page - 1) // page
    first = torch.cat((zero, (need - have).cumsum(0)))
    i = torch.arange(table.shape[1], device=DEV)
    fresh = (i >= have[:, None]) & (i < need[:, None])
    taken = (first[:-1] - have)[:, None] + i
    table.copy_(torch.where(fresh, st["free_pages"][taken.clamp(0, len(st["free_pages"]) - 1)], table))
    row = torch.arange(rows, device=DEV)
    b = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    real = b < len(new)
    b = b.clamp_max(len(new) - 1)
    position = ctx[b] + row - cu[b]
    at = table.view(-1)[b * table.shape[1] + (position // page).clamp_max(table.shape[1] - 1)].long()
    slots = torch.where(real, at * page + position % page, -1)
    return (cu.to(torch.int32), torch.cat((zero, kv.cumsum(0))).to(torch.int32), kv.to(torch.int32),
            torch.where(real, position, -1).to(torch.int32), slots, first[-1:].to(torch.int32), table)


_PLAIN = {"prompt": _plain_prompt, "prompt_bwd": _plain_prompt_bwd, "tree": _plain_tree,
          "tables": _plain_tables}


# ------------------------------------------------------------------------------------ its work

def work(case):
    kind = case["kind"]
    new, old = _lens(case)
    if kind == "tables":
        page = case["page"]
        idx = 4 if case["idx"] == "i32" else 8
        pages = sum(-(-(n + c) // page) - -(-c // page) for n, c in zip(new, old))
        return {"bytes": case["B"] * (2 * idx + 12) + 8 * pages + 12 * (sum(new) + case["spare"]),
                "flops": 0}
    Hq, H, D = case["Hq"], case["H"], case["D"]
    if kind == "tree":
        B, S, P = case["B"], case["S"], case["prefix"]
        row = H * (D + (4 if case["scale"] == "f32" else 1))
        # A draft sees some of the others: what a chain of them would see, at most.
        seen = sum((n - S) * S + S * (S + 1) // 2 for n in new) + B * S * P
        return {"bytes": 2 * (sum(new) + P) * row + 4 * B * S * Hq * D + B * S * S + 4 * B,
                "flops": 4 * seen * Hq * D}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(new, old))
    q, kv = 2 * sum(new) * Hq * D, 2 * (sum(new) + sum(old)) * H * D
    lse = 4 * sum(new) * Hq
    if kind == "prompt":
        return {"bytes": 2 * q + 2 * kv + (lse if case["lse"] else 0), "flops": 4 * pairs * Hq * D}
    return {"bytes": 4 * q + 4 * kv + lse, "flops": 10 * pairs * Hq * D}


# ------------------------------------------------------------------------------------ in 64 bits

def _exact_prompt(st):
    """Head by head, softmax of the scores plus the mask."""
    case = st["case"]
    group = case["Hq"] // case["H"]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEV)
    sums = torch.zeros(st["q"].shape[1], st["q"].shape[0], dtype=torch.float64, device=DEV)
    at = at_k = 0
    for n, m in zip(st["new"], st["both"]):
        mask = torch.full((n, m), float("-inf"), dtype=torch.float64, device=DEV).triu(m - n + 1)
        for h in range(case["Hq"] if n else 0):
            k, v = (st[x][at_k:at_k + m, h // group].double() for x in ("k", "v"))
            x = torch.addmm(mask, st["q"][at:at + n, h].double(), k.t(), alpha=1 / math.sqrt(case["D"]))
            sums[h, at:at + n] = torch.logsumexp(x, -1)
            out[at:at + n, h] = torch.softmax(x, -1) @ v
        at, at_k = at + n, at_k + m
    return (out, sums) if case["lse"] else out


def _exact_prompt_bwd(st):
    """Head by head, the products that the formulas of the gradients have."""
    case = st["case"]
    group, scale = case["Hq"] // case["H"], 1 / math.sqrt(case["D"])
    grads = [torch.zeros(st[x].shape, dtype=torch.float64, device=DEV) for x in ("q", "k", "v")]
    at = at_k = 0
    for n, m in zip(st["new"], st["both"]):
        seen = torch.ones(n, m, dtype=torch.float64, device=DEV).tril(m - n)
        rows, keys = slice(at, at + n), slice(at_k, at_k + m)
        for h in range(case["Hq"] if n else 0):
            q, do, o = (st[x][rows, h].double() for x in ("q", "dout", "out"))
            k, v = (st[x][keys, h // group].double() for x in ("k", "v"))
            p = torch.exp((q @ k.t()) * scale * seen - st["lse"][h, rows, None].double()) * seen
            grads[2][keys, h // group] += p.t() @ do
            t = p * (do @ v.t() - (do * o).sum(1)[:, None]) * scale
            grads[0][rows, h] = t @ k
            grads[1][keys, h // group] += t.t() @ q
        at, at_k = at + n, at_k + m
    return tuple(grads)


def _sequence(st, n, pages, count):
    """The first `count` rows [H, count, D] of a list of pages, in 64 bits."""
    stored = st[n + "_scale"][pages].double()
    s = torch.exp2(stored - 127.0) if st["case"]["scale"] == "ue8m0" else stored
    codes = st[n + "_cache"].view(torch.int8)[pages].view(st[n + "_cache"].dtype).float().double()
    return (codes * s.transpose(2, 3)).transpose(0, 1).flatten(1, 2)[:, :count]


def _exact_tree(st):
    case = st["case"]
    B, S, Hq, H, D, P, page = (case[n] for n in ("B", "S", "Hq", "H", "D", "prefix", "page"))
    lens, _ = _lens(case)
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64, device=DEV)
    for b, c in enumerate(lens):
        pages = st["page_table"][b, :-(-c // page)].long()
        k, v = (_sequence(st, n, pages, c) for n in ("k", "v"))
        if P:
            k, v = (torch.cat((_sequence(st, n, st["prefix_pages"].long(), P), x), 1)
                    for n, x in (("k", k), ("v", v)))
        mask = torch.zeros(S, P + c, dtype=torch.float64, device=DEV)
        mask[:, P + c - S:].masked_fill_(~st["tree_mask"][b], float("-inf"))
        for h in range(Hq):
            x = torch.addmm(mask, st["q"][b, :, h].double(), k[h // (Hq // H)].t(),
                            alpha=1 / math.sqrt(D))
            out[b, :, h] = torch.softmax(x, -1) @ v[h // (Hq // H)]
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "tables":
        return None                                # whole numbers
    return {"prompt": _exact_prompt, "prompt_bwd": _exact_prompt_bwd, "tree": _exact_tree}[kind](
        prepare(case, seed))
