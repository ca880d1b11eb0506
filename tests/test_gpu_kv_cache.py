"""kv_cache_write and kv_cache_read on the GPU: codes, scales and gathered values bit for bit
against the same fp32 steps on the CPU (tests/attention_ref.py), and what they must leave alone."""
import random

import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
FP8, INT8 = torch.float8_e4m3fn, torch.int8


def same(a, b):
    a, b = (t.cpu().contiguous().reshape(-1).view(torch.uint8) for t in (a, b))
    return torch.equal(a, b)


def filled(pkg, P, H, page, D, G, qdt, ue8m0, value=0x5A):
    c, s = pkg.empty_kv_cache(P, H, page, D, G, qdt, ue8m0, device="cpu")
    c.view(torch.uint8).fill_(value)
    s.view(torch.uint8).fill_(value)
    return c, s


def place(cache, scale, codes, scales, slots):
    """The CPU's copy of a write: codes [T, H, D], scales [T, H, groups]."""
    P, H, page, D = cache.shape
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < P * page:
            cache.view(torch.uint8)[s // page, :, s % page] = codes.view(torch.uint8)[t]
            scale[s // page, :, :, s % page] = scales[t]


WRITE = [
    # T, H, D, G, page, pages
    (1, 1, 64, 64, 16, 1), (5, 8, 128, 128, 16, 3), (3, 2, 192, 64, 64, 2), (70, 3, 256, 256, 32, 4),
    (17, 1, 512, 128, 64, 2), (33, 12, 128, 64, 128, 1), (9, 5, 320, 64, 16, 2),
    (2, 1, 1024, 256, 256, 1),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("qdt,ue8m0", [(FP8, False), (FP8, True), (INT8, False), (INT8, True)])
@pytest.mark.parametrize("case", WRITE, ids=str)
def test_write(pkg, gpu, case, dtype, qdt, ue8m0):
    T, H, D, G, page, P = case
    note(f"write {case} {dtype} {qdt} ue8m0={ue8m0}")
    g = torch.Generator().manual_seed(T * D)
    x = torch.randn(2, T, H, D, generator=g) * torch.exp(torch.randn(2, T, H, 1, generator=g) * 3)
    x[0, 0, 0, :G] = 0.0                                   # a group of zeros: the floor scale
    x = x.to(dtype)
    slots = torch.randperm(P * page, generator=g)[:T]
    slots[T // 2] = -1 if T > 1 else slots[0]
    if T > 3:
        slots[1] = P * page
    host = [filled(pkg, P, H, page, D, G, qdt, ue8m0) for _ in range(2)]
    dev = [(c.to(gpu), s.to(gpu)) for c, s in host]
    d = x.to(gpu)
    pkg.kv_cache_write(d[0], d[1], slots.to(gpu), dev[0][0], dev[1][0], dev[0][1], dev[1][1])
    for i in range(2):
        place(*host[i], *ref.quantize(x[i], G, qdt, ue8m0), slots)
        assert same(dev[i][0], host[i][0]) and same(dev[i][1], host[i][1])


def test_write_views_latents_and_int32_slots(pkg, gpu):
    T, H, D, page, P = 21, 4, 128, 32, 2
    note("write views")
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(T, 3 * H, D, generator=g).bfloat16()
    slots = torch.randperm(P * page, generator=g)[:T].int()
    d = qkv.to(gpu)
    host = [filled(pkg, P, H, page, D, 128, FP8, False) for _ in range(2)]
    dev = [(c.to(gpu), s.to(gpu)) for c, s in host]
    vt = d[:, 2 * H:].transpose(0, 1).contiguous().transpose(0, 1)      # heads first
    pkg.kv_cache_write(d[:, H:2 * H], vt, slots.to(gpu), dev[0][0], dev[1][0], dev[0][1], dev[1][1])
    for i in range(2):
        place(*host[i], *ref.quantize(qkv[:, (1 + i) * H:(2 + i) * H], 128, FP8, False), slots)
        assert same(dev[i][0], host[i][0]) and same(dev[i][1], host[i][1])
    lat, (hc, hs) = qkv[:, :1].repeat(1, 1, 4), filled(pkg, P, 1, page, 512, 64, FP8, True)
    dc, ds = hc.to(gpu), hs.to(gpu)
    pkg.kv_cache_write(lat.to(gpu), None, slots.to(gpu), dc, None, ds, None)
    place(hc, hs, *ref.quantize(lat, 64, FP8, True), slots)
    assert same(dc, hc) and same(ds, hs)


def test_a_row_that_is_not_finite_stays_in_its_row(pkg, gpu):
    """Infinities and NaN spoil their own group, no other."""
    T, H, D, page = 6, 2, 128, 16
    note("write not finite")
    x = torch.randn(T, H, D, generator=torch.Generator().manual_seed(9)).bfloat16()
    x[2, 1, 5], x[4, 0, 77] = float("inf"), float("nan")
    host = filled(pkg, 1, H, page, D, 64, FP8, False)
    c, s = host[0].to(gpu), host[1].to(gpu)
    slots = torch.arange(T)
    pkg.kv_cache_write(x.to(gpu), None, slots.to(gpu), c, None, s, None)
    place(*host, *ref.quantize(torch.nan_to_num(x, 0.0, 0.0, 0.0), 64, FP8, False), slots)
    c, s = c.cpu(), s.cpu()
    for t in range(T):
        for h in range(H):
            for grp in range(2):
                if (t, h, grp) in ((2, 1, 0), (4, 0, 1)):
                    continue
                cut = slice(64 * grp, 64 * grp + 64)
                assert same(c[0, h, t, cut], host[0][0, h, t, cut])
                assert same(s[0, h, grp, t], host[1][0, h, grp, t])


def random_cache(pkg, g, P, H, page, D, G, qdt, ue8m0):
    x = torch.randn(P, H, page, D, generator=g) * torch.exp(torch.randn(P, H, page, 1, generator=g))
    codes, scales = ref.quantize(x, G, qdt, ue8m0)
    return codes, scales.transpose(2, 3).contiguous()


READ = [
    # lens, H, D, G, page
    ([1], 1, 64, 64, 16), ([0, 5, 0, 17], 8, 128, 128, 16), ([33, 1, 64], 3, 192, 64, 32),
    ([100, 0], 2, 256, 128, 64), ([40], 1, 512, 256, 16), ([16, 32, 15, 17], 12, 128, 64, 16),
    ([700, 1, 1500], 2, 64, 64, 128), ([3] * 70, 1, 1024, 256, 16),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("qdt,ue8m0", [(FP8, False), (FP8, True), (INT8, False), (INT8, True)])
@pytest.mark.parametrize("case", READ, ids=lambda c: f"{len(c[0])}x{max(c[0])}_{c[1:]}")
def test_read(pkg, gpu, case, dtype, qdt, ue8m0):
    lens, H, D, G, page = case
    note(f"read {case} {dtype} {qdt} ue8m0={ue8m0}")
    rng, g = random.Random(len(lens) * D), torch.Generator().manual_seed(D)
    need = [-(-n // page) for n in lens]
    P, width = sum(need) + 2, max(need) + 1
    order = rng.sample(range(P), P)
    table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    caches = [random_cache(pkg, g, P, H, page, D, G, qdt, ue8m0) for _ in range(2)]
    cu = torch.tensor([0] + lens).cumsum(0).int()
    total, extra = sum(lens), 3                           # rows behind the last stay as they were
    outs = [torch.full((total + extra, H, D), 5.0, dtype=dtype, device=gpu) for _ in range(2)]
    (kc, ks), (vc, vs) = [(c.to(gpu), s.to(gpu)) for c, s in caches]
    got = pkg.kv_cache_read(kc, vc, ks, vs, table.to(gpu), cu.to(gpu), *outs)
    assert got[0] is outs[0] and got[1] is outs[1]
    for (c, s), o in zip(caches, outs):
        values = ref.dequantize(c, s)
        want = torch.cat([ref.token_rows(values, table[b].tolist(), n, P)[0]
                          for b, n in enumerate(lens)]).to(dtype)
        assert same(o[:total], want) and bool((o[total:] == 5.0).all())


@pytest.mark.parametrize("bad", [-1, -7, 9, 2 ** 31 - 1])
def test_read_without_a_page_is_zeros(pkg, gpu, bad):
    note(f"read bad page {bad}")
    g = torch.Generator().manual_seed(1)
    c, s = random_cache(pkg, g, 9, 2, 16, 64, 64, FP8, False)
    table = torch.tensor([[3, bad, 4], [bad, 1, bad]], dtype=torch.int32)
    cu = torch.tensor([0, 48, 70], dtype=torch.int32)      # the second passes the first page only
    out = torch.full((70, 2, 64), 5.0, dtype=BF16, device=gpu)
    pkg.kv_cache_read(c.to(gpu), None, s.to(gpu), None, table.to(gpu), cu.to(gpu), out, None)
    v = ref.dequantize(c, s).bfloat16()
    want = torch.zeros(70, 2, 64, dtype=BF16)
    want[:16], want[32:48] = v[3].transpose(0, 1), v[4].transpose(0, 1)
    want[64:70] = v[1].transpose(0, 1)[:6]
    assert same(out, want)


def test_pages_past_32_bits(pkg, gpu):
    """Codes of a cache of more than 2^32 bytes: the last page's are found."""
    page, H, D = 256, 8, 256
    P = (1 << 32) // (page * H * D) + 2
    note(f"cache of {P * page * H * D} bytes")
    c, s = pkg.empty_kv_cache(P, H, page, D, device=gpu)
    x = torch.randn(3, H, D, generator=torch.Generator().manual_seed(3)).bfloat16()
    slots = torch.tensor([P * page - 1, P * page - 7, 2])
    pkg.kv_cache_write(x.to(gpu), None, slots.to(gpu), c, None, s, None)
    codes, scales = ref.quantize(x, 256, FP8, False)
    for t, slot in enumerate(slots.tolist()):
        assert same(c[slot // page, :, slot % page], codes[t])
        assert same(s[slot // page, :, :, slot % page], scales[t])
    out = torch.empty(256, H, D, dtype=BF16, device=gpu)
    pkg.kv_cache_read(c, None, s, None, torch.tensor([[P - 1]], dtype=torch.int32, device=gpu),
                      torch.tensor([0, 256], dtype=torch.int32, device=gpu), out, None)
    v = (codes.float().double() * scales.double()).float().bfloat16()
    assert same(out[255], v[0]) and same(out[249], v[1])


def test_empty_calls(pkg, gpu):
    c, s = pkg.empty_kv_cache(2, 2, 16, 64, device=gpu)
    c.view(torch.uint8).fill_(1)
    none = torch.empty(0, 2, 64, dtype=BF16, device=gpu)
    pkg.kv_cache_write(none, None, torch.empty(0, dtype=torch.int64, device=gpu), c, None, s, None)
    assert bool((c.view(torch.uint8) == 1).all())
    t0 = torch.empty(0, 1, dtype=torch.int32, device=gpu)
    cu = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert pkg.kv_cache_read(c, None, s, None, t0, cu, none, None)[0] is none
    out = torch.full((2, 2, 64), 5.0, dtype=BF16, device=gpu)
    pkg.kv_cache_read(c, None, s, None, t0, cu, out, None)
    assert bool((out == 5.0).all())


def test_refusals(pkg, gpu):
    c, s = pkg.empty_kv_cache(2, 2, 16, 64, device=gpu)
    x = torch.zeros(3, 2, 64, dtype=BF16, device=gpu)
    sl = torch.arange(3, device=gpu)
    ok = dict(k=x, v=None, slots=sl, k_cache=c, v_cache=None, k_scale=s, v_scale=None)
    for bad in (dict(k=x[:, :1]), dict(slots=sl[:2]), dict(slots=sl.cpu()), dict(k=x.cpu()),
                dict(v=x), dict(v_cache=c), dict(v_scale=s), dict(k_scale=s[:1]),
                dict(k_cache=c.transpose(1, 2)), dict(k_scale=s.expand(2, 2, 3, 16)),
                dict(k=x.transpose(0, 2))):
        with pytest.raises(ValueError):
            pkg.kv_cache_write(**{**ok, **bad})
    for bad in (dict(k=x.double()), dict(slots=sl.float())):
        with pytest.raises(TypeError):
            pkg.kv_cache_write(**{**ok, **bad})
    for page in (8, 24):
        cc, ss = pkg.empty_kv_cache(2, 2, page, 64, device=gpu)
        with pytest.raises(ValueError):
            pkg.kv_cache_write(**{**ok, "k_cache": cc, "k_scale": ss})
    t, cu = torch.zeros(1, 1, dtype=torch.int32, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    ok = dict(k_cache=c, v_cache=None, k_scale=s, v_scale=None, page_table=t, cu_seqlens=cu, k_out=x,
              v_out=None)
    for bad in (dict(k_out=x[:, :1]), dict(page_table=t.long()), dict(cu_seqlens=cu[:1]),
                dict(v_out=x), dict(k_out=x.transpose(0, 1)), dict(page_table=t.cpu())):
        with pytest.raises(ValueError):
            pkg.kv_cache_read(**{**ok, **bad})


@pytest.mark.parametrize("pages,width", [(0, 2), (3, 0), (0, 0)])
def test_read_without_pages_or_table(pkg, gpu, pages, width):
    """All tokens are without a page then: zeros, and the rows behind the last sequence stay."""
    note(f"read of {pages} pages, table of {width}")
    (kc, ks), (vc, vs) = (pkg.empty_kv_cache(pages, 2, 16, 64, device=gpu) for _ in range(2))
    table = torch.zeros(3, width, dtype=torch.int32, device=gpu)
    cu = torch.tensor([0, 5, 5, 9], dtype=torch.int32, device=gpu)
    outs = [torch.full((11, 2, 64), 5.0, dtype=BF16, device=gpu) for _ in range(2)]
    got = pkg.kv_cache_read(kc, vc, ks, vs, table, cu, *outs)
    assert got[0] is outs[0] and got[1] is outs[1]
    for o in outs:
        assert bool((o[:9] == 0).all()) and bool((o[9:] == 5.0).all())
    alone = torch.full((11, 2, 64), 5.0, dtype=BF16, device=gpu)
    pkg.kv_cache_read(kc, None, ks, None, table, cu, alone, None)
    assert torch.equal(alone, outs[0])
