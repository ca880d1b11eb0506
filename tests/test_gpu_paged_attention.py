"""paged_attention on the GPU against the softmax in 64 bits (tests/attention_ref.py has it and
the bounds): lengths from none to some thousand, pages in any order, causal newest tokens, shared
prefixes, every type, and slots that hold NaN and must not be seen."""
import random

import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
FP8, INT8 = torch.float8_e4m3fn, torch.int8


def make(seed, lens, S, Hq, H, D, page, prefix=0, qdt=FP8, ue8m0=False, dtype=BF16, spare=2,
         sharp=2.0):
    """Inputs on the CPU; every slot that no sequence holds is poisoned."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    need = [-(-n // page) for n in lens] + [-(-prefix // page)]
    P, width = sum(need) + spare, max(need[:-1] + [1]) + 1
    order, at = rng.sample(range(P), P), 0
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    live = torch.zeros(P, page, dtype=torch.bool)
    pages = []
    for n, count in zip(list(lens) + [prefix], need):
        mine = order[at:at + count]
        at += count
        pages.append(mine)
        for i, p in enumerate(mine):
            live[p, :max(0, min(page, n - i * page))] = True
    for b in range(len(lens)):
        table[b, :need[b]] = torch.tensor(pages[b], dtype=torch.int32)
    caches = []
    for _ in range(2):
        x = torch.randn(P, H, page, D, generator=g)
        x[..., :2] *= 4.0
        c, s = ref.quantize(x * torch.exp(0.5 * torch.randn(P, H, page, 1, generator=g)), D, qdt, ue8m0)
        s = s.transpose(2, 3).contiguous()
        dead = ~live[:, None, :].expand(P, H, page)
        c.view(torch.uint8)[dead] = 0x7F                   # e4m3fn's NaN
        s.transpose(2, 3)[dead] = 255 if ue8m0 else float("nan")
        caches.append((c, s))
    q = (sharp * torch.randn(len(lens), S, Hq, D, generator=g)).to(dtype)
    pp = torch.tensor(pages[-1], dtype=torch.int32) if prefix else None
    return q, caches, table, torch.tensor(lens, dtype=torch.int32), pp


def run(pkg, gpu, made, prefix=0, **kw):
    q, ((kc, ks), (vc, vs)), table, lens, pp = made
    D = q.shape[-1]
    return pkg.paged_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), ks.to(gpu), vs.to(gpu),
                               table.to(gpu), lens.to(gpu), D ** -0.5,
                               prefix_pages=None if pp is None else pp.to(gpu), prefix_len=prefix, **kw)


def clean(made):
    """The poisoned slots as zeros, for the 64-bit form."""
    out = []
    for c, s in made[1]:
        c, s = c.clone(), s.clone()
        bad = torch.isnan(ref.scale_value(s)) | torch.isinf(ref.scale_value(s))
        c.view(torch.uint8)[bad[:, :, 0]] = 0
        s[bad] = 0
        out.append((c, s))
    return out


def check(pkg, gpu, made, prefix=0, most=None, **kw):
    q, _, table, lens, pp = made
    o = run(pkg, gpu, made, prefix, max_kv_len=most, **kw)
    assert o.dtype == q.dtype and o.shape == q.shape and o.is_contiguous()
    (kc, ks), (vc, vs) = clean(made)
    r, bound = ref.attention(q, kc, vc, ks, vs, table, lens, q.shape[-1] ** -0.5, pp, prefix, most)
    assert ref.outside(o, r, bound, q.dtype) == 0
    return o


CASES = [
    # lens, S, Hq, H, D, page, prefix
    ([1], 1, 1, 1, 64, 16, 0), ([1, 0, 2], 1, 4, 2, 128, 16, 0), ([0, 0], 1, 2, 1, 64, 16, 0),
    ([15, 16, 17, 33], 1, 8, 8, 128, 16, 0), ([31, 32, 33, 65, 63], 1, 16, 4, 64, 32, 0),
    ([255, 257, 1], 1, 10, 2, 256, 64, 0), ([1000, 3, 517], 1, 32, 4, 128, 128, 0),
    ([2500], 1, 40, 1, 128, 16, 0), ([4097], 1, 5, 5, 64, 256, 0), ([70, 130], 1, 128, 1, 128, 64, 0),
    # several newest tokens, causal; lens shorter than them leave the first ones without keys
    ([5, 2, 64], 5, 4, 2, 128, 16, 0), ([40, 16, 0, 3], 16, 8, 8, 64, 32, 0),
    ([300, 129], 7, 24, 3, 256, 64, 0), ([200], 130, 4, 1, 128, 16, 0), ([90, 33], 33, 2, 2, 64, 16, 0),
    # a shared prefix
    ([1, 1, 1], 1, 4, 1, 128, 16, 1), ([0, 0, 0, 0], 1, 8, 2, 64, 16, 40), ([7, 0, 30], 1, 8, 2, 128, 32, 33),
    ([17] * 9, 1, 16, 2, 128, 16, 500), ([5, 40, 0, 2] * 8, 2, 10, 2, 64, 16, 129),
    ([3] * 70, 1, 8, 8, 128, 64, 1100), ([12, 80], 4, 16, 1, 256, 64, 200), ([20] * 40, 1, 64, 4, 128, 64, 700),
]


@pytest.mark.parametrize("qdt,ue8m0,dtype", [(FP8, False, BF16), (FP8, True, F16), (INT8, False, F16),
                                             (INT8, True, BF16)])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}_{'_'.join(map(str, c[1:]))}")
def test_attention(pkg, gpu, case, qdt, ue8m0, dtype):
    lens, S, Hq, H, D, page, prefix = case
    note(f"attention {case} {qdt} {ue8m0} {dtype}")
    check(pkg, gpu, make(len(lens) * 31 + D, lens, S, Hq, H, D, page, prefix, qdt, ue8m0, dtype), prefix)


@pytest.mark.parametrize("seed", range(24))
def test_random(pkg, gpu, seed):
    rng = random.Random(seed)
    H = rng.choice([1, 2, 3, 8])
    S = rng.choice([1, 1, 2, 3, 8, 20])
    page = rng.choice([16, 32, 64, 128])
    prefix = rng.choice([0, 0, rng.randint(1, 900)])
    lens = [rng.choice([0, rng.randint(0, 20), rng.randint(0, 700)]) for _ in range(rng.randint(1, 12))]
    D, Hq = rng.choice([64, 128, 256]), H * rng.choice([1, 2, 4, 5, 8, 16])
    qdt, ue8m0, dtype = rng.choice([FP8, INT8]), rng.random() < 0.5, rng.choice([BF16, F16])
    note(f"attention seed {seed}: {lens} S{S} {Hq}/{H} D{D} page {page} prefix {prefix} {qdt} {ue8m0} {dtype}")
    check(pkg, gpu, make(seed, lens, S, Hq, H, D, page, prefix, qdt, ue8m0, dtype), prefix)


def test_a_prefix_is_the_same_as_own_tokens(pkg, gpu):
    """The 64-bit form holds both; here the two ways to pass the same keys against each other
    (both lie within the bounds of the same reference)."""
    q, caches, table, lens, pp = make(5, [9, 9, 9], 1, 8, 2, 128, 16, 64)
    joined = torch.cat((pp[None].expand(3, -1), table), 1).contiguous()
    made = (q, caches, joined, lens + 64, None)
    check(pkg, gpu, made)
    check(pkg, gpu, (q, caches, table, lens, pp), 64)


@pytest.mark.parametrize("prefix", [0, 48])
def test_tokens_without_a_page_are_left_out(pkg, gpu, prefix):
    note(f"missing pages, prefix {prefix}")
    made = make(6, [100, 64, 33], 2, 8, 2, 128, 16, prefix)
    table = made[2]
    table[0, 2], table[0, 6], table[1, :4], table[2, 0] = -1, 2 ** 31 - 1, -5, -1
    if prefix:
        made[4][1] = -1
    check(pkg, gpu, made, prefix)


def test_lengths_past_the_table_and_the_bound(pkg, gpu):
    made = make(7, [60, 20, 33], 1, 4, 2, 64, 16)
    q, caches, table, lens, pp = made
    table = table[:, :2].contiguous()                     # room for 32 tokens
    note("cut by the table")
    check(pkg, gpu, (q, caches, table, lens, pp))
    note("cut by max_kv_len")
    check(pkg, gpu, made, most=30)
    check(pkg, gpu, made, most=60)
    check(pkg, gpu, (q, caches, table[:, :0].contiguous(), lens, pp))
    none = torch.full_like(lens, -2 ** 31)
    assert bool((run(pkg, gpu, (q, caches, table, none, pp)) == 0).all())


@pytest.mark.parametrize("S", [1, 5])
def test_lengths_of_any_value(pkg, gpu, S):
    note(f"attention with lengths of any value, S {S}")
    low, high = torch.iinfo(torch.int64).min, torch.iinfo(torch.int64).max
    made = make(12, [40] * 6, S, 4, 2, 64, 16)
    table = made[2][:, :3].contiguous()
    lens = torch.tensor([low, low + S, -1, high, high - S, 40], dtype=torch.int64)
    check(pkg, gpu, (made[0], made[1], table, lens, None), most=40)


def test_strided_queries_int64_lengths_and_a_given_output(pkg, gpu):
    made = make(8, [50, 3], 3, 6, 2, 128, 32)
    q, ((kc, ks), (vc, vs)), table, lens, _ = made
    args = [t.to(gpu) for t in (kc, vc, ks, vs, table)] + [lens.long().to(gpu), 128 ** -0.5]
    want = run(pkg, gpu, made)
    wide = torch.zeros(2, 3, 6 + 4, 128, dtype=BF16, device=gpu)
    wide[:, :, 2:8] = q.to(gpu)
    out = torch.full_like(want, 9.0)
    got = pkg.paged_attention(wide[:, :, 2:8], *args, out=out)
    assert got is out and torch.equal(got, want)
    heads_first = q.to(gpu).transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(pkg.paged_attention(heads_first, *args), want)
    one = q[:1, :1, :1].to(gpu).expand(2, 3, 6, 128)
    o = pkg.paged_attention(one, *args)
    for h in range(1, 3):
        assert torch.equal(o[:, :, h], o[:, :, 0])


@pytest.mark.parametrize("lens,S,prefix", [([700, 20, 0], 1, 0), ([300, 5], 4, 600), ([2000], 1, 0)])
def test_workspace(pkg, gpu, lens, S, prefix):
    """Nothing is written past the bytes a caller is told, and what they held does not matter."""
    from fagq_mi355x import kv_cache
    note(f"attention workspace {lens} {S} {prefix}")
    made = make(9, lens, S, 16, 2, 128, 16, prefix)
    need = kv_cache.attention_workspace_bytes(len(lens), S, 16, 2, 128, prefix, made[2].shape[1] * 16)
    want = run(pkg, gpu, made, prefix)
    for fill in (0, 0xFF):
        buf = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=gpu)
        buf[:need] = fill
        got = run(pkg, gpu, made, prefix, workspace=buf[:max(need, 16)])
        assert torch.equal(got, want) and bool((buf[max(need, 16):] == 0xA5).all())


@pytest.mark.parametrize("factor", [2.0 ** -40, 2.0 ** 30])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_scales_of_any_size(pkg, gpu, factor, dtype):
    """Value scales far from 1 move the result by the same factor (a power of two)."""
    note(f"value scales times {factor} {dtype}")
    q, ((kc, ks), (vc, vs)), table, lens, _ = make(10, [130, 40], 1, 8, 2, 64, 16, dtype=dtype)
    small = factor if dtype == BF16 else min(factor, 2.0 ** 4) if factor > 1 else 2.0 ** -8
    made = (q, ((kc, ks), (vc, vs * small)), table, lens, None)
    check(pkg, gpu, made)


@pytest.mark.parametrize("sharp", [0.0, 30.0])
def test_flat_and_sharp_softmax(pkg, gpu, sharp):
    note(f"sharpness {sharp}")
    check(pkg, gpu, make(11, [300, 17], 1, 8, 2, 128, 16, 100, sharp=sharp), 100)


def test_empty_batch_and_cache(pkg, gpu):
    kc, ks = pkg.empty_kv_cache(2, 2, 16, 64, device=gpu)
    q = torch.zeros(0, 1, 4, 64, dtype=BF16, device=gpu)
    t, lens = torch.zeros(0, 1, dtype=torch.int32, device=gpu), torch.zeros(0, dtype=torch.int32, device=gpu)
    assert pkg.paged_attention(q, kc, kc, ks, ks, t, lens, 0.1).shape == q.shape
    kc, ks = pkg.empty_kv_cache(0, 2, 16, 64, device=gpu)
    q = torch.ones(2, 1, 4, 64, dtype=BF16, device=gpu)
    t, lens = torch.zeros(2, 1, dtype=torch.int32, device=gpu), torch.ones(2, dtype=torch.int32, device=gpu)
    assert bool((pkg.paged_attention(q, kc, kc, ks, ks, t, lens, 0.1) == 0).all())


def test_refusals(pkg, gpu):
    kc, ks = pkg.empty_kv_cache(2, 2, 16, 64, device=gpu)
    q = torch.zeros(3, 1, 4, 64, dtype=BF16, device=gpu)
    t, lens = torch.zeros(3, 1, dtype=torch.int32, device=gpu), torch.ones(3, dtype=torch.int32, device=gpu)
    ok = dict(q=q, k_cache=kc, v_cache=kc, k_scale=ks, v_scale=ks, page_table=t, kv_lens=lens, sm_scale=0.1)
    wide = pkg.empty_kv_cache(2, 2, 16, 128, 64, device=gpu)
    for bad in (dict(q=q[:, :, :3]), dict(q=q[..., :32]), dict(page_table=t[:2]), dict(kv_lens=lens[:2]),
                dict(q=q.cpu()), dict(v_cache=None, v_scale=None), dict(prefix_len=5),
                dict(prefix_len=-1), dict(prefix_len=17, prefix_pages=t[:1, 0]),
                dict(prefix_len=5, prefix_pages=t[:, 0].long()), dict(out=q[:2]), dict(out=q.half()),
                dict(max_kv_len=-1), dict(kv_lens=lens.cpu()),
                dict(q=q.repeat(1, 1, 1, 2), k_cache=wide[0], v_cache=wide[0], k_scale=wide[1],
                     v_scale=wide[1])):
        with pytest.raises(ValueError):
            pkg.paged_attention(**{**ok, **bad})
    for bad in (dict(q=q.float()), dict(kv_lens=lens.float())):
        with pytest.raises(TypeError):
            pkg.paged_attention(**{**ok, **bad})
    for bad, status in ((dict(out=q), 9), (dict(sm_scale=float("nan")), 2)):
        with pytest.raises(pkg.FagqError) as e:
            pkg.paged_attention(**{**ok, **bad})
        assert e.value.status == status
