"""paged_tree_attention on the GPU against the softmax in 64 bits (tests/prompt_ref.py): trees, any
masks, sequences shorter than their drafts, shared prefixes, every type, poisoned slots."""
import random

import pytest
import torch

from tests import attention_ref, prompt_ref as ref
from tests.gpu_util import note
from tests.test_gpu_paged_attention import clean, make

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
FP8, INT8 = torch.float8_e4m3fn, torch.int8


def masks(seed, B, S, kind="tree"):
    g = torch.Generator().manual_seed(seed)
    if kind == "any":
        return torch.rand(B, S, S, generator=g) < 0.4
    if kind == "none":
        return torch.zeros(B, S, S, dtype=torch.bool)
    mask = torch.zeros(B, S, S, dtype=torch.bool)
    for b in range(B):
        for s in range(S):
            parent = s - int(torch.randint(1, 5, (1,), generator=g))
            if parent >= 0:
                mask[b, s] = mask[b, parent]
            mask[b, s, s] = True
    return mask


def run(pkg, gpu, made, mask, prefix=0, **kw):
    q, ((kc, ks), (vc, vs)), table, lens, pp = made
    return pkg.paged_tree_attention(q.to(gpu), kc.to(gpu), vc.to(gpu), ks.to(gpu), vs.to(gpu), table.to(gpu),
                                    lens.to(gpu), mask.to(gpu), q.shape[-1] ** -0.5,
                                    prefix_pages=None if pp is None else pp.to(gpu), prefix_len=prefix, **kw)


def check(pkg, gpu, made, mask, prefix=0, most=None):
    q, _, table, lens, pp = made
    o = run(pkg, gpu, made, mask, prefix, max_kv_len=most)
    assert o.dtype == q.dtype and o.shape == q.shape and o.is_contiguous()
    (kc, ks), (vc, vs) = clean(made)
    r, bound = ref.tree(q, kc, vc, ks, vs, table, lens, mask, q.shape[-1] ** -0.5, pp, prefix, most)
    assert attention_ref.outside(o, r, bound, q.dtype) == 0


CASES = [
    # lens, S, Hq, H, D, page, prefix
    ([1], 1, 1, 1, 64, 16, 0), ([2, 9], 2, 4, 2, 128, 16, 0), ([33, 40, 0, 5], 5, 8, 8, 64, 32, 0),
    ([100, 31, 64], 16, 8, 2, 128, 16, 0), ([63, 64, 65], 63, 4, 1, 64, 16, 0), ([300, 7], 33, 12, 3, 256, 64, 0),
    ([500], 65, 8, 1, 128, 128, 0), ([1500, 200], 24, 16, 2, 128, 16, 0), ([140, 129], 128, 4, 2, 64, 16, 0),
    ([10, 3, 16], 8, 8, 2, 128, 16, 40), ([0, 4], 4, 4, 2, 64, 32, 129), ([70] * 5, 40, 16, 2, 128, 64, 500),
    ([20] * 9, 9, 16, 1, 256, 16, 300), ([300], 130, 8, 1, 256, 64, 0), ([66] * 3, 64, 8, 2, 64, 16, 700),
]


@pytest.mark.parametrize("kind", ["tree", "any"])
@pytest.mark.parametrize("qdt,ue8m0,dtype", [(FP8, False, BF16), (INT8, True, F16), (FP8, True, F16)])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}_{'_'.join(map(str, c[1:]))}")
def test_trees(pkg, gpu, case, qdt, ue8m0, dtype, kind):
    lens, S, Hq, H, D, page, prefix = case
    note(f"tree {case} {qdt} {ue8m0} {dtype} {kind}")
    made = make(len(lens) * 37 + S, lens, S, Hq, H, D, page, prefix, qdt, ue8m0, dtype)
    check(pkg, gpu, made, masks(S, len(lens), S, kind), prefix)


def test_a_chain_is_the_causal_attention(pkg, gpu):
    """A chain's mask and paged_attention agree within the bounds of either against the causal formula.
    (Not bit for bit: a step that holds a key which some row does not see takes the key's scale into
    the score before the maximum is subtracted, others in the subtraction, and which steps these are
    differs.)"""
    note("chains")
    for lens, S, prefix in (([50, 3, 20], 8, 0), ([300, 129], 40, 0), ([9, 12], 4, 64)):
        made = make(5, lens, S, 8, 2, 128, 16, prefix)
        q, _, table, kv, pp = made
        chain = torch.ones(S, S, dtype=torch.bool).tril()
        got = run(pkg, gpu, made, chain, prefix)
        (kc, ks), (vc, vs) = clean(made)
        want, bound = attention_ref.attention(q, kc, vc, ks, vs, table, kv, 128 ** -0.5, pp, prefix)
        for b, n in enumerate(lens):
            rows = slice(max(0, S - n), S)               # drafts that exist
            assert attention_ref.outside(got[b, rows], want[b, rows], bound[b, rows], q.dtype) == 0
        assert torch.equal(run(pkg, gpu, made, chain.expand(len(lens), S, S).contiguous(), prefix), got)
        assert torch.equal(run(pkg, gpu, made, chain.to(torch.uint8) * 200, prefix), got)


@pytest.mark.parametrize("qdt,ue8m0,dtype", [(FP8, False, BF16), (INT8, False, F16), (FP8, True, F16)])
@pytest.mark.parametrize("case", [c for c in CASES if c[1] > 3], ids=lambda c: f"{len(c[0])}x{max(c[0])}_{'_'.join(map(str, c[1:]))}")
def test_drafts_that_nobody_sees_may_hold_anything(pkg, gpu, case, qdt, ue8m0, dtype):
    """A padded tree: some drafts are in no row of the mask, and their slots were never written."""
    lens, S, Hq, H, D, page, prefix = case
    note(f"unseen drafts {case} {qdt} {ue8m0} {dtype}")
    made = make(len(lens) * 41 + S, lens, S, Hq, H, D, page, prefix, qdt, ue8m0, dtype)
    q, caches, table, kv, pp = made
    mask = masks(S + 1, len(lens), S)
    dead = [t for t in range(S) if t % 3 == 1 or t >= S - 2]
    mask[:, :, dead] = False
    want = run(pkg, gpu, made, mask, prefix)
    worse = []
    for c, s in caches:
        c, s = c.clone(), s.clone()
        for b, n in enumerate(kv.tolist()):
            for t in dead:
                if n - S + t >= 0:
                    slot = n - S + t
                    at, off = int(table[b, slot // page]), slot % page
                    c.view(torch.uint8)[at, :, off] = 0x7F
                    s[at, :, :, off] = 255 if ue8m0 else float("nan") if t % 2 else float("inf")
        worse.append((c, s))
    got = run(pkg, gpu, (q, worse, table, kv, pp), mask, prefix)
    assert bool(torch.isfinite(got).all()) and torch.equal(got, want)
    check(pkg, gpu, made, mask, prefix)


def test_masks_that_leave_nothing(pkg, gpu):
    note("empty masks")
    made = make(6, [4, 12, 0], 4, 8, 2, 64, 16)
    mask = masks(1, 3, 4, "none")
    o = run(pkg, gpu, made, mask)
    assert bool((o[0] == 0).all()) and bool((o[2] == 0).all()) and not bool((o[1] == 0).any())
    check(pkg, gpu, made, mask)


@pytest.mark.parametrize("prefix", [0, 48])
def test_missing_pages_and_cut_lengths(pkg, gpu, prefix):
    note(f"missing pages, prefix {prefix}")
    made = make(7, [100, 64, 33], 6, 8, 2, 128, 16, prefix)
    table = made[2]
    table[0, 2], table[0, 6], table[1, :4], table[2, 0] = -1, 2 ** 31 - 1, -5, -1
    check(pkg, gpu, made, masks(2, 3, 6), prefix)
    check(pkg, gpu, made, masks(2, 3, 6), prefix, most=70)
    q, caches, table, lens, pp = made
    check(pkg, gpu, (q, caches, table[:, :3].contiguous(), lens, pp), masks(3, 3, 6, "any"), prefix)


def test_lengths_of_any_value(pkg, gpu):
    low, high = torch.iinfo(torch.int64).min, torch.iinfo(torch.int64).max
    note("lengths of any value")
    q, caches, table, _, _ = make(8, [40] * 5, 5, 4, 2, 64, 16)
    lens = torch.tensor([low, -1, high, 4, 40], dtype=torch.int64)
    check(pkg, gpu, (q, caches, table[:, :3].contiguous(), lens, None), masks(4, 5, 5), most=40)


@pytest.mark.parametrize("seed", range(12))
def test_random(pkg, gpu, seed):
    rng = random.Random(seed)
    H, S, page = rng.choice([1, 2, 3, 8]), rng.choice([2, 7, 16, 31, 70]), rng.choice([16, 32, 64])
    prefix = rng.choice([0, 0, rng.randint(1, 600)])
    lens = [rng.choice([rng.randint(0, S), S + rng.randint(0, 500)]) for _ in range(rng.randint(1, 8))]
    D, Hq = rng.choice([64, 128, 256]), H * rng.choice([1, 2, 5, 8])
    qdt, ue8m0, dtype = rng.choice([FP8, INT8]), rng.random() < 0.5, rng.choice([BF16, F16])
    note(f"tree seed {seed}: {lens} S{S} {Hq}/{H} D{D} page {page} prefix {prefix} {qdt} {ue8m0} {dtype}")
    check(pkg, gpu, make(seed, lens, S, Hq, H, D, page, prefix, qdt, ue8m0, dtype),
          masks(seed, len(lens), S, rng.choice(["tree", "any"])), prefix)


@pytest.mark.parametrize("lens,S,prefix", [([700, 20, 0], 16, 0), ([300, 5], 4, 600), ([2000], 40, 0)])
def test_workspace(pkg, gpu, lens, S, prefix):
    from fagq_mi355x import kv_cache
    note(f"tree workspace {lens} {S} {prefix}")
    made = make(9, lens, S, 16, 2, 128, 16, prefix)
    need = kv_cache.tree_attention_workspace_bytes(len(lens), S, 16, 2, 128, prefix, made[2].shape[1] * 16)
    mask = masks(5, len(lens), S)
    want = run(pkg, gpu, made, mask, prefix)
    for fill in (0, 0xFF):
        buf = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=gpu)
        buf[:need] = fill
        got = run(pkg, gpu, made, mask, prefix, workspace=buf[:max(need, 16)])
        assert torch.equal(got, want) and bool((buf[max(need, 16):] == 0xA5).all())


def test_refusals(pkg, gpu):
    kc, ks = pkg.empty_kv_cache(2, 2, 16, 64, device=gpu)
    q = torch.zeros(3, 4, 4, 64, dtype=BF16, device=gpu)
    t, lens = torch.zeros(3, 1, dtype=torch.int32, device=gpu), torch.ones(3, dtype=torch.int32, device=gpu)
    mask = torch.ones(3, 4, 4, dtype=torch.bool, device=gpu)
    ok = dict(q=q, k_cache=kc, v_cache=kc, k_scale=ks, v_scale=ks, page_table=t, kv_lens=lens, tree_mask=mask, sm_scale=0.1)
    for bad in (dict(tree_mask=mask[:2]), dict(tree_mask=mask[:, :3]), dict(tree_mask=mask.float()),
                dict(tree_mask=mask.cpu()), dict(tree_mask=mask.transpose(1, 2)), dict(tree_mask=mask[0, 0]),
                dict(q=q[:, :, :3]), dict(page_table=t[:2]), dict(max_kv_len=-1), dict(v_cache=None, v_scale=None)):
        with pytest.raises(ValueError):
            pkg.paged_tree_attention(**{**ok, **bad})
    for bad in (dict(tree_mask=None), dict(q=q.float())):
        with pytest.raises(TypeError):
            pkg.paged_tree_attention(**{**ok, **bad})
    wide = torch.zeros(1, 4097, 2, 64, dtype=BF16, device=gpu)
    with pytest.raises(ValueError):
        pkg.paged_tree_attention(**{**ok, "q": wide, "page_table": t[:1], "kv_lens": lens[:1],
                                    "tree_mask": torch.zeros(4097, 4097, dtype=torch.bool, device=gpu)})
    for bad, status in ((dict(out=q), 9), (dict(sm_scale=float("nan")), 2)):
        with pytest.raises(pkg.FagqError) as e:
            pkg.paged_tree_attention(**{**ok, **bad})
        assert e.value.status == status
