"""The attention side where offsets pass 32 bits (caches and strided views of more than 4 GiB) and on
the largest pages: the same rows in small tensors give the same bits."""
import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note
from tests.test_gpu_paged_attention import FP8, INT8, check, make

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def room(gpu, gib):
    if torch.cuda.mem_get_info(gpu)[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB")


def wide(rows, width, start, x):
    """x [rows, H, D] as a view of rows of `width` elements, from element `start` of each on."""
    buf = torch.empty(rows, width, dtype=x.dtype, device=x.device)
    v = buf[:, start:start + x.shape[1] * x.shape[2]].view(x.shape)
    v.copy_(x)
    return v


@pytest.mark.parametrize("S,group", [(1, 4), (24, 8)])
def test_cache_of_more_than_4_gib(pkg, gpu, S, group):
    """Pages at both ends of a cache of 4.6 GB of keys and as many of values."""
    note(f"attention over a cache of more than 4 GiB, S {S}")
    room(gpu, 16)
    H, D, page, B, many = 8, 128, 64, 3, 70000
    lens = torch.tensor([150, 64, 31], dtype=torch.int32, device=gpu)
    g = torch.Generator().manual_seed(S)
    k, v = (torch.randn(256, H, D, generator=g).to(BF16).to(gpu) for _ in range(2))
    q = torch.randn(B, S, H * group, D, generator=g).to(BF16).to(gpu)
    small = torch.tensor([[0, 1, 2], [3, -1, -1], [0, -1, -1]], dtype=torch.int32, device=gpu)
    at = torch.tensor([many - 1, 3, many - 2, many - 3], dtype=torch.int32, device=gpu)
    results = []
    for pages, table, where in ((4, small, torch.arange(4, device=gpu)),
                                (many, torch.where(small >= 0, at[small.clamp_min(0).long()], small), at.long())):
        kc, ks = pkg.empty_kv_cache(pages, H, page, D, device=gpu)
        vc, vs = pkg.empty_kv_cache(pages, H, page, D, device=gpu)
        slots = (where[:, None] * page + torch.arange(page, device=gpu)).reshape(-1)
        pkg.kv_cache_write(k, v, slots, kc, vc, ks, vs)
        for most in (192, 1 << 22):      # rows on few keys, and as many as tall units take
            t = torch.full((B, most // page), -1, dtype=torch.int32, device=gpu)
            t[:, :3] = table
            results.append(pkg.paged_attention(q, kc, vc, ks, vs, t, lens, D ** -0.5))
        prefix = table[0].contiguous()
        results.append(pkg.paged_attention(q, kc, vc, ks, vs, t, torch.zeros_like(lens), D ** -0.5,
                                           prefix_pages=prefix, prefix_len=150))
        del kc, ks, vc, vs
    assert all(torch.isfinite(r).all() for r in results)
    for a, b in zip(results[:3], results[3:]):
        assert torch.equal(a, b)
    torch.cuda.empty_cache()


def test_views_of_more_than_4_gib(pkg, gpu):
    note("norm, rotation, write and attention on views of more than 4 GiB")
    room(gpu, 40)
    T, H, D, width = 20000, 3, 64, 131072
    g = torch.Generator().manual_seed(7)
    x, y, dx, dy = (torch.randn(T, H, D, generator=g).to(BF16).to(gpu) for _ in range(4))
    w = torch.ones(D, dtype=BF16, device=gpu)
    cos, sin = (t.to(gpu) for t in ref.tables(T, D))
    pos = torch.arange(T, device=gpu)
    plain = pkg.qk_norm_rope(x, y, w, w, cos, sin, pos)
    grads = pkg.qk_norm_rope_bwd(dx, dy, x, y, w, w, cos, sin, pos)
    cache = [pkg.empty_kv_cache(1300, H, 16, D, device=gpu) for _ in range(4)]
    (kc, ks), (vc, vs), (kc2, ks2), (vc2, vs2) = cache
    for t in (t for c in cache for t in c):
        t.view(torch.uint8).zero_()
    pkg.kv_cache_write(x, y, pos, kc, vc, ks, vs)
    table = torch.arange(1280, dtype=torch.int32, device=gpu).view(64, 20).contiguous()
    lens = torch.full((64,), 300, dtype=torch.int32, device=gpu)
    o = pkg.paged_attention(x[:64 * 312].view(64, 312, H, D)[:, :40], kc, vc, ks, vs, table, lens, D ** -0.5)

    far = wide(T, width, width - H * D, x)               # 5.2 GB
    assert (T - 1) * far.stride(0) > 1 << 31
    out = wide(T, width, 640, torch.zeros_like(x))
    q2, k2 = pkg.qk_norm_rope(far, y, w, w, cos, sin, pos, q_out=out)
    assert torch.equal(q2, plain[0]) and torch.equal(k2, plain[1])
    got = pkg.qk_norm_rope_bwd(dx, dy, far, y, w, w, cos, sin, pos, dq=out)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    pkg.kv_cache_write(far, y, pos, kc2, vc2, ks2, vs2)
    for a, b in zip((kc, ks, vc, vs), (kc2, ks2, vc2, vs2)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    q = far[:64 * 312].view(64, 312, H, D)[:, :40]
    assert torch.equal(pkg.paged_attention(q, kc, vc, ks, vs, table, lens, D ** -0.5), o)
    del far, out, q, q2
    torch.cuda.empty_cache()


@pytest.mark.parametrize("page", [4096, 65536])
def test_large_pages(pkg, gpu, page):
    note(f"attention on pages of {page}")
    check(pkg, gpu, make(page, [page + 70, 5, 0], 1, 4, 1, 64, page, 20, INT8, True, BF16, spare=0), 20)
    check(pkg, gpu, make(page, [90, 300], 90, 2, 1, 128, page, 0, FP8, False, BF16, spare=0))


@pytest.mark.parametrize("B", [3, 700])
@pytest.mark.parametrize("prefix", [0, 37])
def test_no_own_keys_at_all(pkg, gpu, B, prefix):
    """A bound of zero, and a table without pages: what the prefix alone gives."""
    note(f"attention without own keys, {B} sequences, prefix {prefix}")
    made = make(B, [9] * B, 1, 8, 8, 64, 16, prefix)
    o = check(pkg, gpu, made, prefix, most=0)
    q, caches, table, lens, pp = made
    bare = (q, caches, torch.empty(B, 0, dtype=torch.int32), lens, pp)
    assert torch.equal(check(pkg, gpu, bare, prefix), o)
    if not prefix:
        assert not o.any()
