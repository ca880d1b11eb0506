"""Prompts, draft trees and step tables through the CPython binding and through the Python path: the
same outputs (bits, types, strides, identities), the same errors for the same calls."""
import pytest
import torch

from tests.gpu_util import note
from tests.test_gpu_binding_ops import both, same
from tests.test_gpu_paged_attention import make as make_paged
from tests.test_gpu_prompt_attention import make

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_prompts(pkg, gpu, monkeypatch):
    q, k, v, do, cu, _ = [None if t is None else t.to(gpu) for t in make(1, [40, 3, 90], None, 4, 2, 64, spare=3)]
    cu_k = torch.tensor([0, 10, 50, 136], dtype=torch.int32, device=gpu)
    given = torch.zeros_like(q)
    a = dict(q=q, k=k, v=v, cu_seqlens=cu, sm_scale=0.125)
    for kw in ({}, dict(return_lse=True), dict(cu_seqlens_k=cu_k, return_lse=True), dict(out=given), dict(sm_scale=1),
               dict(q=torch.cat((q, q), 1)[:, ::2]), dict(q=q[:0], k=k[:0], v=v[:0]), dict(k=k[:0], v=v[:0], cu_seqlens_k=cu_k * 0),
               # refused
               dict(cu_seqlens_k=cu), dict(q=q.float()), dict(k=k[:-1]), dict(out=q), dict(out=given[:-1]), dict(v=v.half()),
               dict(cu_seqlens=cu.long()), dict(cu_seqlens_k=cu[:2]), dict(sm_scale=float("inf")), dict(q=q[:, :3]),
               dict(q=q[..., :32]), dict(k=None)):
        note(f"binding prompt {sorted(kw)}")
        x, y = both(monkeypatch, lambda: pkg.prompt_attention(**{**a, **kw}))
        same(x, y)
    out, lse = pkg.prompt_attention(**a, return_lse=True)
    a.update(dout=do, out=out, lse=lse)
    fused = torch.zeros(q.shape[0], 8, 64, dtype=BF16, device=gpu)
    for kw in ({}, dict(dout=do[:1, :1].expand(q.shape)), dict(dq=fused[:, :4], dk=fused[:, 4:6], dv=fused[:, 6:]),
               dict(cu_seqlens_k=cu_k), dict(dk=torch.zeros_like(k)),
               dict(dq=q), dict(dk=fused[:, 3:5], dq=fused[:, :4]), dict(lse=lse[:3]), dict(dout=do.half()), dict(out=do[:-1]),
               dict(dv=v.half()), dict(dq=fused)):
        note(f"binding prompt_bwd {sorted(kw)}")
        x, y = both(monkeypatch, lambda: pkg.prompt_attention_bwd(**{**a, **kw}))
        same(x, y)


def test_trees(pkg, gpu, monkeypatch):
    q, caches, table, lens, pp = make_paged(3, [70, 3, 0], 4, 8, 2, 64, 16, 40)
    (kc, ks), (vc, vs) = [(c.to(gpu), s.to(gpu)) for c, s in caches]
    mask = torch.ones(3, 4, 4, dtype=torch.bool, device=gpu).tril()
    a = dict(q=q.to(gpu), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, page_table=table.to(gpu),
             kv_lens=lens.to(gpu), tree_mask=mask, sm_scale=0.125)
    P = dict(prefix_pages=pp.to(gpu), prefix_len=40)
    for kw in ({}, P, dict(tree_mask=mask[0].contiguous()), dict(tree_mask=mask.to(torch.uint8)), dict(max_kv_len=50),
               dict(out=torch.empty_like(a["q"])), dict(kv_lens=a["kv_lens"].long()), dict(q=a["q"][:, :, ::2]),
               dict(tree_mask=None), dict(tree_mask=mask[:2]), dict(tree_mask=mask.int()), dict(tree_mask=mask.cpu()),
               dict(prefix_len=3), dict(q=a["q"].float()), dict(out=a["q"]), dict(v_cache=None), dict(sm_scale=float("nan"))):
        note(f"binding tree {sorted(kw)}")
        same(*both(monkeypatch, lambda: pkg.paged_tree_attention(**{**a, **kw})))


def test_tables(pkg, gpu, monkeypatch):
    i32 = dict(dtype=torch.int32, device=gpu)
    a = dict(context_lens=torch.tensor([3, 0, 40], **i32), new_lens=torch.tensor([20, 5, 1], **i32),
             free_pages=torch.arange(7, 20, **i32), page_size=16, num_tokens=30)
    for kw in ({}, dict(num_tokens=0), dict(free_start=torch.ones(1, **i32)), dict(free_pages=torch.zeros(0, **i32)),
               dict(context_lens=torch.zeros(3, dtype=torch.int64, device=gpu)), dict(page_size=24), dict(page_size=16.0),
               dict(num_tokens=-1), dict(num_tokens=1 << 31), dict(new_lens=torch.zeros(2, **i32)), dict(free_start=torch.ones(2, **i32)),
               dict(free_start=3), dict(context_lens=None)):
        def call():
            table = torch.full((3, 4), -1, **i32)
            out = list(pkg.batch_tables(page_table=table, **{**a, **kw}))
            assert out[4].dtype == torch.int64
            out[4] = out[4].view(torch.int32)              # `same` looks at elements of up to 4 bytes
            return (*out, table)
        note(f"binding tables {sorted(kw)}")
        same(*both(monkeypatch, call))
    out = pkg.batch_tables(page_table=torch.full((3, 4), -1, **i32), **a)
    assert all(t.is_contiguous() and t.data_ptr() % 16 == 0 for t in out)
    keep = [t.clone() for t in out]
    out[3].fill_(77)                                       # outputs do not overlap
    assert all(torch.equal(x, y) for j, (x, y) in enumerate(zip(out, keep)) if j != 3)
