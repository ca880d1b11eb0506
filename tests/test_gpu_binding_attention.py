"""The attention side through the CPython binding and through the Python path: the same outputs
(bits, types, strides, identities), the same errors for the same calls."""
import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note
from tests.test_gpu_binding_ops import both, same
from tests.test_gpu_paged_attention import make

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rope_args(gpu, T=5, Hq=4, Hk=2, D=64, R=32, dtype=BF16, idx=torch.int64):
    g = torch.Generator().manual_seed(T + D)
    x = torch.randn(T, Hq + 2 * Hk, D, generator=g).to(dtype).to(gpu)
    w = torch.nn.Parameter(torch.ones(D, dtype=dtype, device=gpu))
    cos, sin = (t.to(gpu) for t in ref.tables(16, R))
    pos = torch.arange(T).to(idx).to(gpu)
    return dict(q=x[:, :Hq], k=x[:, Hq:Hq + Hk], q_weight=w, k_weight=w, cos=cos, sin=sin, positions=pos)


ROPE = [dict(), dict(T=1, Hq=1, Hk=1, D=128, R=128, dtype=F16), dict(D=80, R=80, dtype=F32, idx=torch.int32),
        dict(T=0), dict(D=72, R=16), dict(R=40), dict(D=528, R=64)]


@pytest.mark.parametrize("c", ROPE, ids=str)
@pytest.mark.parametrize("kw", [{}, dict(eps=1, interleaved=True), dict(eps=-1.0), dict(interleaved=1)], ids=str)
def test_rope(pkg, gpu, monkeypatch, c, kw):
    note(f"binding rope {c} {kw}")
    a = rope_args(gpu, **c)
    x, y = both(monkeypatch, lambda: pkg.qk_norm_rope(**a, **kw))
    same(x, y)
    x, y = both(monkeypatch, lambda: pkg.qk_norm_rope_bwd(a["q"], a["k"], **a, **kw))
    same(x, y)


def test_rope_outputs_and_refusals(pkg, gpu, monkeypatch):
    a = rope_args(gpu)
    qo = torch.zeros(5, 8, 64, dtype=BF16, device=gpu)[:, ::2]
    x, y = both(monkeypatch, lambda: pkg.qk_norm_rope(**a, q_out=qo))
    assert x[0] is qo and y[0] is qo
    x, y = both(monkeypatch, lambda: pkg.qk_norm_rope_bwd(a["q"], a["k"], **a, dq=qo))
    assert x[0] is qo and y[0] is qo
    for bad in (dict(q_out=qo.half()), dict(q_out=a["k"]), dict(k_out=a["q"][:, :2]), dict(q=a["q"].float()),
                dict(positions=a["positions"][:3]), dict(sin=a["sin"].half()), dict(q=a["q"].cpu()),
                dict(q_weight=a["q_weight"][:32])):
        x, y = both(monkeypatch, lambda: pkg.qk_norm_rope(**{**a, **bad}))
        assert isinstance(x[0], type) and x == y, bad


def test_cache_and_attention(pkg, gpu, monkeypatch):
    q, caches, table, lens, pp = make(3, [70, 3, 0], 2, 8, 2, 64, 16, 40)
    (kc, ks), (vc, vs) = [(c.to(gpu), s.to(gpu)) for c, s in caches]
    a = dict(q=q.to(gpu), k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, page_table=table.to(gpu),
             kv_lens=lens.to(gpu), sm_scale=0.125)
    P = dict(prefix_pages=pp.to(gpu), prefix_len=40)
    out = torch.empty_like(a["q"])
    for kw in ({}, P, dict(max_kv_len=50), dict(P, max_kv_len=1 << 40), dict(out=out),
               dict(sm_scale=1), dict(page_table=a["page_table"][:, :0].contiguous()),
               dict(kv_lens=a["kv_lens"].long()), dict(q=a["q"][:, :, ::2]),
               # refused
               dict(P, prefix_len=49), dict(prefix_len=3), dict(max_kv_len=-1), dict(q=a["q"].float()),
               dict(q=a["q"][..., :32]), dict(sm_scale=float("nan")), dict(out=a["q"]), dict(v_cache=None),
               dict(page_table=a["page_table"].long()), dict(kv_lens=a["kv_lens"][:2]), dict(ks=None)):
        note(f"binding attention {sorted(kw)}")
        x, y = both(monkeypatch, lambda: pkg.paged_attention(**{**a, **kw}))
        if isinstance(x, torch.Tensor):
            assert "out" not in kw or (x is out and y is out)
        same(x, y)
    x = torch.randn(9, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    slots = torch.arange(9, device=gpu)
    for kw in ({}, dict(v=None, v_cache=None, v_scale=None), dict(slots=slots.int()), dict(k=x[:0], v=x[:0], slots=slots[:0]),
               dict(v=None), dict(k=x[:, :1]), dict(slots=slots.float()), dict(k=x.double()), dict(k_cache=ks)):
        def write():
            c, s = kc.clone(), ks.clone()
            c2, s2 = kc.clone(), ks.clone()
            pkg.kv_cache_write(**{**dict(k=x, v=x, slots=slots, k_cache=c, v_cache=c2, k_scale=s, v_scale=s2), **kw})
            return c, s, c2, s2
        note(f"binding write {sorted(kw)}")
        same(*both(monkeypatch, write))
    cu = torch.tensor([0, 70, 73, 73], dtype=torch.int32, device=gpu)
    for kw in ({}, dict(v_cache=None, v_scale=None, v_out=None), dict(v_out=None), dict(cu_seqlens=cu[:3]),
               dict(k_out=torch.empty(73, 3, 64, dtype=BF16, device=gpu)), dict(page_table=table)):
        def read():
            o = [torch.full((75, 2, 64), 3.0, dtype=F16, device=gpu) for _ in range(2)]
            r = pkg.kv_cache_read(**{**dict(k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, page_table=a["page_table"],
                                            cu_seqlens=cu, k_out=o[0], v_out=o[1]), **kw})
            return r if r[1] is not None else r[:1]
        note(f"binding read {sorted(kw)}")
        same(*both(monkeypatch, read))
