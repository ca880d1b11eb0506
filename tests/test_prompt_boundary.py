"""The C ABI boundary and the Python checks of the attention of prompts, its gradients, draft trees and
step tables, without a GPU: every refused argument is reported before any device work."""
import ctypes

import pytest
import torch

from tests import prompt_ref
from tests.test_cache_boundary import fake, i64s


def forward(lib, **kw):
    a = dict(q=fake(0), k=fake(1), v=fake(2), cu=fake(3), cu_k=fake(4), out=fake(5), lse=fake(6), ws=fake(7), wsb=1 << 34,
             st=(512, 128, 256, 128, 256, 128), B=3, T=50, Tk=70, Hq=4, H=2, D=128, scale=0.1, dt=0, fill=3)
    a.update(kw)
    return lib.fagq_prompt_attention_launch(
        a["q"], a["k"], a["v"], a["cu"], a["cu_k"], a["out"], a["lse"], a["ws"], a["wsb"], i64s(*a["st"]), a["B"],
        a["T"], a["Tk"], a["Hq"], a["H"], a["D"], a["scale"], a["dt"], a["fill"], None)


def backward(lib, **kw):
    a = dict(do=fake(8), q=fake(0), k=fake(1), v=fake(2), out=fake(5), lse=fake(6), cu=fake(3), cu_k=fake(4), dq=fake(9),
             dk=fake(10), dv=fake(11), ws=fake(7), wsb=1 << 34, sdo=(512, 128), sq=(512, 128), sk=(256, 128), sv=(256, 128),
             sdq=(512, 128), sdk=(256, 128), sdv=(256, 128), B=3, T=50, Tk=70, Hq=4, H=2, D=128, scale=0.1, dt=0, fill=7)
    a.update(kw)
    st = sum((a[n] for n in ("sdo", "sq", "sk", "sv", "sdq", "sdk", "sdv")), ())
    return lib.fagq_prompt_attention_bwd_launch(
        a["do"], a["q"], a["k"], a["v"], a["out"], a["lse"], a["cu"], a["cu_k"], a["dq"], a["dk"], a["dv"], a["ws"],
        a["wsb"], i64s(*st), a["B"], a["T"], a["Tk"], a["Hq"], a["H"], a["D"], a["scale"], a["dt"], a["fill"], None)


SIZES = [
    (dict(B=-1), 2), (dict(T=-1), 2), (dict(Tk=-1), 2), (dict(H=0), 2), (dict(Hq=3), 2), (dict(Hq=1), 2), (dict(D=96), 2),
    (dict(D=512), 2), (dict(D=0), 2), (dict(scale=float("nan")), 2), (dict(scale=float("inf")), 2), (dict(dt=2), 5),
    (dict(dt=-1), 5), (dict(fill=8), 5), (dict(fill=-1), 5), (dict(B=(1 << 24) + 1), 7), (dict(T=1 << 31), 7),
    (dict(Tk=1 << 31), 7), (dict(Hq=8192), 7), (dict(T=(1 << 31) - 1, Hq=64), 7), (dict(cu=None), 1), (dict(q=None), 1),
    (dict(k=None), 1), (dict(v=None), 1), (dict(out=None), 1), (dict(cu=fake(3, 2)), 4), (dict(cu_k=fake(4, 2)), 4),
    (dict(q=fake(0, 8)), 4), (dict(v=fake(2, 8)), 4), (dict(out=fake(5, 8)), 4), (dict(lse=fake(6, 2)), 4),
    (dict(ws=fake(7, 8)), 4), (dict(cu_k=None), 2),
    (dict(T=(1 << 31) - 1023, Hq=1, H=1), 7), (dict(Tk=(1 << 31) - 1023, Hq=1, H=1), 7),
]


@pytest.mark.parametrize("kw,status", SIZES + [
    (dict(st=(512, 128, 256, 128, 256, -8)), 2), (dict(st=(1 << 24, 128, 256, 128, 256, 128)), 7),
    (dict(st=(512, 1 << 31, 256, 128, 256, 128)), 7), (dict(st=(512, 128, 260, 128, 256, 128)), 4),
    (dict(out=fake(0)), 9), (dict(out=fake(2, 512)), 9), (dict(out=fake(3)), 9), (dict(lse=fake(1)), 9), (dict(lse=fake(5)), 9),
    (dict(T=0), 0), (dict(B=0, T=0, Tk=0, k=None, v=None, cu_k=None), 0),
])
def test_forward_validation(lib, kw, status):
    assert forward(lib, **kw) == status


@pytest.mark.parametrize("kw,status", SIZES + [
    (dict(do=None), 1), (dict(lse=None), 1), (dict(dq=None), 1), (dict(dk=None), 1), (dict(dv=None), 1), (dict(ws=None), 1),
    (dict(wsb=16, T=5000, Tk=5000), 2), (dict(sdo=(512, -8)), 2), (dict(sdk=(1 << 24, 128)), 7), (dict(sdv=(256, 132)), 4),
    (dict(do=fake(8, 8)), 4), (dict(dk=fake(10, 8)), 4), (dict(dq=fake(0)), 9), (dict(dq=fake(8)), 9), (dict(dk=fake(9, 512)), 9),
    (dict(dv=fake(10)), 9), (dict(dk=fake(5)), 9), (dict(dv=fake(4)), 9), (dict(dq=fake(7)), 9), (dict(ws=fake(1)), 9),
    (dict(ws=fake(5)), 9), (dict(ws=fake(6)), 9), (dict(sdq=(0, 128)), 9), (dict(sdq=(512, 0)), 9), (dict(sdk=(128, 128)), 9),
    (dict(B=0, T=0, Tk=0, cu_k=None, q=None, k=None, v=None, do=None, out=None, lse=None, dq=None, dk=None, dv=None, ws=None,
          wsb=0), 0),
])
def test_backward_validation(lib, kw, status):
    if status in (1, 2, 4, 9) and ("ws" in kw or kw.get("dq") is not None):
        kw = {**dict(T=5000, Tk=5000, B=1), **kw}          # a call that has a workspace
    assert backward(lib, **kw) == status


def past_the_checks(status):
    return status < 0 or status == 8


def test_calls_that_pass(lib):
    """Without a GPU a valid call ends at the device check."""
    if torch.cuda.is_available():
        pytest.skip("the pointers are made up")
    for kw in ({}, dict(lse=None, fill=1), dict(cu_k=None, Tk=50), dict(Tk=0, k=None, v=None), dict(B=0), dict(D=64, st=(512, 64) * 3),
               dict(scale=-3.0), dict(st=((1 << 24) - 8, 128) * 3)):
        assert past_the_checks(forward(lib, **kw)), kw
    for kw in ({}, dict(Tk=0, k=None, v=None, dk=None, dv=None),
               dict(T=0, q=None, do=None, out=None, lse=None, dq=None),
               # views of one buffer for the inputs, and of one for the gradients
               dict(cu_k=None, T=70, q=fake(0), k=fake(0, 1024), v=fake(0, 1536), sq=(1024, 128), sk=(1024, 128), sv=(1024, 128),
                    dq=fake(9), dk=fake(9, 1024), dv=fake(9, 1536), sdq=(1024, 128), sdk=(1024, 128), sdv=(1024, 128))):
        assert past_the_checks(backward(lib, **kw)), kw
    # One head too many reaches into the neighbour.
    assert backward(lib, cu_k=None, T=70, dq=fake(9), dk=fake(9, 768), sdq=(1024, 128), sdk=(1024, 128)) == 9


def test_workspaces(lib):
    f, b = lib.fagq_prompt_attention_workspace_bytes, lib.fagq_prompt_attention_bwd_workspace_bytes
    assert f(4, 16384, 16384, 64, 8, 128) == 0             # fills the GPU as it is
    assert f(1, 128, 65536, 8, 8, 128) % (128 * 8 * 130 * 4) == 0 < f(1, 128, 65536, 8, 8, 128)
    assert f(0, 0, 0, 4, 2, 64) == 0 and b(0, 0, 0, 4, 2, 64) == 0
    assert b(1, 64, 64, 4, 2, 64) == 0                     # one launch, no parts
    assert b(1, 8192, 8192, 32, 8, 128) == 2 * 32 * 8192 * 4
    for bad in ((-1, 4, 4, 4, 2, 64), (1, -1, 4, 4, 2, 64), (1, 4, 4, 3, 2, 64), (1, 4, 4, 4, 0, 64), (1, 4, 4, 4, 2, 80),
                (1, 1 << 31, 4, 4, 2, 64), (1 << 25, 4, 4, 4, 2, 64)):
        assert f(*bad) == -1 and b(*bad) == -1


def tree(lib, **kw):
    a = dict(q=fake(0), kc=fake(1), vc=fake(2), ks=fake(3), vs=fake(4), pt=fake(5), lens=fake(6), pp=fake(7), mask=fake(10),
             shared=0, out=fake(8), ws=fake(9), wsb=1 << 31, st=(6144, 1024, 128), B=3, S=6, Hq=8, H=2, D=128, P=9, page=16,
             width=4, prefix=20, most=64, scale=0.1, dt=0, qf=1, sf=0, idx=0)
    a.update(kw)
    return lib.fagq_paged_tree_attention_launch(
        a["q"], a["kc"], a["vc"], a["ks"], a["vs"], a["pt"], a["lens"], a["pp"], a["mask"], a["shared"], a["out"], a["ws"],
        a["wsb"], i64s(*a["st"]), a["B"], a["S"], a["Hq"], a["H"], a["D"], a["P"], a["page"], a["width"], a["prefix"],
        a["most"], a["scale"], a["dt"], a["qf"], a["sf"], a["idx"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(mask=None), 1), (dict(q=None), 1), (dict(pp=None), 1), (dict(S=4097, B=1), 7), (dict(S=0), 2), (dict(Hq=7), 2),
    (dict(out=fake(10)), 9), (dict(out=fake(10, 96)), 9), (dict(ws=fake(10, 64)), 9), (dict(out=fake(1)), 9), (dict(D=96), 2),
    (dict(dt=2), 5), (dict(idx=3), 5), (dict(page=24), 2), (dict(wsb=0), 2), (dict(B=0), 0),
])
def test_tree_validation(lib, kw, status):
    assert tree(lib, **kw) == status


def test_tree_masks_of_one_and_of_all(lib):
    if torch.cuda.is_available():
        pytest.skip("the pointers are made up")
    assert past_the_checks(tree(lib)) and past_the_checks(tree(lib, shared=1)) and past_the_checks(tree(lib, mask=fake(10, 1)))
    # 36 bytes of one mask, 108 of three: what lies behind them is free for outputs.
    assert past_the_checks(tree(lib, shared=1, out=fake(10, 48))) and tree(lib, out=fake(10, 48)) == 9
    f = lib.fagq_paged_tree_attention_workspace_bytes
    assert f(3, 6, 8, 2, 128, 20, 64) >= 0 and f(0, 6, 8, 2, 128, 0, 64) == 0 and f(3, 4097, 8, 2, 128, 0, 64) == -1


def tables(lib, **kw):
    a = dict(ctx=fake(0), new=fake(1), free=fake(2), start=fake(3), pt=fake(4), cu=fake(5), cu_k=fake(6), lens=fake(7), pos=fake(8),
             slots=fake(9), end=fake(10), B=3, rows=50, F=9, page=16, width=4, idx=0)
    a.update(kw)
    return lib.fagq_batch_tables_launch(a["ctx"], a["new"], a["free"], a["start"], a["pt"], a["cu"], a["cu_k"], a["lens"],
                                        a["pos"], a["slots"], a["end"], a["B"], a["rows"], a["F"], a["page"], a["width"],
                                        a["idx"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(ctx=None), 1), (dict(new=None), 1), (dict(free=None), 1), (dict(pt=None), 1), (dict(cu=None), 1), (dict(cu_k=None), 1),
    (dict(lens=None), 1), (dict(pos=None), 1), (dict(slots=None), 1), (dict(end=None), 1), (dict(B=-1), 2), (dict(rows=-1), 2),
    (dict(F=-1), 2), (dict(width=-1), 2), (dict(page=8), 2), (dict(page=48), 2), (dict(page=131072), 7), (dict(idx=2), 5),
    (dict(B=(1 << 24) + 1), 7), (dict(rows=1 << 31), 7), (dict(F=1 << 31), 7), (dict(width=1 << 31), 7), (dict(ctx=fake(0, 4), idx=1), 4),
    (dict(slots=fake(9, 4)), 4), (dict(pos=fake(8, 2)), 4), (dict(start=fake(3, 2)), 4), (dict(pt=fake(2)), 9), (dict(pt=fake(0)), 9),
    (dict(end=fake(3)), 9), (dict(lens=fake(1)), 9), (dict(cu=fake(6, 8)), 9), (dict(slots=fake(8)), 9), (dict(lens=fake(0, 8)), 9),
])
def test_tables_validation(lib, kw, status):
    assert tables(lib, **kw) == status


def test_tables_of_nothing(lib):
    if torch.cuda.is_available():
        pytest.skip("the pointers are made up")
    for kw in ({}, dict(start=None), dict(F=0, free=None), dict(rows=0, pos=None, slots=None), dict(width=0, pt=None),
               dict(B=0, ctx=None, new=None, lens=None, pt=None)):
        assert past_the_checks(tables(lib, **kw)), kw


def test_python_refuses_cpu_tensors(pkg):
    q, cu = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ValueError):
        pkg.prompt_attention(q, q, q, cu, 0.1)
    with pytest.raises(ValueError):
        pkg.prompt_attention_bwd(q, q, q, q, q, torch.zeros(2, 4), cu, 0.1)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        pkg.batch_tables(i, i, i, i[:, None], 16, 4)
    c, s = pkg.empty_kv_cache(2, 2, 16, 64, device="cpu")
    with pytest.raises(ValueError):
        pkg.paged_tree_attention(q[None], c, c, s, s, i[:, None], i, torch.ones(4, 4, dtype=torch.bool), 0.1)


def test_the_binding_leaves_cpu_tensors_and_odd_arguments_to_python(pkg):
    from fagq_mi355x import _lib
    if _lib.fast_launch() is None:
        pytest.skip("binding not built")
    b, err = _lib._fast_mod, _lib.FAST_ARG_ERROR
    q, cu = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    lse, i = torch.zeros(2, 4), torch.zeros(1, dtype=torch.int32)
    assert b.prompt(q, q, q, cu, None, 0.1, False, None, 0) == err and b.prompt(q, q, q, cu, None, 0.1, 1, None, 0) == err
    assert b.prompt_bwd(q, q, q, cu, None, 0.1, q, q, lse, None, None, None, 0) == err
    assert b.tables(i, i, i, i[:, None], 16, 4, None, 0) == err and b.tables(i, i, i, i[:, None], 16.0, 4, None, 0) == err
    c, s = pkg.empty_kv_cache(2, 2, 16, 64, device="cpu")
    assert b.tree_attention(q[None], c, c, s, s, i[:, None], i, 0.1, None, 0, None, None, 0, i) == err
    for fn, n in ((b.prompt, 9), (b.prompt_bwd, 13), (b.tables, 8), (b.tree_attention, 14), (b.bind_prompts, 7)):
        with pytest.raises(TypeError):
            fn(*[0] * (n - 1))
    with pytest.raises(ValueError):
        b.bind_prompts(*[0] * 7)


def test_the_gradients_formula_against_differences():
    """prompt_ref's own gradients: slopes of its forward in 64 bits."""
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(n, h, 8, generator=g, dtype=torch.float64) for n, h in ((9, 4), (12, 2), (12, 2), (9, 4)))
    cu, cu_k = torch.tensor([0, 4, 4, 9]), torch.tensor([0, 7, 9, 12])
    HALF = prompt_ref.HALF
    HALF[torch.float64] = prompt_ref.LOST[torch.float64] = 0.0
    try:
        out, _, lse, _ = prompt_ref.forward(q, k, v, cu, 0.3, cu_k)
        grads = prompt_ref.backward(do, q, k, v, out, lse, cu, 0.3, cu_k)
        for i in range(3):
            way = torch.randn([q, k, v][i].shape, generator=g, dtype=torch.float64)
            ends = []
            for sign in (1, -1):
                moved = [t.clone() for t in (q, k, v)]
                moved[i] += sign * 1e-5 * way
                ends.append((prompt_ref.forward(*moved, cu, 0.3, cu_k)[0] * do).sum())
            assert abs(float((ends[0] - ends[1]) / 2e-5 - (grads[i][0] * way).sum())) < 1e-7
    finally:
        del HALF[torch.float64], prompt_ref.LOST[torch.float64]
