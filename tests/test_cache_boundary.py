"""The C ABI boundary and the Python checks of qk_norm_rope, the paged cache and the attention
over it, without a GPU: every refused argument is reported before any device work, and whatever
page tables and lengths hold, the lookups stay in range."""
import ctypes
import random

import pytest
import torch

BASE = 0x10_0000_0000
I64 = ctypes.c_int64


def fake(i, off=0):
    return ctypes.c_void_p(BASE + i * 0x1_0000_0000 + off)


def i64s(*v):
    return (I64 * len(v))(*v)


# ------------------------------------------------------------------------------------ rope

def rope(lib, bwd=False, **kw):
    a = dict(q=fake(0), k=fake(1), qw=fake(2), kw=fake(3), cos=fake(4), sin=fake(5), pos=fake(6),
             qo=fake(7), ko=fake(8), dqo=fake(9), dko=fake(10), dqw=fake(11), dkw=fake(12),
             ws=fake(13), wsb=1 << 30, T=5, Hq=4, Hk=2, D=128, R=128, table=64, eps=1e-6, inter=0,
             dt=0, idx=1, sq=(512, 128), sk=(256, 128), sqo=(512, 128), sko=(256, 128),
             sdqo=(512, 128), sdko=(256, 128))
    a.update(kw)
    tail = [a["T"], a["Hq"], a["Hk"], a["D"], a["R"], a["table"], a["eps"], a["inter"], a["dt"],
            a["idx"], None]
    if bwd:
        return lib.fagq_qk_norm_rope_bwd_launch(
            a["dqo"], a["dko"], a["q"], a["k"], a["qw"], a["kw"], a["cos"], a["sin"], a["pos"],
            a["qo"], a["ko"], a["dqw"], a["dkw"], a["ws"], a["wsb"],
            i64s(*a["sdqo"], *a["sdko"], *a["sq"], *a["sk"], *a["sqo"], *a["sko"]), *tail)
    return lib.fagq_qk_norm_rope_launch(
        a["q"], a["k"], a["qw"], a["kw"], a["cos"], a["sin"], a["pos"], a["qo"], a["ko"],
        i64s(*a["sq"], *a["sk"], *a["sqo"], *a["sko"]), *tail)


COMMON = [
    (dict(q=None), 1), (dict(k=None), 1), (dict(qw=None), 1), (dict(cos=None), 1),
    (dict(sin=None), 1), (dict(pos=None), 1), (dict(qo=None), 1), (dict(ko=None), 1),
    (dict(dt=3), 5), (dict(dt=-1), 5), (dict(idx=2), 5), (dict(eps=-1.0), 6),
    (dict(eps=float("nan")), 6), (dict(eps=float("inf")), 6), (dict(T=-1), 2), (dict(Hq=0), 2),
    (dict(Hk=0), 2), (dict(D=0, R=0), 2), (dict(D=120), 2), (dict(R=24), 2), (dict(R=0), 2),
    (dict(R=144), 2), (dict(table=-1), 2), (dict(D=528), 7), (dict(T=(1 << 24) + 1), 7),
    (dict(sq=(-512, 128)), 2), (dict(sq=(1 << 31, 128)), 7), (dict(sk=(256, 132)), 4),
    (dict(sqo=(516, 128)), 4), (dict(q=fake(0, 8)), 4), (dict(cos=fake(4, 4)), 4),
    (dict(pos=fake(6, 4)), 4), (dict(qo=fake(1)), 9), (dict(ko=fake(0, 256)), 9),
    (dict(ko=fake(7)), 9), (dict(qo=fake(2)), 9), (dict(qo=fake(5)), 9), (dict(qo=fake(6)), 9),
    (dict(sqo=(0, 128)), 9), (dict(sqo=(512, 0)), 9), (dict(sqo=(256, 128)), 9),
]


@pytest.mark.parametrize("kw,status", COMMON)
@pytest.mark.parametrize("bwd", [False, True])
def test_rope_validation(lib, kw, status, bwd):
    assert rope(lib, bwd, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(T=0), 0), (dict(qo=fake(0, 2048)), 9),
    (dict(qo=fake(0), sqo=(1024, 128)), 9),                  # q's place, other strides
    (dict(dt=2, sq=(512, 132), sqo=(512, 132), qo=fake(0, 4)), 4),
])
def test_rope_fwd_validation(lib, kw, status):
    assert rope(lib, **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(dqo=None), 1), (dict(dko=None), 1), (dict(dqw=None), 1), (dict(dkw=None), 1),
    (dict(ws=None), 1), (dict(wsb=16), 2), (dict(ws=fake(13, 8)), 4), (dict(dqw=fake(11, 4)), 4),
    (dict(qo=fake(9)), 9), (dict(qo=fake(0)), 9), (dict(dqw=fake(12)), 9), (dict(ws=fake(12)), 9),
    (dict(ws=fake(9)), 9), (dict(ws=fake(7)), 9), (dict(dkw=fake(3)), 9), (dict(dqw=fake(0)), 9),
])
def test_rope_bwd_validation(lib, kw, status):
    assert rope(lib, True, **kw) == status


def test_rope_accepts_views_of_one_buffer(lib):
    """Heads that lie side by side in a fused buffer do not overlap, in place and apart; a valid
    call gets past the argument checks (here, without a GPU, to the device check)."""
    fused = dict(q=fake(0), k=fake(0, 4 * 256), sq=(1024, 128), sk=(1024, 128))
    ok = rope(lib, **fused)
    assert ok < 0 or ok == 8
    for kw in (dict(qo=fake(0), ko=fake(0, 4 * 256), sqo=(1024, 128), sko=(1024, 128)),
               dict(qo=fake(7), ko=fake(7, 4 * 256), sqo=(1024, 128), sko=(1024, 128)),
               dict(qo=fake(0, 6 * 256), sqo=(1024, 128), Hq=2)):  # a third slice of the buffer
        assert rope(lib, **{**fused, **kw}) == ok
    # One head too many reaches into the neighbour.
    assert rope(lib, **{**fused, "qo": fake(7), "ko": fake(7, 3 * 256), "sqo": (1024, 128),
                        "sko": (1024, 128)}) == 9
    assert rope(lib, **{**fused, "qo": fake(0, 7 * 256), "sqo": (1024, 128), "Hq": 2}) == 9


def test_rope_workspace(lib):
    f = lib.fagq_qk_norm_rope_bwd_workspace_bytes
    assert f(0, 4, 2, 128) == 0
    for T in (1, 7, 4096, 1 << 24):
        n = f(T, 32, 8, 128)
        assert 0 < n <= 768 * 128 * 4 and n % (128 * 4) == 0
    assert f(-1, 4, 2, 128) == -1 and f(4, 0, 2, 128) == -1 and f(4, 4, 2, 100) == -1
    assert f(4, 4, 2, 1024) == -1


# ------------------------------------------------------------------------------------ cache

def write(lib, **kw):
    a = dict(k=fake(0), v=fake(1), slots=fake(2), kc=fake(3), vc=fake(4), ks=fake(5), vs=fake(6),
             st=(1024, 128, 1024, 128), T=5, H=8, D=128, G=128, P=9, page=16, dt=0, qf=1, sf=0,
             idx=1)
    a.update(kw)
    return lib.fagq_kv_cache_write_launch(a["k"], a["v"], a["slots"], a["kc"], a["vc"], a["ks"],
                                          a["vs"], i64s(*a["st"]), a["T"], a["H"], a["D"], a["G"],
                                          a["P"], a["page"], a["dt"], a["qf"], a["sf"], a["idx"],
                                          None)


@pytest.mark.parametrize("kw,status", [
    (dict(k=None), 1), (dict(slots=None), 1), (dict(kc=None), 1), (dict(ks=None), 1),
    (dict(v=None), 1), (dict(vc=None), 1), (dict(vs=None), 1),
    (dict(dt=3), 5), (dict(qf=2), 5), (dict(sf=2), 5), (dict(idx=2), 5),
    (dict(G=32), 3), (dict(G=512), 3), (dict(G=256), 2), (dict(H=0), 2), (dict(D=0), 2),
    (dict(page=8), 2), (dict(page=24), 2), (dict(page=131072), 7), (dict(P=-1), 2),
    (dict(P=1 << 31), 7), (dict(D=2048), 7), (dict(T=-1), 2), (dict(T=(1 << 24) + 1), 7),
    (dict(st=(1028, 128, 1024, 128)), 4), (dict(st=(1024, 128, 1024, -8)), 2),
    (dict(st=(1 << 31, 128, 1024, 128)), 7), (dict(k=fake(0, 8)), 4), (dict(kc=fake(3, 8)), 4),
    (dict(ks=fake(5, 2)), 4), (dict(slots=fake(2, 4)), 4), (dict(kc=fake(0)), 9),
    (dict(vc=fake(3)), 9), (dict(vs=fake(4, 64)), 9), (dict(ks=fake(2)), 9),
    (dict(T=0), 0), (dict(P=0), 0),
])
def test_write_validation(lib, kw, status):
    assert write(lib, **kw) == status


def read(lib, **kw):
    a = dict(kc=fake(0), vc=fake(1), ks=fake(2), vs=fake(3), pt=fake(4), cu=fake(5), ko=fake(6),
             vo=fake(7), B=3, rows=50, H=8, D=128, G=128, P=9, page=16, width=4, dt=0, qf=1, sf=0)
    a.update(kw)
    return lib.fagq_kv_cache_read_launch(a["kc"], a["vc"], a["ks"], a["vs"], a["pt"], a["cu"],
                                         a["ko"], a["vo"], a["B"], a["rows"], a["H"], a["D"],
                                         a["G"], a["P"], a["page"], a["width"], a["dt"], a["qf"],
                                         a["sf"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(kc=None), 1), (dict(ks=None), 1), (dict(pt=None), 1), (dict(cu=None), 1),
    (dict(ko=None), 1), (dict(vc=None), 1), (dict(vs=None), 1), (dict(vo=None), 1),
    (dict(dt=3), 5), (dict(qf=2), 5), (dict(sf=2), 5), (dict(G=100), 3), (dict(D=192), 2),
    (dict(page=48), 2), (dict(B=-1), 2), (dict(rows=-1), 2), (dict(width=-1), 2),
    (dict(rows=1 << 31), 7), (dict(B=(1 << 24) + 1), 7), (dict(ko=fake(6, 8)), 4),
    (dict(kc=fake(0, 8)), 4), (dict(pt=fake(4, 2)), 4), (dict(vo=fake(6)), 9),
    (dict(ko=fake(0)), 9), (dict(vo=fake(2)), 9), (dict(ko=fake(4)), 9), (dict(vo=fake(5)), 9),
    (dict(B=0), 0), (dict(rows=0), 0),
])
def test_read_validation(lib, kw, status):
    assert read(lib, **kw) == status


@pytest.mark.parametrize("kw", [
    dict(pt=None, width=0), dict(kc=None, vc=None, ks=None, vs=None, P=0),
    dict(kc=None, vc=None, ks=None, vs=None, P=0, pt=None, width=0), dict(kc=None, ks=None, vo=None, vc=None, vs=None, P=0),
])
def test_read_takes_tables_and_caches_of_nothing(lib, kw):
    # Every token is one without a page; without a GPU the call ends at the device check.
    if torch.cuda.is_available():
        pytest.skip("the pointers are made up")
    ok = read(lib)
    assert (ok < 0 or ok == 8) and read(lib, **kw) == ok
    assert read(lib, **kw, cu=None) == 1 and read(lib, **kw, ko=None) == 1


def attend(lib, **kw):
    a = dict(q=fake(0), kc=fake(1), vc=fake(2), ks=fake(3), vs=fake(4), pt=fake(5), lens=fake(6),
             pp=fake(7), out=fake(8), ws=fake(9), wsb=1 << 31, st=(1024, 1024, 128), B=3, S=1, Hq=8,
             H=2, D=128, P=9, page=16, width=4, prefix=20, most=64, scale=0.1, dt=0, qf=1, sf=0,
             idx=0)
    a.update(kw)
    return lib.fagq_paged_attention_launch(
        a["q"], a["kc"], a["vc"], a["ks"], a["vs"], a["pt"], a["lens"], a["pp"], a["out"], a["ws"],
        a["wsb"], i64s(*a["st"]), a["B"], a["S"], a["Hq"], a["H"], a["D"], a["P"], a["page"],
        a["width"], a["prefix"], a["most"], a["scale"], a["dt"], a["qf"], a["sf"], a["idx"], None)


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(kc=None), 1), (dict(vc=None), 1), (dict(ks=None), 1),
    (dict(vs=None), 1), (dict(pt=None), 1), (dict(lens=None), 1), (dict(pp=None), 1),
    (dict(out=None), 1), (dict(dt=2), 5), (dict(qf=3), 5), (dict(sf=-1), 5), (dict(idx=2), 5),
    (dict(scale=float("nan")), 2), (dict(scale=float("inf")), 2), (dict(B=-1), 2), (dict(S=0), 2),
    (dict(H=0), 2), (dict(Hq=7), 2), (dict(Hq=1), 2), (dict(D=96), 2), (dict(D=512), 2),
    (dict(prefix=-1), 2), (dict(most=-1), 2), (dict(page=8), 2), (dict(page=17), 2),
    (dict(P=-1), 2), (dict(width=-1), 2), (dict(B=65536), 7), (dict(Hq=8192, H=1), 7),
    (dict(S=65535, B=65535), 7), (dict(prefix=1 << 31), 7), (dict(most=1 << 31), 7),
    (dict(page=131072), 7), (dict(st=(1024, 1024, 132)), 4), (dict(st=(1024, -8, 128)), 2),
    (dict(st=(1 << 31, 1024, 128)), 7), (dict(q=fake(0, 8)), 4), (dict(ks=fake(3, 2)), 4),
    (dict(lens=fake(6, 4), idx=1), 4), (dict(pp=fake(7, 2)), 4), (dict(out=fake(8, 8)), 4),
    (dict(out=fake(0)), 9), (dict(out=fake(2)), 9), (dict(out=fake(5)), 9), (dict(out=fake(7)), 9),
    (dict(B=0), 0),
])
def test_attention_validation(lib, kw, status):
    assert attend(lib, **kw) == status


def test_attention_workspace_is_checked(lib):
    f = lib.fagq_paged_attention_workspace_bytes
    for bad in ((-1, 1, 8, 2, 128, 0, 64), (1, 0, 8, 2, 128, 0, 64), (1, 1, 8, 3, 128, 0, 64),
                (1, 1, 8, 2, 100, 0, 64), (1, 1, 8, 2, 128, -1, 64), (1, 1, 8, 2, 128, 0, -1)):
        assert f(*bad) == -1
    need = f(3, 1, 8, 2, 128, 20, 64)
    assert need >= 0
    if need:
        assert attend(lib, ws=None) == 1
        assert attend(lib, wsb=need - 1) == 2
        assert attend(lib, ws=fake(9, 8)) == 4
        assert attend(lib, ws=fake(8)) == 9
        assert attend(lib, ws=fake(2)) == 9


@pytest.mark.parametrize("large,small", [
    (dict(B=64, S=1, Hq=64, H=8, D=128, most=1024), dict(B=16)),
    (dict(B=112, S=16, Hq=32, H=8, D=256, most=9409), dict(most=8190)),
    (dict(B=83, S=16, Hq=64, H=8, D=256, most=2574), dict(B=41)),
])
def test_a_smaller_call_may_need_a_larger_workspace(lib, large, small):
    # As documented: the larger call's workspace is refused then, before any device work.
    small = {**large, **small}
    size = lambda c: lib.fagq_paged_attention_workspace_bytes(c["B"], c["S"], c["Hq"], c["H"], c["D"], 0, c["most"])
    call = lambda c, n: attend(lib, **c, width=1 << 10, prefix=0, wsb=n, ws=fake(9),
                               st=(c["S"] * c["Hq"] * c["D"], c["Hq"] * c["D"], c["D"]))
    assert 0 <= size(large) < size(small)
    assert call(small, size(large)) == 2
    assert call(small, size(small) - 1) == 2


def test_attention_refuses_what_no_grid_holds(lib):
    # The largest grid is below 2^24 workgroups, and the joining kernel may have one for each row.
    f = lib.fagq_paged_attention_workspace_bytes
    assert f(65535, 1, 256, 256, 128, 0, 64) >= 0
    assert f(4096, 1, 4096, 4096, 128, 0, 64) == -1
    assert attend(lib, B=4096, Hq=4096, H=4096, prefix=0) == 7
    # 65535 * 256 units of own keys, and those of the prefix ahead of them.
    assert f(65535, 1, 256, 256, 128, 64, 64) == -1
    assert attend(lib, B=65535, Hq=256, H=256, prefix=64) == 7


def test_attention_workspace_of_any_size_is_moderate(lib):
    # A row has few parts, however its keys are cut: rows x parts of (D + 2) floats.
    f = lib.fagq_paged_attention_workspace_bytes
    for B, S, H in ((1, 1, 1), (1, 1, 8), (3, 1, 5), (1, 512, 1), (64, 1, 8), (700, 2, 3)):
        for prefix, most in ((0, 1), (0, 100000), (0, 1 << 22), (1 << 20, 64), (5000, 5000)):
            need = f(B, S, 8 * H, H, 128, prefix, most)
            assert 0 <= need <= (B * S * 8 * H * 1100 + 512 * 2 * 64) * 130 * 4 + 4 * (B + 1)


# ------------------------------------------------------------------------------------ lookups

def slots(lib, table, cu, pages, page, rows):
    B, width = len(table), len(table[0]) if table else 0
    flat = (ctypes.c_int32 * max(1, B * width))(*[x for r in table for x in r])
    out = (I64 * max(1, rows))(*([7] * max(1, rows)))
    st = lib.fagq_diag_cache_slots(flat, (ctypes.c_int32 * len(cu))(*cu), B, width, pages, page,
                                   out, rows)
    assert st == 0
    return list(out)[:rows]


def test_lookups_of_ragged_batches(lib):
    # 3 tokens, none, 17 tokens over two pages of 16, 1 token; two rows behind the last.
    table = [[4, -1], [-1, -1], [2, 0], [9, 3]]
    got = slots(lib, table, [0, 3, 3, 20, 21], 10, 16, 23)
    want = [64, 65, 66] + [32 + i for i in range(16)] + [0] + [144] + [-2, -2]
    assert got == want


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 10, 2 ** 31 - 1])
def test_pages_outside_the_cache_are_no_pages(lib, bad):
    got = slots(lib, [[1, bad, 2]], [0, 48], 10, 16, 48)
    assert got == list(range(16, 32)) + [-1] * 16 + list(range(32, 48))


def test_tokens_past_the_table_have_no_page(lib):
    assert slots(lib, [[1]], [0, 20], 10, 16, 20) == list(range(16, 32)) + [-1] * 4


def test_lookups_stay_in_range_for_any_content(lib):
    rng = random.Random(5)
    wild = lambda: rng.choice([rng.randint(-5, 40), rng.randint(-2 ** 31, 2 ** 31 - 1)])
    for _ in range(200):
        B, width, pages = rng.randint(0, 5), rng.randint(1, 4), rng.randint(0, 12)
        table = [[wild() for _ in range(width)] for _ in range(B)]
        cu = [wild() for _ in range(B + 1)]
        for v in slots(lib, table, cu, pages, 16, 40):
            assert -2 <= v < pages * 16


# ------------------------------------------------------------------------------------ Python

def meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype)


def test_python_refuses_cpu_tensors_and_bad_arguments(pkg):
    q, k, w = meta(3, 4, 64), meta(3, 2, 64), meta(64)
    cos = meta(8, 32, dtype=torch.float32)
    pos = meta(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="no CPU path"):
        pkg.qk_norm_rope(q, k, w, w, cos, cos, pos)
    with pytest.raises(TypeError):
        pkg.qk_norm_rope(q.int(), k, w, w, cos, cos, pos)
    with pytest.raises(ValueError):
        pkg.qk_norm_rope(q[0], k, w, w, cos, cos, pos)
    with pytest.raises(ValueError, match="no CPU path"):
        pkg.qk_norm_rope_bwd(q, k, q, k, w, w, cos, cos, pos)
    kc, ks = pkg.empty_kv_cache(2, 2, 16, 64, device="cpu")
    assert kc.shape == (2, 2, 16, 64) and ks.shape == (2, 2, 1, 16) and ks.dtype == torch.float32
    with pytest.raises(ValueError, match="no CPU path"):
        pkg.kv_cache_write(k, None, pos, kc, None, ks, None)
    with pytest.raises(ValueError, match="no CPU path"):
        pkg.kv_cache_read(kc, None, ks, None, meta(1, 1, dtype=torch.int32),
                          meta(2, dtype=torch.int32), k, None)
    with pytest.raises(ValueError, match="no CPU path"):
        pkg.paged_attention(meta(1, 1, 2, 64), kc, kc, ks, ks, meta(1, 1, dtype=torch.int32),
                            meta(1, dtype=torch.int32), 0.1)
    with pytest.raises(TypeError):
        pkg.kv_cache_write(k, None, pos, meta(2, 2, 16, 64), None, ks, None)
    with pytest.raises(TypeError):
        pkg.kv_cache_write(k, None, pos, kc, None, ks.double(), None)


def test_empty_kv_cache_formats(pkg):
    c, s = pkg.empty_kv_cache(3, 1, 64, 512, 128, torch.int8, True, device="cpu")
    assert c.dtype == torch.int8 and s.dtype == torch.uint8 and s.shape == (3, 1, 4, 64)
    for D, G in ((512, None), (96, None), (128, 256), (128, 32)):
        with pytest.raises(ValueError):
            pkg.empty_kv_cache(3, 1, 64, D, G, device="cpu")


def test_empty_kv_cache_refuses_codes_that_no_operator_takes(pkg):
    with pytest.raises(TypeError, match="float8_e4m3fn or int8"):
        pkg.empty_kv_cache(2, 2, 16, 64, dtype=torch.bfloat16, device="cpu")
