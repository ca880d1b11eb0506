"""qk_norm_rope and its gradients on the GPU against 64-bit formulas (tests/attention_ref.py has
them and the bounds), against differences, and the calls that its documentation allows: views of
a fused buffer, in place, padding rows, every type, width and pairing."""
import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
P = 96


def inputs(T, Hq, Hk, D, R, dtype, seed, idx=torch.int64, padding=False):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(T, Hq + 2 * Hk, D, generator=g)
    qkv[..., :2] *= 8.0
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype) for _ in range(2)]
    pos = torch.randint(0, P, (T,), generator=g)
    if padding:
        pos[::3] = torch.tensor([-1, P, -2 ** 31, 2 ** 31 - 1])[torch.arange(len(pos[::3])) % 4]
    return qkv.to(dtype), w, ref.tables(P, R), pos.to(idx)


CASES = [
    # T, Hq, Hk, D, R, interleaved
    (1, 1, 1, 16, 16, False), (1, 32, 8, 128, 128, False), (3, 5, 1, 64, 32, True),
    (7, 12, 12, 96, 32, True), (33, 3, 2, 80, 80, False), (5, 4, 4, 112, 48, False),
    (65, 64, 8, 128, 128, False), (17, 9, 3, 192, 64, False), (2, 16, 2, 256, 256, True),
    (9, 2, 1, 512, 512, False), (4, 3, 3, 320, 16, True), (129, 17, 1, 128, 64, False),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_forward(pkg, gpu, case, dtype):
    T, Hq, Hk, D, R, inter = case
    note(f"qk_norm_rope {case} {dtype}")
    qkv, (wq, wk), (cos, sin), pos = inputs(T, Hq, Hk, D, R, dtype, T * D + R)
    d = qkv.to(gpu)
    yq, yk = pkg.qk_norm_rope(d[:, :Hq], d[:, Hq:Hq + Hk], wq.to(gpu), wk.to(gpu), cos.to(gpu),
                              sin.to(gpu), pos.to(gpu), 1e-6, interleaved=inter)
    for y, x, w in ((yq, qkv[:, :Hq], wq), (yk, qkv[:, Hq:Hq + Hk], wk)):
        assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
        r, bound = ref.rope(x, w, cos, sin, pos, 1e-6, inter)
        assert ref.outside(y, r, bound, dtype) == 0
    assert torch.equal(d.cpu(), qkv)                       # the inputs are as they were


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_backward(pkg, gpu, case, dtype):
    T, Hq, Hk, D, R, inter = case
    note(f"qk_norm_rope_bwd {case} {dtype}")
    qkv, (wq, wk), (cos, sin), pos = inputs(T, Hq, Hk, D, R, dtype, T * D + R, torch.int32)
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(T, Hq + Hk, D, generator=g).to(dtype)
    d, dd = qkv.to(gpu), dy.to(gpu)
    dq, dk, dwq, dwk = pkg.qk_norm_rope_bwd(
        dd[:, :Hq], dd[:, Hq:], d[:, :Hq], d[:, Hq:Hq + Hk], wq.to(gpu), wk.to(gpu), cos.to(gpu),
        sin.to(gpu), pos.to(gpu), 1e-6, interleaved=inter)
    for dx, dw, y, x, w in ((dq, dwq, dy[:, :Hq], qkv[:, :Hq], wq),
                            (dk, dwk, dy[:, Hq:], qkv[:, Hq:Hq + Hk], wk)):
        rx, bx, rw, bw = ref.rope_bwd(y, x, w, cos, sin, pos, 1e-6, inter)
        assert ref.outside(dx, rx, bx, dtype) == 0
        assert dw.dtype == F32 and ref.outside(dw, rw, bw, F32) == 0


@pytest.mark.parametrize("T", [1, 2, 511, 2048, 4095, 5000])
def test_every_split_of_the_work(pkg, gpu, T):
    """The heads of a token are shared out over waves in few tokens, and the backward's
    workgroups take several tokens in many."""
    Hq, Hk, D = 24, 3, 64
    note(f"split T={T}")
    qkv, (wq, wk), (cos, sin), pos = inputs(T, Hq, Hk, D, D, BF16, T)
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(T, Hq + Hk, D, generator=g).bfloat16()
    d, dd = qkv.to(gpu), dy.to(gpu)
    args = (wq.to(gpu), wk.to(gpu), cos.to(gpu), sin.to(gpu), pos.to(gpu))
    yq, yk = pkg.qk_norm_rope(d[:, :Hq], d[:, Hq:Hq + Hk], *args)
    got = pkg.qk_norm_rope_bwd(dd[:, :Hq], dd[:, Hq:], d[:, :Hq], d[:, Hq:Hq + Hk], *args)
    for y, dx, dw, o, x, w in ((yq, got[0], got[2], dy[:, :Hq], qkv[:, :Hq], wq),
                               (yk, got[1], got[3], dy[:, Hq:], qkv[:, Hq:Hq + Hk], wk)):
        r, bound = ref.rope(x, w, cos, sin, pos, 1e-6, False)
        assert ref.outside(y, r, bound, BF16) == 0
        rx, bx, rw, bw = ref.rope_bwd(o, x, w, cos, sin, pos, 1e-6, False)
        assert ref.outside(dx, rx, bx, BF16) == 0 and ref.outside(dw, rw, bw, F32) == 0
    again = pkg.qk_norm_rope_bwd(dd[:, :Hq], dd[:, Hq:], d[:, :Hq], d[:, Hq:Hq + Hk], *args)
    assert all(torch.equal(a, b) for a, b in zip(got, again))     # no order to change


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_padding_rows_are_zeros_and_add_nothing(pkg, gpu, dtype):
    T, Hq, Hk, D = 50, 6, 2, 128
    note(f"padding {dtype}")
    qkv, (wq, wk), (cos, sin), pos = inputs(T, Hq, Hk, D, 64, dtype, 3, padding=True)
    pad = (pos < 0) | (pos >= P)
    qkv[pad] = float("nan")                               # what padding rows hold does not matter
    g = torch.Generator().manual_seed(1)
    dy = torch.randn(T, Hq + Hk, D, generator=g).to(dtype)
    dy[pad] = float("inf")
    d, dd = qkv.to(gpu), dy.to(gpu)
    args = (wq.to(gpu), wk.to(gpu), cos.to(gpu), sin.to(gpu), pos.to(gpu))
    y = pkg.qk_norm_rope(d[:, :Hq], d[:, Hq:Hq + Hk], *args)
    got = pkg.qk_norm_rope_bwd(dd[:, :Hq], dd[:, Hq:], d[:, :Hq], d[:, Hq:Hq + Hk], *args)
    clean, cdy = qkv.clone(), dy.clone()
    clean[pad], cdy[pad] = 1.0, 1.0
    for i, (lo, hi, w) in enumerate(((0, Hq, wq), (Hq, Hq + Hk, wk))):
        r, bound = ref.rope(clean[:, lo:hi], w, cos, sin, pos, 1e-6, False)
        assert ref.outside(y[i], r, bound, dtype) == 0 and bool((y[i].cpu()[pad] == 0).all())
        rx, bx, rw, bw = ref.rope_bwd(cdy[:, lo:hi], clean[:, lo:hi], w, cos, sin, pos, 1e-6, False)
        assert ref.outside(got[i], rx, bx, dtype) == 0 and bool((got[i].cpu()[pad] == 0).all())
        assert ref.outside(got[2 + i], rw, bw, F32) == 0


def test_layouts_in_place_and_fused_gradients(pkg, gpu):
    T, Hq, Hk, D = 37, 8, 2, 128
    note("layouts")
    qkv, (wq, wk), (cos, sin), pos = inputs(T, Hq, Hk, D, D, BF16, 11)
    args = (wq.to(gpu), wk.to(gpu), cos.to(gpu), sin.to(gpu), pos.to(gpu))
    d = qkv.to(gpu)
    q, k = d[:, :Hq], d[:, Hq:Hq + Hk]
    want = pkg.qk_norm_rope(q, k, *args)
    # heads first
    qt, kt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k))
    qo = torch.empty(Hq, T, D, dtype=BF16, device=gpu).transpose(0, 1)
    got = pkg.qk_norm_rope(qt, kt, *args, q_out=qo)
    assert got[0] is qo and torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # one row for all heads and tokens
    one = pkg.qk_norm_rope(q[:1, :1].expand(T, Hq, D), k, *args)[0]
    for h in range(1, Hq):
        assert torch.equal(one[:, h], one[:, 0])
    # in place, within the fused buffer
    fused = d.clone()
    fq, fk = fused[:, :Hq], fused[:, Hq:Hq + Hk]
    r = pkg.qk_norm_rope(fq, fk, *args, q_out=fq, k_out=fk)
    assert r[0] is fq and r[1] is fk
    assert torch.equal(fq, want[0]) and torch.equal(fk, want[1])
    assert torch.equal(fused[:, Hq + Hk:], d[:, Hq + Hk:])
    # gradients into one buffer, the third part untouched
    dy = torch.randn(T, Hq + Hk, D, generator=torch.Generator().manual_seed(1)).bfloat16().to(gpu)
    plain = pkg.qk_norm_rope_bwd(dy[:, :Hq], dy[:, Hq:], q, k, *args)
    dqkv = torch.full_like(d, 7.0)
    from fagq_mi355x import qk_rope
    need = qk_rope.bwd_workspace_bytes(T, Hq, Hk, D)
    ws = torch.full((need + 4096,), 0xFF, dtype=torch.uint8, device=gpu)
    got = pkg.qk_norm_rope_bwd(dy[:, :Hq], dy[:, Hq:], q, k, *args, dq=dqkv[:, :Hq],
                               dk=dqkv[:, Hq:Hq + Hk], workspace=ws[:need])
    assert all(torch.equal(a, b) for a, b in zip(got, plain))
    assert bool((dqkv[:, Hq + Hk:] == 7.0).all()) and bool((ws[need:] == 0xFF).all())


@pytest.mark.parametrize("inter", [False, True])
def test_gradients_against_differences(pkg, gpu, inter):
    """(L(x + h v) - L(x - h v)) / 2h of the kernel's own fp32 forward, L = sum dy y in 64 bits,
    against the kernel's gradients times v.  The difference's error: what the formula in 64 bits
    itself has at this h, and the outputs' rounding (ref.rope's bound and half a step) over h."""
    T, Hq, Hk, D, R, h = 6, 4, 2, 64, 32, 2.0 ** -6
    note(f"differences {inter}")
    qkv, (wq, wk), (cos, sin), pos = inputs(T, Hq, Hk, D, R, F32, 21)
    g = torch.Generator().manual_seed(2)
    q, k = qkv[:, :Hq].contiguous(), qkv[:, Hq:Hq + Hk].contiguous()
    dy = [torch.randn(t.shape, generator=g) for t in (q, k)]
    v = [torch.randn(t.shape, generator=g) for t in (q, k, wq, wk)]
    consts = [t.to(gpu) for t in (cos, sin, pos)]
    grads = pkg.qk_norm_rope_bwd(*[t.to(gpu) for t in (*dy, q, k, wq, wk)], *consts, 1e-6, inter)
    slope = sum(float((a.double().cpu() * b).sum()) for a, b in zip(grads, v))

    def losses(sign):
        moved = [(t.double() + sign * h * s).float() for t, s in zip((q, k, wq, wk), v)]
        y = pkg.qk_norm_rope(*[t.to(gpu) for t in moved], *consts, 1e-6, inter)
        got = sum(float((a.double().cpu() * b).sum()) for a, b in zip(y, dy))
        plain = noise = 0.0
        for x, w, o in ((moved[0], moved[2], dy[0]), (moved[1], moved[3], dy[1])):
            r, bound = ref.rope(x, w, cos, sin, pos, 1e-6, inter)
            plain += float((r * o).sum())
            noise += float(((bound + ref.rounding(r, F32)) * o.abs()).sum())
        return got, plain, noise

    up, down = losses(1), losses(-1)
    exact, gb = 0.0, 0.0
    for i in (0, 1):
        rx, bx, rw, bw = ref.rope_bwd(dy[i], (q, k)[i], (wq, wk)[i], cos, sin, pos, 1e-6, inter)
        exact += float((rx * v[i]).sum()) + float((rw * v[2 + i]).sum())
        gb += float(((bx + ref.rounding(rx, F32)) * v[i].abs()).sum())
        gb += float(((bw + ref.rounding(rw, F32)) * v[2 + i].abs()).sum())
    # Rounding the moved inputs to fp32 is part of both `got` and `plain`.
    own = abs((up[1] - down[1]) / (2 * h) - exact)
    tol = own + (up[2] + down[2]) / (2 * h) + gb
    assert tol < 0.05 * abs(exact) + 1.0                  # the test can tell a wrong gradient
    assert abs((up[0] - down[0]) / (2 * h) - slope) <= tol


def test_no_tokens(pkg, gpu):
    z = torch.empty(0, 4, 64, dtype=BF16, device=gpu)
    w = torch.ones(64, dtype=BF16, device=gpu)
    cos, sin = (t.to(gpu) for t in ref.tables(4, 64))
    pos = torch.empty(0, dtype=torch.int64, device=gpu)
    a, b = pkg.qk_norm_rope(z, z, w, w, cos, sin, pos)
    assert a.shape == b.shape == z.shape
    got = pkg.qk_norm_rope_bwd(z, z, z, z, w, w, cos, sin, pos)
    assert got[0].shape == z.shape and bool((got[2] == 0).all()) and bool((got[3] == 0).all())


def test_refusals(pkg, gpu):
    q = torch.zeros(3, 4, 64, dtype=BF16, device=gpu)
    k, w = q[:, :2].contiguous(), torch.ones(64, dtype=BF16, device=gpu)
    cos, sin = (t.to(gpu) for t in ref.tables(4, 64))
    pos = torch.zeros(3, dtype=torch.int64, device=gpu)
    ok = dict(q=q, k=k, q_weight=w, k_weight=w, cos=cos, sin=sin, positions=pos)
    for bad in (dict(k=k.half()), dict(k=k[:2]), dict(q_weight=w.float()), dict(cos=cos.double()),
                dict(sin=sin[:, :16]), dict(positions=pos[:2]), dict(q=q.transpose(1, 2)),
                dict(cos=cos[:, :12], sin=sin[:, :12]), dict(k=k.cpu()), dict(positions=pos.cpu()),
                dict(q_out=q[:, :3])):
        with pytest.raises(ValueError):
            pkg.qk_norm_rope(**{**ok, **bad})
    with pytest.raises(TypeError):
        pkg.qk_norm_rope(**{**ok, "positions": pos.float()})
    wide = torch.zeros(3, 4 * 64 + 4, dtype=BF16, device=gpu)
    odd = wide[:, 4:].unflatten(1, (4, 64))                # rows at 8-byte boundaries
    with pytest.raises(pkg.FagqError) as e:
        pkg.qk_norm_rope(**{**ok, "q": odd})
    assert e.value.status == 4
    with pytest.raises(pkg.FagqError) as e:
        pkg.qk_norm_rope(**ok, q_out=q[:1].expand(3, 4, 64))
    assert e.value.status == 9
    with pytest.raises(pkg.FagqError) as e:
        pkg.qk_norm_rope(**ok, eps=-1.0)
    assert e.value.status == 6
    with pytest.raises(pkg.FagqError) as e:
        pkg.qk_norm_rope_bwd(q, k, **ok, dq=q)
    assert e.value.status == 9
    with pytest.raises(ValueError):
        pkg.qk_norm_rope_bwd(q, k, **ok, workspace=torch.empty(8, dtype=torch.uint8, device=gpu))
