"""prompt_attention and prompt_attention_bwd on the GPU against their formulas in 64 bits
(tests/prompt_ref.py has them and the bounds): lengths from none to some hundred, keys longer and
shorter than queries, every type and head dim, grouped heads, views, and rows outside of all
sequences."""
import random

import pytest
import torch

from tests import attention_ref, prompt_ref as ref
from tests.gpu_util import note

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
NAN = float("nan")


def cumulative(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32)


def make(seed, lens, lens_k, Hq, H, D, dtype=BF16, spare=0, sharp=1.5):
    """q, k, v, dout, cu, cu_k on the CPU; `spare` rows of NaN behind the last sequence."""
    g = torch.Generator().manual_seed(seed)
    T, Tk = sum(lens), sum(lens if lens_k is None else lens_k)

    def rows(n, heads, f=1.0):
        x = torch.randn(n + spare, heads, D, generator=g) * f
        x[..., :2] *= 3.0
        x[n:] = NAN
        return x.to(dtype)

    q, k, v, do = rows(T, Hq, sharp), rows(Tk, H), rows(Tk, H), rows(T, Hq)
    return q, k, v, do, cumulative(lens), None if lens_k is None else cumulative(lens_k)


def forward(pkg, gpu, made, scale, **kw):
    q, k, v, _, cu, cu_k = made
    return pkg.prompt_attention(q.to(gpu), k.to(gpu), v.to(gpu), cu.to(gpu), scale,
                                cu_seqlens_k=None if cu_k is None else cu_k.to(gpu), return_lse=True, **kw)


def check(pkg, gpu, made, scale=None, bwd=True):
    q, k, v, do, cu, cu_k = made
    T, Tk = int(cu[-1]), int((cu if cu_k is None else cu_k)[-1])
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = forward(pkg, gpu, made, scale)
    assert out.dtype == q.dtype and out.shape == q.shape and out.is_contiguous()
    assert lse.dtype == torch.float32 and lse.shape == q.shape[1::-1]
    assert bool((out[T:] == 0).all()) and bool((lse[:, T:] == float("-inf")).all())
    o, o_off, s, s_off = ref.forward(q[:T], k[:Tk], v[:Tk], cu, scale, cu_k)
    assert attention_ref.outside(out[:T], o, o_off, q.dtype) == 0
    got = lse[:, :T].double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(s))
    some = ~torch.isinf(s)
    assert bool(((got - s).abs()[some] <= s_off[some]).all())
    if not bwd:
        return
    note("   backward")
    grads = pkg.prompt_attention_bwd(do.to(gpu), q.to(gpu), k.to(gpu), v.to(gpu), out, lse, cu.to(gpu),
                                     scale, cu_seqlens_k=None if cu_k is None else cu_k.to(gpu))
    want = ref.backward(do[:T], q[:T], k[:Tk], v[:Tk], out[:T].cpu(), lse[:, :T].cpu(), cu, scale, cu_k)
    for name, t, like, n, (r, off) in zip(("dq", "dk", "dv"), grads, (q, k, v), (T, Tk, Tk), want):
        assert t.dtype == q.dtype and t.shape == like.shape, name
        assert bool((t[n:] == 0).all()), name
        assert attention_ref.outside(t[:n], r, off, q.dtype) == 0, name


CASES = [
    # lens, lens_k, Hq, H, D, spare
    ([1], None, 1, 1, 64, 0), ([1, 0, 2], None, 4, 2, 128, 0), ([0, 0], None, 2, 1, 64, 3),
    ([31, 32, 33], None, 3, 3, 128, 0), ([63, 64, 65, 1], None, 8, 2, 64, 70), ([127, 128, 129], None, 4, 1, 128, 0),
    ([255, 257], None, 2, 1, 256, 5), ([300, 7, 0, 150], None, 10, 2, 128, 130), ([513], None, 5, 5, 64, 0),
    ([700], None, 16, 1, 128, 1), ([1] * 70, None, 2, 2, 64, 0), ([3, 40] * 40, None, 4, 4, 128, 9),
    # keys longer than queries, and shorter: the first queries see nothing
    ([1], [5], 1, 1, 64, 0), ([5], [1], 2, 1, 128, 0), ([33, 0, 64], [100, 7, 64], 4, 2, 128, 4),
    ([64, 200], [10, 0], 2, 2, 64, 0), ([1, 1, 1], [700, 1, 64], 8, 1, 256, 0), ([130], [1000], 6, 2, 128, 0),
    ([300], [70], 4, 1, 256, 2), ([17, 140], [400, 141], 12, 4, 64, 0), ([0, 0], [64, 3], 2, 1, 128, 0),
    ([40, 3], [0, 0], 2, 1, 128, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{len(c[0])}x{max(c[0])}k{max(c[1] or [0])}_{'_'.join(map(str, c[2:]))}")
def test_prompts(pkg, gpu, case, dtype):
    lens, lens_k, Hq, H, D, spare = case
    note(f"prompts {case} {dtype}")
    check(pkg, gpu, make(len(lens) * 31 + D, lens, lens_k, Hq, H, D, dtype, spare))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("case", [
    ([10], [1500], 4, 2, 64, 3), ([10, 0, 70], [1300, 9, 600], 3, 1, 128, 0), ([140], [2000], 4, 1, 256, 0),
    ([600], [1900], 8, 4, 64, 0), ([1030, 70], [1500, 3], 16, 16, 64, 5), ([1100], None, 16, 4, 128, 0),
    ([300, 200], [0, 2500], 4, 4, 128, 0), ([90], [700], 16, 2, 256, 1), ([400, 380], [1500, 1600], 4, 1, 256, 0),
], ids=lambda c: f"{len(c[0])}x{max(c[0])}k{max(c[1] or [0])}_{'_'.join(map(str, c[2:]))}")
def test_keys_in_parts(pkg, gpu, case, dtype):
    """Few queries of many keys: both directions cut a query tile's keys."""
    lens, lens_k, Hq, H, D, spare = case
    note(f"parts {case} {dtype}")
    check(pkg, gpu, make(len(lens) + D, lens, lens_k, Hq, H, D, dtype, spare))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("Hq,H", [(512, 256), (1024, 2)])
def test_many_heads_of_long_keys(pkg, gpu, Hq, H, dtype):
    """Workgroups of two heads: some heads against 64 bits, rows behind the last sequence filled."""
    note(f"two heads {Hq} {H} {dtype}")
    lens, lens_k = [130, 60], [2400, 2300]
    q, k, v, _, cu, cu_k = made = make(Hq, lens, lens_k, Hq, H, 128, dtype, 140)
    out, lse = forward(pkg, gpu, made, 0.09)
    T, Tk, group = sum(lens), sum(lens_k), Hq // H
    assert bool((out[T:] == 0).all()) and bool((lse[:, T:] == float("-inf")).all())
    for h in (0, H // 2, H - 1):
        for first in {0, group - 2}:
            own = slice(h * group + first, h * group + first + 2)
            o, o_off, s, s_off = ref.forward(q[:T, own], k[:Tk, h:h + 1], v[:Tk, h:h + 1], cu, 0.09, cu_k)
            assert attention_ref.outside(out[:T, own], o, o_off, dtype) == 0
            assert bool(((lse[own, :T].double().cpu() - s).abs() <= s_off).all())


@pytest.mark.parametrize("B", [64, 65, 255, 256, 257, 513, 1025])
def test_places_among_many_sequences(pkg, gpu, B):
    """Sequences of none to three tiles, the longest last or first, empty ones at either end."""
    note(f"places {B}")
    lens = [[0, 3, 1, 140, 0, 260][(i * 5 + i // 7) % 6] if 2 < i < B - 2 else 0 for i in range(B)]
    for order in (lens, lens[::-1]):
        q, k, v, do, cu, _ = made = make(B, order, None, 2, 1, 64, spare=200)
        T = sum(order)
        out, lse = forward(pkg, gpu, made, 0.2)
        assert bool((out[T:] == 0).all()) and bool((lse[:, T:] == float("-inf")).all())
        o, o_off, s, s_off = ref.forward(q[:T], k[:T], v[:T], cu, 0.2, None)
        assert attention_ref.outside(out[:T], o, o_off, BF16) == 0
        assert bool(((lse[:, :T].double().cpu() - s).abs() <= s_off).all())
        grads = pkg.prompt_attention_bwd(do.to(gpu), q.to(gpu), k.to(gpu), v.to(gpu), out, lse, cu.to(gpu), 0.2)
        want = ref.backward(do[:T], q[:T], k[:T], v[:T], out[:T].cpu(), lse[:, :T].cpu(), cu, 0.2, None)
        for t, (r, off) in zip(grads, want):
            assert bool((t[T:] == 0).all()) and attention_ref.outside(t[:T], r, off, BF16) == 0


@pytest.mark.parametrize("seed", range(16))
def test_random(pkg, gpu, seed):
    rng = random.Random(seed)
    H = rng.choice([1, 2, 3, 8])
    B = rng.randint(1, 9)
    lens = [rng.choice([0, rng.randint(1, 20), rng.randint(1, 260)]) for _ in range(B)]
    lens_k = [max(0, n + rng.randint(-30, 300)) for n in lens] if rng.random() < 0.5 else None
    D, Hq, dtype = rng.choice([64, 128, 256]), H * rng.choice([1, 2, 4, 5]), rng.choice([BF16, F16])
    spare = rng.choice([0, 1, 200])
    note(f"prompts seed {seed}: {lens} {lens_k} {Hq}/{H} D{D} {dtype} spare {spare}")
    check(pkg, gpu, make(seed, lens, lens_k, Hq, H, D, dtype, spare))


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_scales_of_either_sign(pkg, gpu, scale):
    note(f"prompts, scale {scale}")
    check(pkg, gpu, make(3, [100, 40], [130, 20], 4, 2, 128, sharp=0.5), scale)


@pytest.mark.parametrize("sharp", [0.0, 20.0])
def test_flat_and_sharp_softmax(pkg, gpu, sharp):
    note(f"prompts, sharpness {sharp}")
    check(pkg, gpu, make(4, [300, 17], None, 8, 2, 128, sharp=sharp))


def test_rising_scores(pkg, gpu):
    """Every key scores higher than the ones before: the running maximum moves with each step."""
    q, k, v, do, cu, _ = make(5, [600], None, 2, 1, 64)
    q[:] = 1.0
    k[:] = (torch.arange(600) / 600 * 8.0)[:, None, None].to(BF16)
    note("rising scores")
    check(pkg, gpu, (q, k, v, do, cu, None), 0.5)


def test_hidden_keys_do_not_matter(pkg, gpu):
    """Keys behind a query may hold anything, infinities and NaN among them."""
    made = make(6, [200], None, 4, 2, 128)
    q, k, v, do, cu, _ = made
    note("hidden keys")
    out, lse = forward(pkg, gpu, made, 0.1)
    for bad in (NAN, float("inf"), float("-inf"), torch.finfo(BF16).min):
        worse = k.clone()
        worse[150:] = bad
        o, s = forward(pkg, gpu, (q, worse, v, do, cu, None), 0.1)
        assert torch.equal(o[:150], out[:150]) and torch.equal(s[:, :150], lse[:, :150])


def test_views_of_fused_buffers(pkg, gpu):
    """q, k and v as slices of one projection, gradients into slices of another, any strides."""
    q, k, v, do, cu, _ = make(7, [150, 3, 60], None, 6, 2, 128)
    note("views")
    T = q.shape[0]
    made = [t.to(gpu) for t in (q, k, v, do, cu)]
    out, lse = pkg.prompt_attention(*made[:3], made[4], 0.1, return_lse=True)
    want = pkg.prompt_attention_bwd(made[3], *made[:3], out, lse, made[4], 0.1)
    fused = torch.cat(made[:3], 1)
    qv, kv, vv = fused[:, :6], fused[:, 6:8], fused[:, 8:]
    given = torch.full_like(out, 9.0)
    o, s = pkg.prompt_attention(qv, kv, vv, made[4], 0.1, return_lse=True, out=given)
    assert o is given and torch.equal(o, out) and torch.equal(s, lse)
    grad = torch.zeros_like(fused)
    heads_first = made[3].transpose(0, 1).contiguous().transpose(0, 1)
    got = pkg.prompt_attention_bwd(heads_first, qv, kv, vv, out, lse, made[4], 0.1, dq=grad[:, :6],
                                   dk=grad[:, 6:8], dv=grad[:, 8:])
    assert got[0].data_ptr() == grad.data_ptr()
    assert torch.equal(grad, torch.cat(want, 1))
    one = made[3][:1, :1].expand(T, 6, 128)
    a = pkg.prompt_attention_bwd(one, *made[:3], out, lse, made[4], 0.1)
    b = pkg.prompt_attention_bwd(one.contiguous(), *made[:3], out, lse, made[4], 0.1)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_rows_behind_the_last_sequence_of_given_outputs(pkg, gpu):
    made = make(8, [100, 30], None, 4, 2, 64, spare=300)
    q, k, v, do, cu, _ = [None if t is None else t.to(gpu) for t in made]
    note("rows behind the last sequence")
    out = torch.full_like(q, 7.0)
    _, lse = pkg.prompt_attention(q, k, v, cu, 0.1, return_lse=True, out=out)
    assert bool((out[130:] == 7.0).all()) and not bool((out[:130] == 7.0).any(-1).all())
    grads = [torch.full_like(t, 7.0) for t in (q, k, v)]
    got = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.1, dq=grads[0], dk=grads[1], dv=grads[2])
    clean = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.1)
    for a, b in zip(got, clean):
        assert bool((a[130:] == 7.0).all()) and bool((b[130:] == 0.0).all())
        assert torch.equal(a[:130], b[:130])


@pytest.mark.parametrize("cu", [[0, 500, 90], [-5, 40, 2 ** 31 - 1], [100, 50, 0], [0, 0, 0], [30, 60, 90],
                                [-2 ** 31, -1, 20]])
def test_lengths_of_any_value(pkg, gpu, cu):
    """Nothing is read or written outside the tensors, whatever the lengths hold."""
    note(f"lengths {cu}")
    buf = [torch.full((90 + 64, 2, 64), 3.0, dtype=BF16, device=gpu) for _ in range(8)]
    q, k, v, do, out, dq, dk, dv = [t[32:122] for t in buf]
    cu = torch.tensor(cu, dtype=torch.int32, device=gpu)
    good = torch.tensor([0, 45, 90], dtype=torch.int32, device=gpu)
    for a, b in ((cu, None), (good, cu), (cu, good)):
        _, lse = pkg.prompt_attention(q, k, v, a, 0.1, cu_seqlens_k=b, return_lse=True, out=out)
        pkg.prompt_attention_bwd(do, q, k, v, out, lse, a, 0.1, cu_seqlens_k=b, dq=dq, dk=dk, dv=dv)
        torch.cuda.synchronize()
        assert all(bool((t[:32] == 3.0).all()) and bool((t[122:] == 3.0).all()) for t in buf)


def test_lengths_that_add_up_to_any_number(pkg, gpu):
    """65536 sequences of which every second one claims all of 2^24 rows: 2^32 tiles."""
    T, B = 1 << 24, 1 << 16
    note("overlapping sequences")
    buf = torch.full((T + 64, 1, 64), 3.0, dtype=BF16, device=gpu)
    q, k = torch.zeros(T, 1, 64, dtype=BF16, device=gpu), torch.zeros(8, 1, 64, dtype=BF16, device=gpu)
    cu = torch.tensor([0, T], dtype=torch.int32, device=gpu).repeat(B // 2 + 1)[:B + 1].contiguous()
    pkg.prompt_attention(q, k, k, cu, 0.1, cu_seqlens_k=torch.zeros_like(cu), out=buf[32:T + 32])
    torch.cuda.synchronize()
    assert bool((buf[:32] == 3.0).all()) and bool((buf[T + 32:] == 3.0).all())
    assert bool(((buf == 0.0) | (buf == 3.0)).all()) and bool((buf == 0.0).any())


@pytest.mark.parametrize("lens,Hq,H,D", [([300, 20, 0], 4, 1, 128), ([900], 8, 2, 64), ([64], 2, 2, 256)])
def test_workspaces(pkg, gpu, lens, Hq, H, D):
    """Nothing is written past the bytes a caller is told, and what they held does not matter."""
    from fagq_mi355x import prompt
    note(f"workspaces {lens} {Hq} {H} {D}")
    q, k, v, do, cu, _ = [None if t is None else t.to(gpu) for t in make(9, lens, None, Hq, H, D)]
    sizes = (len(lens), q.shape[0], q.shape[0], Hq, H, D)
    out, lse = pkg.prompt_attention(q, k, v, cu, 0.1, return_lse=True)
    want = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.1)
    for fill in (0, 0xFF):
        for need, call, ok in (
                (prompt.workspace_bytes(*sizes),
                 lambda w: [pkg.prompt_attention(q, k, v, cu, 0.1, workspace=w)], [out]),
                (prompt.bwd_workspace_bytes(*sizes),
                 lambda w: pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.1, workspace=w), want)):
            buf = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=gpu)
            buf[:need] = fill
            got = call(buf[:max(need, 16)])
            assert all(torch.equal(a, b) for a, b in zip(got, ok))
            assert bool((buf[max(need, 16):] == 0xA5).all())
            if need:
                with pytest.raises(ValueError):
                    call(buf[:need - 1])


def test_gradients_against_differences(pkg, gpu):
    """The slope of sum(dout out) along a direction, from the formula in 64 bits at two points."""
    q, k, v, do, cu, cu_k = made = make(10, [40, 70], [90, 64], 4, 2, 64, F16)
    note("differences")
    out, lse = forward(pkg, gpu, made, 0.125)
    grads = pkg.prompt_attention_bwd(do.to(gpu), q.to(gpu), k.to(gpu), v.to(gpu), out, lse, cu.to(gpu),
                                     0.125, cu_seqlens_k=cu_k.to(gpu))
    want = ref.backward(do, q, k, v, out.cpu(), lse.cpu(), cu, 0.125, cu_k)
    # delta of the rounded out: half a step of each value, in the units of P k and P q.
    exact = ref.forward(q, k, v, cu, 0.125, cu_k)
    unrounded = ref.backward(do, q, k, v, exact[0], exact[2], cu, 0.125, cu_k)
    g, step = torch.Generator().manual_seed(11), 1e-5
    for i, x in enumerate((q, k, v)):
        way = torch.randn(x.shape, generator=g, dtype=torch.float64)
        ends = []
        for sign in (1, -1):
            moved = [t.double() for t in (q, k, v)]
            moved[i] = moved[i] + sign * step * way
            ends.append((ref_double(*moved, cu, 0.125, cu_k) * do.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * step)
        assert abs(float((unrounded[i][0] * way).sum() - slope)) <= 1e-6 * float((unrounded[i][0] * way).abs().sum())
        off = want[i][1] + attention_ref.rounding(want[i][0].abs() + want[i][1], F16) + \
            (want[i][0] - unrounded[i][0]).abs()
        assert abs(float((grads[i].double().cpu() * way).sum() - slope)) <= float((off * way.abs()).sum())


def ref_double(q, k, v, cu, scale, cu_k):
    """The output alone, in 64 bits from 64-bit inputs."""
    out = torch.zeros_like(q)
    g = q.shape[1] // k.shape[1]
    for rows, keys in ref.spans(cu, cu_k):
        hide = ref.hidden(rows.stop - rows.start, keys.stop - keys.start)
        some = ~hide.all(1)
        for h in range(q.shape[1]):
            x = (q[rows, h] @ k[keys, h // g].T * scale).masked_fill(hide, float("-inf"))
            p = torch.softmax(torch.where(some[:, None], x, 0.0), 1) * some[:, None]
            out[rows, h] = p @ v[keys, h // g]
    return out


def test_empty_calls(pkg, gpu):
    q = torch.zeros(0, 4, 64, dtype=BF16, device=gpu)
    k = torch.zeros(0, 2, 64, dtype=BF16, device=gpu)
    for B in (0, 3):
        cu = torch.zeros(B + 1, dtype=torch.int32, device=gpu)
        out, lse = pkg.prompt_attention(q, k, k, cu, 0.1, return_lse=True)
        assert out.shape == q.shape and lse.shape == (4, 0)
        assert [t.shape for t in pkg.prompt_attention_bwd(q, q, k, k, out, lse, cu, 0.1)] == \
            [q.shape, k.shape, k.shape]
    rows = torch.ones(5, 4, 64, dtype=BF16, device=gpu)
    cu, none = torch.tensor([0, 5], dtype=torch.int32, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    out, lse = pkg.prompt_attention(rows, k, k, cu, 0.1, cu_seqlens_k=none, return_lse=True)
    assert bool((out == 0).all()) and bool((lse == float("-inf")).all())
    dq, dk, _ = pkg.prompt_attention_bwd(rows, rows, k, k, out, lse, cu, 0.1, cu_seqlens_k=none)
    assert bool((dq == 0).all()) and dk.shape == k.shape
    out = torch.empty(0, 4, 64, dtype=BF16, device=gpu)
    dq, dk, dv = pkg.prompt_attention_bwd(q, q, rows[:, :2], rows[:, :2], out, torch.empty(4, 0, device=gpu),
                                          none, 0.1, cu_seqlens_k=cu)
    assert bool((dk == 0).all()) and bool((dv == 0).all())


def test_refusals(pkg, gpu):
    q, k, v, do, cu, _ = [None if t is None else t.to(gpu) for t in make(12, [20, 12], None, 4, 2, 64)]
    out, lse = pkg.prompt_attention(q, k, v, cu, 0.1, return_lse=True)
    ok = dict(q=q, k=k, v=v, cu_seqlens=cu, sm_scale=0.1)
    shared = (dict(q=q[:, :3]), dict(q=q[:, 0]), dict(q=q.cpu()), dict(k=k[:-1]), dict(v=v[:-1]), dict(v=v.half()),
              dict(k=k.cpu()), dict(cu_seqlens=cu.long()), dict(cu_seqlens=cu.cpu()), dict(cu_seqlens=cu[:0]),
              dict(cu_seqlens_k=cu[:2]), dict(q=q[..., ::2].repeat(1, 1, 2)[..., ::2]),
              dict(q=q[..., :32], k=k[..., :32], v=v[..., :32]), dict(workspace=torch.empty(64, device="cpu")))
    for bad in shared + (dict(out=out[:-1]), dict(out=out.half())):
        with pytest.raises(ValueError):
            pkg.prompt_attention(**{**ok, **bad})
    back = dict(ok, dout=do, out=out, lse=lse)
    for bad in shared + (dict(dout=do[:-1]), dict(out=out[:-1]), dict(lse=lse.t()), dict(lse=lse.double()),
                         dict(dq=q[:-1].clone()), dict(dk=k.half())):
        with pytest.raises(ValueError):
            pkg.prompt_attention_bwd(**{**back, **bad})
    for f, a in ((pkg.prompt_attention, ok), (pkg.prompt_attention_bwd, back)):
        with pytest.raises(TypeError):
            f(**{**a, "q": q.float()})
        for bad, status in ((dict(sm_scale=NAN), 2), (dict(q=torch.zeros(32, 4, 68, device=gpu, dtype=BF16)[..., :64]), 4)):
            with pytest.raises(pkg.FagqError) as e:
                f(**{**a, **bad})
            assert e.value.status == status
    for f, a in ((pkg.prompt_attention, dict(ok, out=q)), (pkg.prompt_attention_bwd, dict(back, dq=q)),
                 (pkg.prompt_attention_bwd, dict(back, dk=k, dv=v)), (pkg.prompt_attention_bwd, dict(back, dq=do)),
                 (pkg.prompt_attention_bwd, dict(back, dk=torch.zeros_like(k[:1]).expand(32, 2, 64)))):
        with pytest.raises(pkg.FagqError) as e:
            f(**a)
        assert e.value.status == 9
