"""prompt_attention_bwd where 16 bits are short of range or of bits: gradients scaled far up or down, and
of thousands of tokens.  Against the formulas in 64 bits, from the out and lse that the call is given.

`excess`: the error's root mean square over that of rounding the formula's result to the type.  A sum
of n products whose factors are rounded once each, as the result is, errs by as much as the result's
rounding where its terms are of any sign, and by less where they add up: together sqrt(2), and 1.6 is
asked for.  Where factors keep twice the bits, only the rounding of the result is left (the rest are 32
bit sums, of 2^-24 a step): 1.1, which the same calls with one term of dS and P are past (1.31 to 1.47,
the formula in 32 bits with that rounding)."""
import pytest
import torch

from tests.gpu_util import note

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
ONCE, TWICE = 1.6, 1.1


def excess(got, want):
    rms = lambda t: float(t.double().pow(2).mean().sqrt())
    return rms(got.double() - want) / rms(want.to(got.dtype).double() - want)


def gradients(do, q, k, v, out, lse, scale, ahead=0):
    """dq, dk, dv of one sequence in 64 bits, on the tensors' device."""
    g, n, m = q.shape[1] // k.shape[1], q.shape[0], k.shape[0]
    hide = torch.ones(n, m, dtype=torch.bool, device=q.device).triu(ahead + 1)
    grads = [torch.zeros(t.shape, dtype=torch.float64, device=q.device) for t in (q, k, v)]
    for h in range(q.shape[1]):
        qq, gg, oo = (t[:, h].double() for t in (q, do, out))
        kk, vv = k[:, h // g].double(), v[:, h // g].double()
        p = torch.exp((qq @ kk.T * scale).masked_fill(hide, float("-inf")) - lse[h].double()[:, None])
        t = p * (gg @ vv.T - (gg * oo).sum(1)[:, None])
        grads[0][:, h] = t @ kk * scale
        grads[1][:, h // g] += t.T @ qq * scale
        grads[2][:, h // g] += p.T @ gg
    return grads


def run(pkg, gpu, seed, n, m, Hq, H, D, dtype, size, rise=0.0):
    """Gradients and the formula's; dout of standard deviation `size`, times 2^rise from the first query to
    the last."""
    g = torch.Generator().manual_seed(seed)
    q, do = (torch.randn(n, Hq, D, generator=g) for _ in range(2))
    k, v = (torch.randn(m, H, D, generator=g) for _ in range(2))
    do = do * size * torch.exp2(torch.arange(n) / n * rise)[:, None, None]
    assert float(do.abs().max()) < 65504.0
    q, k, v, do = (t.to(dtype).to(gpu) for t in (q, k, v, do))
    cu, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=gpu) for x in (n, m))
    scale = D ** -0.5
    out, lse = pkg.prompt_attention(q, k, v, cu, scale, cu_seqlens_k=cu_k, return_lse=True)
    got = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, scale, cu_seqlens_k=cu_k)
    want = gradients(do, q, k, v, out, lse, scale, m - n)
    for x in want:                                          # results that the type holds
        assert float(x.abs().max()) < torch.finfo(dtype).max
    return got, want


# One launch for both passes (two terms for dk and dv), two launches, keys or steps in parts.
SHAPES = [(512, 512, 1, 1, 128, True), (200, 200, 4, 2, 64, True), (150, 150, 2, 1, 256, True),
          (60, 3000, 2, 2, 64, True), (1300, 1300, 16, 4, 64, False), (1200, 1200, 16, 8, 128, False),
          (1100, 1100, 16, 16, 256, False), (400, 4000, 48, 8, 128, False)]
IDS = lambda s: "_".join(map(str, s[:5])) if isinstance(s, tuple) else None


def accurate(got, want, one_launch, bands=1):
    """bands: of rows, each measured by itself."""
    for name, x, r in zip(("dq", "dk", "dv"), got, want):
        assert bool(torch.isfinite(x).all()), name
        e = [excess(a, b) for a, b in zip(x.tensor_split(bands), r.tensor_split(bands))]
        print(f"   {name}", *(f"{v:.3f}" for v in e), flush=True)
        assert max(e) <= (TWICE if one_launch or name == "dq" else ONCE), name


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("size", ["largest", 6000.0, 1.0, 1e-3, 1e-4])
def test_gradients_of_any_size(pkg, gpu, shape, size):
    """fp16 gradients of scaled losses: dS leaves the type at either end, the results do not."""
    *sizes, one_launch = shape
    note(f"fp16 gradients {sizes} of {size}")
    if size == "largest":                                   # that dout and the results allow
        most = max(float(x.abs().max()) for x in run(pkg, gpu, 5, *sizes, F16, 1.0)[1])
        size = min(12000.0, 50000.0 / most)
    accurate(*run(pkg, gpu, 5, *sizes, F16, size), one_launch)


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_gradients_in_bf16(pkg, gpu, shape):
    *sizes, one_launch = shape
    note(f"bf16 gradients {sizes}")
    accurate(*run(pkg, gpu, 6, *sizes, BF16, 1.0), one_launch)


@pytest.mark.parametrize("rise", [20.0, -20.0])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_gradients_that_rise_and_fall(pkg, gpu, shape, rise):
    """dout 2^20 apart within a sequence: what a sum is scaled by moves with its largest term."""
    *sizes, one_launch = shape
    note(f"fp16 gradients {sizes}, 2^{rise}")
    accurate(*run(pkg, gpu, 7, *sizes, F16, 6000.0 * 2.0 ** -max(rise, 0.0), rise), one_launch, 6)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_gradients_of_thousands_of_tokens(pkg, gpu, D, dtype):
    note(f"gradients of 5000 tokens, heads of {D}, {dtype}")
    accurate(*run(pkg, gpu, 8, 5000, 5000, 4, 2, D, dtype, 1e-3 if dtype == F16 else 1.0), False)


def test_gradients_of_nothing(pkg, gpu):
    """dout of zeros, and of one query only."""
    note("fp16 gradients of zeros")
    n, D = 300, 64
    g = torch.Generator().manual_seed(9)
    q, k, v = (torch.randn(n, 2, D, generator=g).to(F16).to(gpu) for _ in range(3))
    cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    out, lse = pkg.prompt_attention(q, k, v, cu, 0.125, return_lse=True)
    do = torch.zeros_like(q)
    assert all(bool((x == 0).all()) for x in pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.125))
    do[170] = 1000.0
    got, want = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, 0.125), gradients(do, q, k, v, out, lse, 0.125)
    for x, r in zip(got, want):
        assert bool(torch.isfinite(x).all()) and bool((x[171:] == 0).all())
        assert excess(x, r) <= TWICE


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,Hq,H,D", [(200, 4, 2, 64), (1300, 16, 4, 64), (150, 2, 1, 256), (1200, 16, 16, 128)])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_an_overflow_is_not_hidden(pkg, gpu, n, Hq, H, D, dtype, bad):
    """A dout that a scaled loss has driven to infinity shows in every gradient that it enters, and in no
    other sequence's."""
    note(f"dout of {bad} {n} {Hq} {H} {D} {dtype}")
    g = torch.Generator().manual_seed(10)
    q, do = (torch.randn(n, Hq, D, generator=g).to(dtype).to(gpu) for _ in range(2))
    k, v = (torch.randn(n, H, D, generator=g).to(dtype).to(gpu) for _ in range(2))
    cu = torch.tensor([0, n - 70, n], dtype=torch.int32, device=gpu)
    out, lse = pkg.prompt_attention(q, k, v, cu, D ** -0.5, return_lse=True)
    clean = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, D ** -0.5)
    i, h = n - 100, Hq - 1
    do[i, h, 3] = bad
    dq, dk, dv = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, D ** -0.5)
    lost = lambda t: ~torch.isfinite(t)
    assert bool(lost(dq[i, h]).any()) and bool(lost(dk[:i + 1, H - 1]).any(-1).all())
    assert bool(lost(dv[:i + 1, H - 1, 3]).all())
    for x, y in zip((dq, dk, dv), clean):
        assert torch.equal(x[n - 70:], y[n - 70:])
    assert torch.equal(dq[:, :h], clean[0][:, :h]) and torch.equal(dq[:i, h], clean[0][:i, h])


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_fp16_scales_of_either_sign(pkg, gpu, scale):
    note(f"fp16 gradients, scale {scale}")
    g = torch.Generator().manual_seed(11)
    q, do = (torch.randn(130, 4, 64, generator=g).to(F16).to(gpu) for _ in range(2))
    k, v = (torch.randn(130, 2, 64, generator=g).to(F16).to(gpu) for _ in range(2))
    cu = torch.tensor([0, 130], dtype=torch.int32, device=gpu)
    out, lse = pkg.prompt_attention(q, k, v, cu, scale, return_lse=True)
    got = pkg.prompt_attention_bwd(do, q, k, v, out, lse, cu, scale)
    want = gradients(do, q, k, v, out, lse, scale)
    if scale == 0.0:
        assert bool((got[0] == 0).all()) and bool((got[1] == 0).all())
        got, want = got[2:], want[2:]
    assert all(excess(x, r) <= TWICE for x, r in zip(got, want))
