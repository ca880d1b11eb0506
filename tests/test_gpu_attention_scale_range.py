"""paged_attention with value scales at both ends of the documented range (0 to 2^64) in one row, at
scores of like size, whichever comes first: every key counts in the softmax's denominator however much
or little its value counts in the sum.

All value scales are set to one end, then one token's to the other; the token stands in the first step, in
a later one of the same wave, in another wave, chunk or share, in the prefix and behind it.

The kernel keeps a row's contributions relative to the largest of score + log2(value scale), scales below
2^-64 counting as 2^-64 there: probability x value scale is rounded to fp16, half a step of each (2^-11), and
at most 2^-24 of that largest for those that fp16 holds as subnormals.  The denominator's terms lie at
2^-64 of fp32's one and above, so what fp32 flushes below 2^-126 is 2^-62 of it for each key."""
import pytest
import torch

from tests import attention_ref as ref
from tests.gpu_util import note
from tests.test_gpu_attention_scales import FORMS, place
from tests.test_gpu_attention_schedule import widened
from tests.test_gpu_paged_attention import BF16, F16, FP8, INT8, clean, make, run

pytestmark = pytest.mark.gpu

LEAST = 2.0 ** -64


def expected(made, prefix, sm):
    """(out, bound) in 64 bits."""
    q, _, table, lens, pp = made
    (kc, ks), (vc, vs) = clean(made)
    B, S, Hq, D = q.shape
    P, H, g = kc.shape[0], kc.shape[1], Hq // kc.shape[1]
    wide = lambda s: ref.scale_value(s).double()[:, :, 0, :, None]
    kd, code, scale = kc.float().double() * wide(ks), vc.float().double(), wide(vs).expand(vc.shape)
    out = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    off = torch.zeros_like(out)
    for b in range(B):
        rows = [torch.cat([ref.token_rows(t, pp.tolist() if prefix else [], prefix, P)[0],
                           ref.token_rows(t, table[b].tolist(), int(lens[b]), P)[0]]) for t in (kd, code, scale)]
        for s in range(S):
            n = prefix + max(0, int(lens[b]) - S + s + 1)
            if n == 0:
                continue
            k, c, w = (r[:n] for r in rows)
            for h in range(H):
                at = (b, s, slice(h * g, (h + 1) * g))
                qq = q[at].double()
                mx = (qq.abs() @ k[:, h].abs().T * sm).amax(-1, keepdim=True)
                p = torch.softmax(qq @ k[:, h].T * sm, -1)
                top = (p * w[:, h, 0].clamp_min(LEAST)).amax(-1, keepdim=True)
                p = p * w[:, h, 0]
                out[at] = p @ c[:, h]
                off[at] = (p @ c[:, h].abs() * (2.0 ** -11 + 4 * mx * (D + 4) * ref.U + (n + 40) * ref.U + n * 2.0 ** -62)
                           + 2.0 ** -24 * top * c[:, h].abs().sum(0))
    return out, off


def set_scales(made, prefix, common, one, where):
    """Every value scale that is not poisoned becomes `common`, those of token `where` of each sequence
    (of the prefix ahead of it, once) `one`."""
    vs, lens = made[1][1][1], made[3]
    stored = lambda v: v if vs.dtype == torch.float32 else int(torch.tensor(v).log2()) + 127
    dead = torch.isnan(vs) if vs.dtype == torch.float32 else vs == 255
    vs[~dead] = stored(common)
    for b in range(len(lens)):
        if where < prefix + int(lens[b]):
            page, at = place(made, prefix, where, b)
            vs[page, :, 0, at] = stored(one)


ENDS = [
    # scale of all, of one token; fp16 holds no result near 2^64
    (FP8, False, BF16, 0.0, 2.0 ** 64), (FP8, False, BF16, 2.0 ** -64, 2.0 ** 64), (INT8, True, BF16, 2.0 ** -64, 2.0 ** 64),
    (INT8, False, BF16, 2.0 ** 64, 0.0), (FP8, True, BF16, 2.0 ** 64, 2.0 ** -64), (INT8, True, BF16, 2.0 ** -40, 2.0 ** 60),
    (FP8, False, F16, 0.0, 2.0 ** 4), (INT8, False, F16, 2.0 ** -64, 1.0), (FP8, True, F16, 2.0 ** -10, 2.0 ** -64),
    (INT8, False, BF16, 2.0 ** -64, 2.0 ** -64), (FP8, False, BF16, 2.0 ** 64, 2.0 ** 64), (FP8, False, BF16, 0.0, 0.0),
]


@pytest.mark.parametrize("ends", ENDS, ids=lambda e: "_".join(str(x).replace("torch.", "") for x in e))
@pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{len(f[0])}x{max(f[0])}_{'_'.join(map(str, f[1:]))}")
def test_both_ends_in_any_order(pkg, gpu, form, ends):
    lens, S, Hq, H, D, prefix, most = form
    qdt, ue8m0, dtype, common, one = ends
    note(f"scale range {form} {ends}")
    for where in (0, 37, 131, 165, max(lens) + prefix - 1):
        made = make(D + where, lens, S, Hq, H, D, 16, prefix, qdt, ue8m0, dtype, sharp=0.5)
        set_scales(made, prefix, common, one, where)
        for equal in (False, True):
            if equal:                      # codes of zero: every score is 0
                codes, scales = made[1][0]
                live = (scales[:, :, 0] != 255) if ue8m0 else ~torch.isnan(scales[:, :, 0])
                codes.view(torch.uint8)[live] = 0
            r, bound = expected(made, prefix, D ** -0.5)
            o = run(pkg, gpu, made if most is None else widened(made, most, 16), prefix)
            assert ref.outside(o, r, bound, dtype) == 0, (where, equal)
